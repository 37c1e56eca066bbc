// AdamW over many tensors in one launch, moments in 32 bits or as e4m3 blocks of 256.
//
//     m = b1 m + (1 - b1) g,   v = b2 v + (1 - b2) g^2
//     p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// A pure stream: 28 bytes an element with 32-bit moments and fp32 parameters, 16 with 8-bit ones (22 and 10 for 16-bit
// parameters), so the kernel is bound by memory, and for a small model by the launch.  90 M elements take 374 us at
// 6.7 TB/s and 235 at 6.2 TB/s (295 at 6.7, and 232 at 3.9: at 10 bytes an element its instructions bound it, the schedulers
// issue in 90 % of the cycles).
//
// The table of tensors (pointers, sizes, the prefix of their block counts) travels in the launch's own parameters: no
// copy to the device, nothing to keep alive, and a captured graph owns its table.  A warp takes 256 consecutive
// elements of one tensor: lane l holds elements 4 l .. 4 l + 3 and 128 + 4 l .. 128 + 4 l + 3, so every access of a
// warp is contiguous, and the block of an 8-bit moment is the warp's own.
//
// 8-bit moments: m and sqrt(v) are held as e4m3 codes with a scale per 256 elements.  The square root halves the
// exponent range that v needs; the code of sqrt(v) is at least the type's smallest value where v > 0, so that no
// element divides by eps alone because its neighbours are large.  The update itself uses the new moments in 32
// bits, before they are rounded for storage.
#include "lowp.cuh"

namespace gnnagg {
namespace {

constexpr int kThreads = 256;
constexpr int kWarpElems = 256;                          // elements of a warp's turn, and of a moment's block
constexpr int kBlockElems = kThreads / 32 * kWarpElems;  // elements of one block of the grid

struct Entry {
    void *p;             // parameter (fp32, bf16 or fp16)
    const void *g;       // gradient, same type
    void *m, *v;         // moments: fp32, or codes
    float *scales;       // [blocks of 256][2], 8-bit moments only
    float *master;       // fp32 copy of a 16-bit parameter, or null
    int64_t n;
    int64_t vec;         // every pointer allows 4-element accesses
};

struct Scalars {
    float decay, step_size, inv_sqrt_c2, b1, one_minus_b1, b2, one_minus_b2, eps;
};

template <int CAP>
struct Table {
    Entry e[CAP];
    alignas(16) int32_t first[CAP];  // grid block that starts each tensor; behind the last one the largest value
    Scalars s;
    const Scalars *device_scalars;  // used instead of s when set
};
constexpr int kNear = 16;  // entries that are compared without a search
constexpr int kSmallCap = kNear, kMidCap = 64, kLargeCap = 480;
static_assert(sizeof(Table<kLargeCap>) <= 32764, "kernel parameters");

// Four elements as they lie in memory, those behind the end as zeros; converted after the last load, in pairs.  With
// the conversion inside the branch below, a 16-bit type's loads wait for one another: 90 M bf16 parameters took 352 us
// instead of 293, and with 8-bit moments a third longer.
template <typename T>
struct Raw4 {
    uint32_t w[sizeof(T)];
};
template <typename T>
__device__ __forceinline__ Raw4<T> load4(const T *p, int64_t at, int64_t n, bool vec) {
    Raw4<T> r;
    if (vec && at + 4 <= n) {
        if (sizeof(T) == 4) {
            const uint4 u = __ldcs(reinterpret_cast<const uint4 *>(p + at));
            r.w[0] = u.x, r.w[1] = u.y, r.w[2 % sizeof(T)] = u.z, r.w[3 % sizeof(T)] = u.w;
        } else {
            const uint2 u = __ldcs(reinterpret_cast<const uint2 *>(p + at));
            r.w[0] = u.x, r.w[1] = u.y;
        }
    } else if (sizeof(T) == 4) {
        const uint32_t *q = reinterpret_cast<const uint32_t *>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) r.w[i % sizeof(T)] = at + i < n ? q[at + i] : 0;
    } else {
        const uint16_t *q = reinterpret_cast<const uint16_t *>(p);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t a = at + 2 * i < n ? q[at + 2 * i] : 0, b = at + 2 * i + 1 < n ? q[at + 2 * i + 1] : 0;
            r.w[i] = a | (b << 16);
        }
    }
    return r;
}
template <typename T>
__device__ __forceinline__ void put(Raw4<float> &to, const Raw4<T> &from) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T); ++i) to.w[i] = from.w[i];
}
template <typename T>
__device__ __forceinline__ Raw4<T> first(const Raw4<float> &from) {
    Raw4<T> r;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T); ++i) r.w[i] = from.w[i];
    return r;
}
template <typename T>
__device__ __forceinline__ void convert4(const Raw4<T> &r, float (&f)[4]) {
    if (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(r.w[i % sizeof(T)]);
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (std::is_same<T, __nv_bfloat16>::value) {  // the upper half of an fp32
                f[2 * i] = __uint_as_float(r.w[i] << 16), f[2 * i + 1] = __uint_as_float(r.w[i] & 0xFFFF0000u);
            } else {
                const float2 v = __half22float2(*reinterpret_cast<const __half2 *>(&r.w[i]));
                f[2 * i] = v.x, f[2 * i + 1] = v.y;
            }
        }
    }
}
template <typename T>
__device__ __forceinline__ void store4(T *p, int64_t at, int64_t n, bool vec, const float (&f)[4]) {
    if (vec && at + 4 <= n) {
        if (sizeof(T) == 4) {
            __stcs(reinterpret_cast<float4 *>(p + at), make_float4(f[0], f[1], f[2], f[3]));
        } else {
            uint32_t u[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (std::is_same<T, __nv_bfloat16>::value) {
                    const __nv_bfloat162 b = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
                    u[i] = *reinterpret_cast<const uint32_t *>(&b);
                } else {
                    const __half2 b = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
                    u[i] = *reinterpret_cast<const uint32_t *>(&b);
                }
            }
            __stcs(reinterpret_cast<uint2 *>(p + at), make_uint2(u[0], u[1]));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (at + i < n) p[at + i] = from_f32<T>(f[i]);
    }
}
__device__ __forceinline__ uint32_t load_codes(const uint8_t *p, int64_t at, int64_t n, bool vec) {
    if (vec && at + 4 <= n) return __ldcs(reinterpret_cast<const uint32_t *>(p + at));
    uint32_t u = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (at + i < n) u |= (uint32_t)p[at + i] << (8 * i);
    return u;
}
__device__ __forceinline__ void store_codes(uint8_t *p, int64_t at, int64_t n, bool vec, uint32_t u) {
    if (vec && at + 4 <= n) {
        __stcs(reinterpret_cast<uint32_t *>(p + at), u);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (at + i < n) p[at + i] = (uint8_t)(u >> (8 * i));
    }
}
// The root to one ulp, where it is used only in the update; the quotient there is good to two (its denominator is far
// below 2^126).  The exact ones cost a third of the kernel's instructions.
__device__ __forceinline__ float sqrt_approx(float x) {
    float r;
    asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint32_t warp_max(uint32_t v) { return __reduce_max_sync(kFullMask, v); }

template <typename T, bool EIGHT, int CAP>
__global__ void __launch_bounds__(kThreads) adamw_kernel(const __grid_constant__ Table<CAP> t) {
    // The tensor of this block: the last entry whose first block is not behind it.  Halving down to 16 entries, then one
    // comparison each: those do not wait for one another (13 tensors of 245 M elements together: 598 -> 588 us).
    const int block = (int)blockIdx.x;
    int lo = 0;
    if (CAP > kNear) {
        int parts = CAP / kNear;
        while (parts > 1) {
            const int half = parts >> 1;
            if (t.first[lo + half * kNear] <= block) {
                lo += half * kNear;
                parts -= half;
            } else {
                parts = half;
            }
        }
    }
    int before = 0;
#pragma unroll
    for (int i = 1; i < kNear; ++i) before += t.first[lo + i] <= block;
    lo += before;
    const Entry &e = t.e[lo];
    const int lane = threadIdx.x & 31;
    const int64_t n = e.n;
    const int64_t base = (int64_t)(block - t.first[lo]) * kBlockElems + (threadIdx.x >> 5) * kWarpElems;
    if (base >= n) return;  // whole warps
    const bool vec = e.vec != 0;
    T *p = static_cast<T *>(e.p);
    const T *g = static_cast<const T *>(e.g);
    const int64_t at[2] = {base + 4 * lane, base + 128 + 4 * lane};
    Raw4<T> raw_g[2];
    Raw4<float> raw_w[2], raw_m[2], raw_v[2];  // raw_w: the master copy, or in its first words the parameter
    uint32_t mc[2], vc[2];
    float2 sc = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if (e.master != nullptr)
            raw_w[h] = load4<float>(e.master, at[h], n, vec);
        else
            put(raw_w[h], load4<T>(p, at[h], n, vec));
        raw_g[h] = load4<T>(g, at[h], n, vec);
        if (EIGHT) {
            mc[h] = load_codes(static_cast<const uint8_t *>(e.m), at[h], n, vec);
            vc[h] = load_codes(static_cast<const uint8_t *>(e.v), at[h], n, vec);
        } else {
            raw_m[h] = load4<float>(static_cast<const float *>(e.m), at[h], n, vec);
            raw_v[h] = load4<float>(static_cast<const float *>(e.v), at[h], n, vec);
        }
    }
    if (EIGHT) sc = *reinterpret_cast<const float2 *>(e.scales + 2 * (base / kWarpElems));
    const Scalars s = t.device_scalars != nullptr ? *t.device_scalars : t.s;
    uint32_t top_m = 0, top_r = 0;
    float w[2][4], m[2][4], v[2][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float gr[4];
        if (e.master != nullptr)
            convert4(raw_w[h], w[h]);
        else
            convert4(first<T>(raw_w[h]), w[h]);
        convert4(raw_g[h], gr);
        if (!EIGHT) {
            convert4(raw_m[h], m[h]);
            convert4(raw_v[h], v[h]);
        } else {
            const float4 a = from_e4m3x4(mc[h]), b = from_e4m3x4(vc[h]);
            m[h][0] = __fmul_rn(a.x, sc.x), m[h][1] = __fmul_rn(a.y, sc.x);
            m[h][2] = __fmul_rn(a.z, sc.x), m[h][3] = __fmul_rn(a.w, sc.x);
            v[h][0] = __fmul_rn(b.x, sc.y), v[h][1] = __fmul_rn(b.y, sc.y);
            v[h][2] = __fmul_rn(b.z, sc.y), v[h][3] = __fmul_rn(b.w, sc.y);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[h][i] = __fmul_rn(v[h][i], v[h][i]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            // each step rounded on its own: an 8-bit moment's code then depends on the formula alone
            const float x = gr[i];
            m[h][i] = __fadd_rn(__fmul_rn(m[h][i], s.b1), __fmul_rn(x, s.one_minus_b1));
            v[h][i] = __fadd_rn(__fmul_rn(v[h][i], s.b2), __fmul_rn(__fmul_rn(x, x), s.one_minus_b2));
            const float r = EIGHT ? __fsqrt_rn(v[h][i]) : sqrt_approx(v[h][i]);
            w[h][i] = w[h][i] * s.decay - __fdividef(s.step_size * m[h][i], r * s.inv_sqrt_c2 + s.eps);
            if (EIGHT) {
                top_m = max(top_m, abs_bits(m[h][i]));
                top_r = max(top_r, abs_bits(r));
                v[h][i] = r;
            }
        }
        if (e.master != nullptr) store4<float>(e.master, at[h], n, vec, w[h]);
        store4<T>(p, at[h], n, vec, w[h]);
        if (!EIGHT) {
            store4<float>(static_cast<float *>(e.m), at[h], n, vec, m[h]);
            store4<float>(static_cast<float *>(e.v), at[h], n, vec, v[h]);
        }
    }
    if (EIGHT) {
        // elements behind the tensor's end are zeros (zero gradient, zero codes) and raise no maximum
        const float am = block_amax(warp_max(top_m)), ar = block_amax(warp_max(top_r));
        const float fm = block_factor(am), fr = block_factor(ar);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float r[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float u = __fmul_rn(v[h][i], fr);
                r[i] = v[h][i] > 0.0f && u < 0.001953125f ? 0.001953125f : u;
            }
            store_codes(static_cast<uint8_t *>(e.m), at[h], n, vec,
                        e4m3x4(__fmul_rn(m[h][0], fm), __fmul_rn(m[h][1], fm), __fmul_rn(m[h][2], fm),
                               __fmul_rn(m[h][3], fm)));
            store_codes(static_cast<uint8_t *>(e.v), at[h], n, vec, e4m3x4(r[0], r[1], r[2], r[3]));
        }
        if (lane == 0)
            *reinterpret_cast<float2 *>(e.scales + 2 * (base / kWarpElems)) = make_float2(block_scale(am), block_scale(ar));
    }
}

Scalars scalars_of(double lr, double b1, double b2, double eps, double weight_decay, double t) {
    Scalars s;
    s.decay = (float)(1.0 - lr * weight_decay);
    s.step_size = (float)(lr / -expm1(t * log(b1)));
    s.inv_sqrt_c2 = (float)(1.0 / sqrt(-expm1(t * log(b2))));
    s.b1 = (float)b1, s.one_minus_b1 = (float)(1.0 - b1);
    s.b2 = (float)b2, s.one_minus_b2 = (float)(1.0 - b2);
    s.eps = (float)eps;
    return s;
}

// The step count and the rate on the device, for launches that a graph replays: counts the step and leaves the
// scalars of this one.  The bias corrections are taken in 64 bits: 1 - 0.999^t at t = 1 keeps 4 digits in 32.
__global__ void adamw_tick_kernel(int64_t *step, const float *lr, double host_lr, double b1, double b2, double eps,
                                  double weight_decay, Scalars *out) {
    const int64_t t = *step + 1;
    *step = t;
    const double rate = lr != nullptr ? (double)*lr : host_lr;
    Scalars s;
    s.decay = (float)(1.0 - rate * weight_decay);
    s.step_size = (float)(rate / -expm1((double)t * log(b1)));
    s.inv_sqrt_c2 = (float)(1.0 / sqrt(-expm1((double)t * log(b2))));
    s.b1 = (float)b1, s.one_minus_b1 = (float)(1.0 - b1);
    s.b2 = (float)b2, s.one_minus_b2 = (float)(1.0 - b2);
    s.eps = (float)eps;
    *out = s;
}

bool vec4(const void *p, int size) { return reinterpret_cast<uintptr_t>(p) % (4 * size) == 0; }

template <typename T, bool EIGHT, int CAP>
int launch(const gnnagg_adamw_tensor *ts, int count, const Scalars &s, const Scalars *device_scalars, cudaStream_t st) {
    Table<CAP> t;
    int64_t blocks = 0;
    int used = 0;
    for (int i = 0; i < count; ++i) {
        const gnnagg_adamw_tensor &x = ts[i];
        if (x.n == 0) continue;
        Entry &e = t.e[used++];
        e.p = x.param, e.g = x.grad, e.m = x.exp_avg, e.v = x.exp_avg_sq, e.scales = x.scales, e.master = x.master;
        e.n = x.n;
        t.first[used - 1] = (int32_t)blocks;
        const int ms = EIGHT ? 1 : 4;
        e.vec = vec4(e.p, (int)sizeof(T)) && vec4(e.g, (int)sizeof(T)) && vec4(e.m, ms) && vec4(e.v, ms) &&
                (e.master == nullptr || vec4(e.master, 4));
        blocks += div_up(x.n, kBlockElems);
        if (blocks >= 0x7FFFFFFF) return fail(GNNAGG_ERR_UNSUPPORTED, "adamw_step: too many elements for one launch");
    }
    if (used == 0) return GNNAGG_OK;
    t.s = s;
    t.device_scalars = device_scalars;
    for (int i = used; i < CAP; ++i) t.first[i] = 0x7FFFFFFF;
    adamw_kernel<T, EIGHT, CAP><<<(unsigned)blocks, kThreads, 0, st>>>(t);
    return check_launch("adamw_kernel");
}

// Tables of three sizes: a launch carries all of its parameters, 32 KB with 480 entries, 1 KB with 16.
template <typename T, bool EIGHT>
int launch_all(const gnnagg_adamw_tensor *ts, int64_t count, const Scalars &s, const Scalars *ds, cudaStream_t st) {
    for (int64_t i = 0; i < count; i += kLargeCap) {
        const int part = (int)(count - i < kLargeCap ? count - i : kLargeCap);
        const int rc = part <= kSmallCap ? launch<T, EIGHT, kSmallCap>(ts + i, part, s, ds, st)
                       : part <= kMidCap ? launch<T, EIGHT, kMidCap>(ts + i, part, s, ds, st)
                                         : launch<T, EIGHT, kLargeCap>(ts + i, part, s, ds, st);
        if (rc != GNNAGG_OK) return rc;
    }
    return GNNAGG_OK;
}

}  // namespace
}  // namespace gnnagg

using namespace gnnagg;

extern "C" size_t gnnagg_adamw_scalars_bytes(void) { return sizeof(Scalars); }

extern "C" int gnnagg_adamw_tick(int64_t *step, const float *lr, double host_lr, double beta1, double beta2, double eps,
                                 double weight_decay, void *scalars, void *stream) {
    if (step == nullptr || scalars == nullptr) return fail(GNNAGG_ERR_ARG, "adamw_tick: null pointer");
    if (!(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0))
        return fail(GNNAGG_ERR_ARG, "adamw_tick: betas must be in [0, 1)");
    adamw_tick_kernel<<<1, 1, 0, static_cast<cudaStream_t>(stream)>>>(step, lr, host_lr, beta1, beta2, eps, weight_decay,
                                                                      static_cast<Scalars *>(scalars));
    return check_launch("adamw_tick_kernel");
}

extern "C" int gnnagg_adamw_step(const gnnagg_adamw_tensor *tensors, int64_t count, int32_t type, int32_t state_bits,
                                 double lr, double beta1, double beta2, double eps, double weight_decay, int64_t step,
                                 const void *device_scalars, void *stream) {
    if (count < 0 || (count > 0 && tensors == nullptr)) return fail(GNNAGG_ERR_ARG, "adamw_step: null table or negative count");
    if (type_size(type) == 0) return fail(GNNAGG_ERR_ARG, "adamw_step: unknown element type %d", type);
    if (state_bits != 32 && state_bits != 8) return fail(GNNAGG_ERR_ARG, "adamw_step: moments have 32 or 8 bits");
    if (!(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0))
        return fail(GNNAGG_ERR_ARG, "adamw_step: betas must be in [0, 1)");
    if (device_scalars == nullptr && step < 1) return fail(GNNAGG_ERR_ARG, "adamw_step: the first step is 1");
    for (int64_t i = 0; i < count; ++i) {
        const gnnagg_adamw_tensor &x = tensors[i];
        if (x.n < 0) return fail(GNNAGG_ERR_ARG, "adamw_step: tensor %lld has a negative size", (long long)i);
        if (x.n == 0) continue;
        if (x.param == nullptr || x.grad == nullptr || x.exp_avg == nullptr || x.exp_avg_sq == nullptr ||
            (state_bits == 8 && x.scales == nullptr))
            return fail(GNNAGG_ERR_ARG, "adamw_step: tensor %lld has a null pointer", (long long)i);
        if (state_bits == 8 && reinterpret_cast<uintptr_t>(x.scales) % 8 != 0)
            return fail(GNNAGG_ERR_UNSUPPORTED, "adamw_step: scales of tensor %lld are not 8-byte aligned", (long long)i);
    }
    Scalars s = {};
    if (device_scalars == nullptr) s = scalars_of(lr, beta1, beta2, eps, weight_decay, (double)step);
    const Scalars *ds = static_cast<const Scalars *>(device_scalars);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool eight = state_bits == 8;
    switch (type) {
        case kTypeF32:
            return eight ? launch_all<float, true>(tensors, count, s, ds, st) : launch_all<float, false>(tensors, count, s, ds, st);
        case kTypeBf16:
            return eight ? launch_all<__nv_bfloat16, true>(tensors, count, s, ds, st)
                         : launch_all<__nv_bfloat16, false>(tensors, count, s, ds, st);
        default:
            return eight ? launch_all<__half, true>(tensors, count, s, ds, st) : launch_all<__half, false>(tensors, count, s, ds, st);
    }
}
