// Root-mean-square norm with the residual's addition, its gradients, and its output as e4m3 codes.
//
//     h = x + residual (rounded to the stream's type: h is an output, and the norm is of what is stored)
//     y = h * r * w,   r = rsqrt(mean(h^2) + eps)
//     dh = gh + r * (w gy - hat * mean(w gy hat)),  hat = h r;   dw = sum over rows of gy hat
//
// Forward is one pass: a row stays in registers, as it lies in memory, between the sum of squares and the scaling.  A
// row of up to 16 16-byte chunks belongs to half a warp, of up to 128 to a warp (short ones two at a time, so that a warp
// has 1 to 2 KB on their way), a longer one to a block of as many threads as it fills.  Backward reads h and the two gradients
// once, writes dh once and keeps the column sums of dw in registers over all rows of a persistent block; a second kernel
// adds the blocks' sums in a fixed order (no atomics).
//
// Bound by memory forward: 612500 x 256 bf16 with a residual in 192 us, 6.5 TB/s (codes: 195, 5.7 TB/s); 8191 x 5000 in 56.
// Backward 227 us, 5.5 TB/s, and 84 us, column sums included (9 of them each).  In the wide one nothing is full: the
// schedulers issue in 56 % of the cycles, DRAM reads at 51 % of its rate; a block waits for its row, reduces it and waits at
// the barrier, with the next row on its way and three blocks an SM to fill the gaps.
//
// As codes: with t = h w and a = max |t| over 128 columns, code = e4m3(t * (448 / a)) and scale = a / 448 * r.
// The row's statistic enters the scale alone, so the codes are ready before the sum of squares is, and do not
// depend on its order of summation.
#include "lowp.cuh"

namespace gnnagg {
namespace {

constexpr int kRowThreads = 256;    // block of the warp-per-row forms: eight rows at a time
constexpr int kBlockThreads = 512;  // largest block of the block-per-row forms
constexpr int kWideThreads = 1024;  // block of rows too wide for these
constexpr int kMaxWidth = 16384;

// Threads of a row: L = 32 or 16 lanes of a warp, or (L = 0) the block.
// Sum over them; every one gets it.  `red` holds a value per warp of up to 32, zero for those that the block lacks
// (clear_sums), and is on 16 bytes.
template <int N>
__device__ __forceinline__ void clear_sums(float (&red)[N][32]) {
    for (int i = threadIdx.x; i < N * 32; i += blockDim.x) red[i / 32][i % 32] = 0.0f;
    __syncthreads();
}
template <int L>
__device__ __forceinline__ float row_sum(float v, float *red) {
#pragma unroll
    for (int off = L == 16 ? 8 : 16; off > 0; off >>= 1) v += __shfl_xor_sync(kFullMask, v, off);
    if (L > 0) return v;
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    const float4 *r = reinterpret_cast<const float4 *>(red);
    float4 s = r[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) {
        if (i >= 4 && blockDim.x <= 512) break;
        const float4 u = r[i];
        s.x += u.x, s.y += u.y, s.z += u.z, s.w += u.w;
    }
    return (s.x + s.y) + (s.z + s.w);
}

// The weights of a thread's pieces (see load_pieces), of the rows' type or fp32.
template <typename T, int P>
__device__ __forceinline__ void load_weight(const void *w, bool w_f32, int first, int step, int F, float (&f)[Vec<T>::N]) {
#pragma unroll
    for (int q = 0; q < Vec<T>::N / P; ++q) {
        const int c = first + q * step;
#pragma unroll
        for (int i = 0; i < P; ++i) f[q * P + i] = 0.0f;
        if (c >= F) continue;
        if (P == Vec<T>::N && !w_f32) {
            unpack16<T>(__ldg(reinterpret_cast<const uint4 *>(static_cast<const T *>(w) + c)), f);
        } else if (P >= 4) {
#pragma unroll
            for (int i = 0; i < P; i += 4) {
                const float4 v = __ldg(reinterpret_cast<const float4 *>(static_cast<const float *>(w) + c + i));
                f[q * P + i] = v.x, f[q * P + i + 1] = v.y, f[q * P + i + 2] = v.z, f[q * P + i + 3] = v.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < P; ++i)
                f[q * P + i] = w_f32 ? __ldg(static_cast<const float *>(w) + c + i) : to_f32(static_cast<const T *>(w)[c + i]);
        }
    }
}

// Where a thread's chunks of a row begin: a warp (half a warp) covers neighbouring columns.
template <typename T, int L, int NV, int P>
struct Columns {
    static constexpr int V = Vec<T>::N, kLanes = L == 16 ? 16 : 32, kStep = P * kLanes;
    int base;
    __device__ __forceinline__ Columns()
        : base((L == 0 ? (int)(threadIdx.x >> 5) * kLanes * V * NV : 0) + (int)(threadIdx.x & (kLanes - 1)) * P) {}
    __device__ __forceinline__ int first(int j) const { return base + j * V * kLanes; }
    // element i of chunk j
    __device__ __forceinline__ int at(int j, int i) const { return first(j) + i / P * kStep + i % P; }
};

struct FwdParams {
    const void *x, *residual, *w;
    void *h, *y;      // y: the stream's type, or codes
    float *scales, *rstd;
    int64_t ldx, ldr, ldh, ldy, lds;
    int64_t rows;
    int F, w_f32;
    float eps;
};

// NV chunks a thread and row, R rows a group of threads at once.
template <typename T, int L, int NV, int R, int P, bool FP8>
__global__ void __launch_bounds__(L > 0 ? kRowThreads : kBlockThreads) rms_norm_fwd_kernel(const FwdParams p) {
    constexpr int V = Vec<T>::N;
    __shared__ __align__(16) float red[1][32];
    if (L == 0) clear_sums(red);
    const Columns<T, L, NV, P> cols;
    constexpr int kStep = cols.kStep;
    const int lane = L > 0 ? threadIdx.x & (L - 1) : threadIdx.x;
    const int64_t row0 = L > 0 ? ((int64_t)blockIdx.x * (kRowThreads / (L + !L)) + threadIdx.x / (L + !L)) * R : blockIdx.x;
    if (L == 32 && row0 >= p.rows) return;  // whole warps; half a warp stays for the other half's exchanges
    uint4 h[R][NV], res[R][NV];
#pragma unroll
    for (int k = 0; k < R; ++k)
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const bool in = (L != 16 && R == 1) || row0 + k < p.rows;
            h[k][j] = res[k][j] = make_uint4(0, 0, 0, 0);
            if (in) h[k][j] = load_pieces<T, P>(static_cast<const T *>(p.x) + (row0 + k) * p.ldx, cols.first(j), kStep, p.F);
            if (in && p.residual != nullptr)
                res[k][j] = load_pieces<T, P>(static_cast<const T *>(p.residual) + (row0 + k) * p.ldr, cols.first(j), kStep, p.F);
        }
#pragma unroll
    for (int k = 0; k < R; ++k) {
        const int64_t row = row0 + k;
        if (L != 16 && R > 1 && row >= p.rows) break;
        const bool live = L != 16 || row < p.rows;
        float ss = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            float v[V];
            unpack16<T>(h[k][j], v);
            if (p.residual != nullptr) {
                float r[V];
                unpack16<T>(res[k][j], r);
#pragma unroll
                for (int i = 0; i < V; ++i) v[i] += r[i];
                h[k][j] = pack16<T>(v);
                unpack16<T>(h[k][j], v);  // the norm is of the rounded sum
                if (live) store_pieces<T, P>(static_cast<T *>(p.h) + row * p.ldh, cols.first(j), kStep, p.F, h[k][j]);
            }
#pragma unroll
            for (int i = 0; i < V; ++i) ss = fmaf(v[i], v[i], ss);
        }
        const float rstd = rsqrtf(row_sum<L>(ss, red[0]) / (float)p.F + p.eps);
        if (lane == 0 && live && p.rstd != nullptr) p.rstd[row] = rstd;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int first = cols.first(j);
            float v[V], w[V];
            unpack16<T>(h[k][j], v);
            load_weight<T, P>(p.w, p.w_f32 != 0, first, kStep, p.F, w);
            if (!FP8) {
#pragma unroll
                for (int i = 0; i < V; ++i) v[i] = v[i] * rstd * w[i];
                if (live) store_pieces<T, P>(static_cast<T *>(p.y) + row * p.ldy, first, kStep, p.F, pack16<T>(v));
                continue;
            }
            uint8_t *codes = static_cast<uint8_t *>(p.y) + row * p.ldy;
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = __fmul_rn(v[i], w[i]);
            if (P == V) {
                // 128 columns are 128 / V neighbouring threads: a whole or half a warp (or all of the row)
                uint32_t m = 0;
#pragma unroll
                for (int i = 0; i < V; ++i) m = max(m, abs_bits(v[i]));
#pragma unroll
                for (int off = L == 16 ? 8 : 64 / V; off > 0; off >>= 1) m = max(m, __shfl_xor_sync(kFullMask, m, off));
                const float a = block_amax(m), f = block_factor(a);
                if (first < p.F && live) {
                    uint32_t c[V / 4];
#pragma unroll
                    for (int i = 0; i < V / 4; ++i)
                        c[i] = e4m3x4(v[4 * i] * f, v[4 * i + 1] * f, v[4 * i + 2] * f, v[4 * i + 3] * f);
                    uint32_t *dst = reinterpret_cast<uint32_t *>(codes + first);
                    if (V == 8)
                        __stcs(reinterpret_cast<uint2 *>(dst), make_uint2(c[0], c[V / 4 - 1]));
                    else
                        __stcs(dst, c[0]);
                    if ((first & 127) == 0) p.scales[(int64_t)(first >> 7) * p.lds + row] = block_scale(a) * rstd;
                }
            } else {
                // 128 columns are E elements of every lane
                constexpr int E = V * cols.kLanes >= 128 ? 128 / cols.kLanes : V;
#pragma unroll
                for (int e = 0; e < V; e += E) {
                    uint32_t m = 0;
#pragma unroll
                    for (int i = e; i < e + E; ++i) m = max(m, abs_bits(v[i]));
#pragma unroll
                    for (int off = cols.kLanes / 2; off > 0; off >>= 1) m = max(m, __shfl_xor_sync(kFullMask, m, off));
                    const float a = block_amax(m), f = block_factor(a);
#pragma unroll
                    for (int i = e; i < e + E; i += P) {
                        const int c = cols.at(j, i);
                        if (c < p.F && live) {
                            const uint32_t b = e4m3x4(v[i] * f, v[i + P - 1] * f, 0.0f, 0.0f);
                            if (P == 2)
                                *reinterpret_cast<uint16_t *>(codes + c) = (uint16_t)b;
                            else
                                codes[c] = (uint8_t)b;
                        }
                    }
                    const int c0 = cols.at(j, e);
                    if ((c0 & 127) == 0 && c0 < p.F && live) p.scales[(int64_t)(c0 >> 7) * p.lds + row] = block_scale(a) * rstd;
                }
            }
        }
    }
}

struct BwdParams {
    const void *gy, *gh, *h, *w;
    const float *rstd;
    void *gx;
    float *partial;   // [blocks][F]
    int64_t ldgy, ldgh, ldh, ldgx;
    int64_t rows;
    int F, w_f32;
};

// Blocks per SM that the register limit is set for, as measured: more rows on their way against registers that spill.
template <typename T, int L, int NV, int P>
__global__ void __launch_bounds__(L > 0 ? kRowThreads : kBlockThreads, L > 0 ? (NV == 1 ? 4 : NV == 2 ? 3 : 2) : NV == 4 ? 1 : 2)
rms_norm_bwd_kernel(const BwdParams p) {
    constexpr int V = Vec<T>::N;
    constexpr int kRows = L > 0 ? kRowThreads / (L + !L) : 1, kWarpRows = L == 16 ? 2 : 1;
    __shared__ __align__(16) float red[2][32];
    __shared__ float sums[L > 0 ? kRowThreads * V : 1];
    const Columns<T, L, NV, P> cols;
    constexpr int kStep = cols.kStep;
    const int lane = L > 0 ? threadIdx.x & (L - 1) : threadIdx.x;
    const int slot = L > 0 ? threadIdx.x / (L + !L) : 0;
    if (L == 0) clear_sums(red);
    const float inv_f = 1.0f / (float)p.F;
    float dw[NV][V];
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) dw[j][i] = 0.0f;
    int turn = 0;
    // a warp's rows go round together: its halves meet in the exchanges
    for (int64_t base = (int64_t)blockIdx.x * kRows + slot / kWarpRows * kWarpRows; base < p.rows;
         base += (int64_t)gridDim.x * kRows, turn ^= 1) {
        const int64_t row = base + slot % kWarpRows;
        const bool live = L != 16 || row < p.rows;
        uint4 h[NV], g[NV], gh[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            h[j] = g[j] = gh[j] = make_uint4(0, 0, 0, 0);
            if (live) {
                const int first = cols.first(j);
                h[j] = load_pieces<T, P>(static_cast<const T *>(p.h) + row * p.ldh, first, kStep, p.F);
                g[j] = load_pieces<T, P>(static_cast<const T *>(p.gy) + row * p.ldgy, first, kStep, p.F);
                if (p.gh != nullptr) gh[j] = load_pieces<T, P>(static_cast<const T *>(p.gh) + row * p.ldgh, first, kStep, p.F);
            }
        }
        const float rstd = live ? __ldg(p.rstd + row) : 0.0f;
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            float x[V], y[V], w[V];
            unpack16<T>(h[j], x);
            unpack16<T>(g[j], y);
            load_weight<T, P>(p.w, p.w_f32 != 0, cols.first(j), kStep, p.F, w);  // from L1: cheaper than its registers
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float hat = x[i] * rstd;
                dw[j][i] = fmaf(y[i], hat, dw[j][i]);
                s = fmaf(y[i] * w[i], hat, s);
            }
        }
        const float minus = -rstd * row_sum<L>(s, red[turn]) * inv_f;  // two buffers: a warp may be a row ahead of another
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            float x[V], y[V], w[V], o[V];
            unpack16<T>(h[j], x);
            unpack16<T>(g[j], y);
            unpack16<T>(gh[j], o);
            load_weight<T, P>(p.w, p.w_f32 != 0, cols.first(j), kStep, p.F, w);
#pragma unroll
            for (int i = 0; i < V; ++i) o[i] = fmaf(rstd, fmaf(x[i], minus, y[i] * w[i]), o[i]);
            if (live) store_pieces<T, P>(static_cast<T *>(p.gx) + row * p.ldgx, cols.first(j), kStep, p.F, pack16<T>(o));
        }
    }
    float *out = p.partial + (int64_t)blockIdx.x * p.F;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        if (L > 0) {  // the block's rows add up in their order
            __syncthreads();
#pragma unroll
            for (int i = 0; i < V; ++i) sums[(slot * V + i) * L + lane] = dw[j][i];
            __syncthreads();
            for (int e = threadIdx.x; e < L * V; e += kRowThreads) {
                float s = 0.0f;
#pragma unroll
                for (int r = 0; r < kRows; ++r) s += sums[r * L * V + e];
                const int i = e / (L + !L), c = (e % (L + !L)) * P + j * V * L + i / P * kStep + i % P;
                if (c < p.F) out[c] = s;
            }
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (cols.at(j, i) < p.F) out[cols.at(j, i)] = dw[j][i];
        }
    }
}

// The block-per-row form on 16-byte rows: the next row's chunks are copied to shared memory (cp.async, every thread its
// own, so that no barrier is needed for them) while the block works on this one.  Without, a block's three loads, its
// reduction and its store follow one another: 16384 x 4096 bf16 in 116 us instead of 104 (109 with cold caches).
template <typename T, int NV>
__global__ void __launch_bounds__(kBlockThreads) rms_norm_bwd_ahead_kernel(const BwdParams p) {
    constexpr int V = Vec<T>::N;
    extern __shared__ __align__(16) uint4 ahead[];  // [2][3 * NV][threads]
    __shared__ __align__(16) float red[2][32];
    const int tid = threadIdx.x, step = blockDim.x;
    clear_sums(red);
    const float inv_f = 1.0f / (float)p.F;
    auto slot = [&](int turn, int k) -> uint4 * { return ahead + (turn * 3 * NV + k) * step + tid; };
    auto fetch = [&](int64_t row, int turn) {
        if (row < p.rows) {
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int col = (tid + step * j) * V;
                if (col < p.F) {
                    cp_async_16(slot(turn, 3 * j), static_cast<const T *>(p.h) + row * p.ldh + col);
                    cp_async_16(slot(turn, 3 * j + 1), static_cast<const T *>(p.gy) + row * p.ldgy + col);
                    if (p.gh != nullptr) cp_async_16(slot(turn, 3 * j + 2), static_cast<const T *>(p.gh) + row * p.ldgh + col);
                }
            }
        }
        cp_async_commit();
    };
    float dw[NV][V];
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) dw[j][i] = 0.0f;
    fetch(blockIdx.x, 0);
    float next = __ldg(p.rstd + blockIdx.x);  // there are no more blocks than rows
    int turn = 0;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
        const float rstd = next;
        if (row + gridDim.x < p.rows) next = __ldg(p.rstd + row + gridDim.x);
        fetch(row + gridDim.x, turn ^ 1);
        cp_async_wait<1>();
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int col = (tid + step * j) * V;
            if (col < p.F) {
                float x[V], y[V], w[V];
                unpack16<T>(*slot(turn, 3 * j), x);
                unpack16<T>(*slot(turn, 3 * j + 1), y);
                load_weight<T, V>(p.w, p.w_f32 != 0, col, V, p.F, w);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float hat = x[i] * rstd;
                    dw[j][i] = fmaf(y[i], hat, dw[j][i]);
                    s = fmaf(y[i] * w[i], hat, s);
                }
            }
        }
        const float minus = -rstd * row_sum<0>(s, red[turn]) * inv_f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int col = (tid + step * j) * V;
            if (col < p.F) {
                float x[V], y[V], w[V], o[V];
                unpack16<T>(*slot(turn, 3 * j), x);
                unpack16<T>(*slot(turn, 3 * j + 1), y);
#pragma unroll
                for (int i = 0; i < V; ++i) o[i] = 0.0f;
                if (p.gh != nullptr) unpack16<T>(*slot(turn, 3 * j + 2), o);
                load_weight<T, V>(p.w, p.w_f32 != 0, col, V, p.F, w);
#pragma unroll
                for (int i = 0; i < V; ++i) o[i] = fmaf(rstd, fmaf(x[i], minus, y[i] * w[i]), o[i]);
                store_chunk<T, true>(static_cast<T *>(p.gx) + row * p.ldgx + col, V, o);
            }
        }
    }
    cp_async_wait<0>();
    float *out = p.partial + (int64_t)blockIdx.x * p.F;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int col = (tid + step * j) * V;
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (col + i < p.F) out[col + i] = dw[j][i];
    }
}

// Rows too wide for the registers of a block: two sweeps over the row (the second finds it in L1 / L2), and the
// column sums of dw in shared memory, where every thread adds to columns of its own.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kWideThreads) rms_norm_bwd_wide_kernel(const BwdParams p) {
    constexpr int V = Vec<T>::N;
    extern __shared__ float dw[];  // [V][chunks]
    __shared__ __align__(16) float red[2][32];
    const int chunks = (p.F + V - 1) / V;
    const float inv_f = 1.0f / (float)p.F;
    for (int i = threadIdx.x; i < chunks * V; i += kWideThreads) dw[i] = 0.0f;
    clear_sums(red);
    int turn = 0;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
        const float rstd = __ldg(p.rstd + row);
        const T *h = static_cast<const T *>(p.h) + row * p.ldh, *gy = static_cast<const T *>(p.gy) + row * p.ldgy;
        float s = 0.0f;
        for (int k = threadIdx.x; k < chunks; k += kWideThreads) {
            const int col = k * V, valid = p.F - col;
            float hat[V], g[V], w[V];
            load_chunk<T, VEC>(h + col, valid, hat);
            load_chunk<T, VEC>(gy + col, valid, g);
            load_weight<T, VEC ? V : 1>(p.w, p.w_f32 != 0, col, 1, p.F, w);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                hat[i] *= rstd;
                dw[i * chunks + k] = fmaf(g[i], hat[i], dw[i * chunks + k]);
                s = fmaf(g[i] * w[i], hat[i], s);
            }
        }
        const float minus = -rstd * row_sum<0>(s, red[turn]) * inv_f;
        for (int k = threadIdx.x; k < chunks; k += kWideThreads) {
            const int col = k * V, valid = p.F - col;
            float hat[V], g[V], w[V], gh[V];
            load_chunk<T, VEC>(h + col, valid, hat);
            load_chunk<T, VEC>(gy + col, valid, g);
            load_weight<T, VEC ? V : 1>(p.w, p.w_f32 != 0, col, 1, p.F, w);
#pragma unroll
            for (int i = 0; i < V; ++i) gh[i] = 0.0f;
            if (p.gh != nullptr) load_chunk<T, VEC>(static_cast<const T *>(p.gh) + row * p.ldgh + col, valid, gh);
#pragma unroll
            for (int i = 0; i < V; ++i) gh[i] = fmaf(rstd, fmaf(hat[i], minus, g[i] * w[i]), gh[i]);
            store_chunk<T, VEC>(static_cast<T *>(p.gx) + row * p.ldgx + col, valid, gh);
        }
    }
    float *out = p.partial + (int64_t)blockIdx.x * p.F;
    for (int k = threadIdx.x; k < chunks; k += kWideThreads)
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (k * V + i < p.F) out[k * V + i] = dw[i * chunks + k];
}

// How a row of F elements of `size` bytes is spread: over half a warp, a warp (lanes = 16, 32) or a block (lanes = 0) of
// `threads`, with nv 16-byte chunks a thread; nv = 0: too wide for registers.
struct Spread {
    int lanes, threads, nv;
};
Spread spread_of(int F, int size) {
    const int chunks = (int)div_up(F, 16 / size);
    if (chunks <= 16) return {16, kRowThreads, 1};
    if (chunks <= 128) return {32, kRowThreads, chunks <= 32 ? 1 : chunks <= 64 ? 2 : 4};
    const int nv = chunks <= 256 ? 1 : chunks <= 2 * kBlockThreads ? 2 : 4;
    if (chunks > 4 * kBlockThreads) return {0, kWideThreads, 0};
    return {0, (int)div_up(div_up(chunks, nv), 32) * 32, nv};
}

// Most blocks a backward launch has: the partial sums' rows.
constexpr int kMostPerSm = 6;
int bwd_blocks(int64_t rows, int F, int size) {
    const Spread s = spread_of(F, size);
    const int64_t need = div_up(rows, s.lanes > 0 ? kRowThreads / s.lanes : 1);
    const int64_t cap = (int64_t)kNumSMs * (s.nv == 0 ? 2 : kMostPerSm);
    return (int)(need < cap ? need : cap);
}

// Blocks of `threads` threads (and of their shared memory) that an SM holds of KERNEL: a persistent grid is one full wave (with a block too many or
// too few per SM the backward takes up to a third longer).
template <auto KERNEL>
int resident(int threads, size_t smem = 0) {
    static int known[PerDeviceOnce::kMaxDevices][kWideThreads / 32 + 1];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= PerDeviceOnce::kMaxDevices) return 1;
    int n = __atomic_load_n(&known[dev][threads / 32], __ATOMIC_RELAXED);
    if (n == 0) {
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, KERNEL, threads, smem) != cudaSuccess || n < 1) n = 1;
        __atomic_store_n(&known[dev][threads / 32], n, __ATOMIC_RELAXED);
    }
    return n < kMostPerSm ? n : kMostPerSm;
}

template <typename F32, typename BF16, typename F16>
int by_type(int type, F32 a, BF16 b, F16 c) {
    return type == kTypeF32 ? a() : type == kTypeBf16 ? b() : c();
}

template <typename T, int P, bool FP8>
int launch_fwd(const FwdParams &p, cudaStream_t st) {
    const Spread s = spread_of(p.F, (int)sizeof(T));
#define RMS_WARP(L, NV, R) \
    rms_norm_fwd_kernel<T, L, NV, R, P, FP8><<<(unsigned)div_up(p.rows, kRowThreads / L * R), kRowThreads, 0, st>>>(p)
#define RMS_BLOCK(NV, THREADS) rms_norm_fwd_kernel<T, 0, NV, 1, P, FP8><<<(unsigned)p.rows, THREADS, 0, st>>>(p)
    if (s.lanes == 16) RMS_WARP(16, 1, 2);
    else if (s.lanes == 32 && s.nv == 1) RMS_WARP(32, 1, 2);
    else if (s.lanes == 32 && s.nv == 2) RMS_WARP(32, 2, 1);
    else if (s.lanes == 32) RMS_WARP(32, 4, 1);
    else if (s.nv == 1) RMS_BLOCK(1, s.threads);
    else if (s.nv == 2) RMS_BLOCK(2, s.threads);
    else if (s.nv == 4) RMS_BLOCK(4, s.threads);
    else RMS_BLOCK(8, kBlockThreads);  // fp32 rows above 8192 columns
#undef RMS_WARP
#undef RMS_BLOCK
    return check_launch("rms_norm_fwd_kernel");
}

// `blocks`: at most this many; becomes the number of blocks (rows of partial sums).
template <typename T, int P>
int launch_bwd(const BwdParams &p, int &blocks, cudaStream_t st) {
    constexpr bool VEC = P == Vec<T>::N;
    const Spread s = spread_of(p.F, (int)sizeof(T));
#define RMS_LAUNCH(L, NV)                                                                    \
    do {                                                                                     \
        const int wave = kNumSMs * resident<rms_norm_bwd_kernel<T, L, NV, P>>(s.threads);  \
        if (blocks > wave) blocks = wave;                                                    \
        rms_norm_bwd_kernel<T, L, NV, P><<<blocks, s.threads, 0, st>>>(p);                 \
    } while (0)
#define RMS_AHEAD(NV)                                                                                            \
    do {                                                                                                         \
        static PerDeviceOnce attr_done;                                                                          \
        const size_t smem = (size_t)2 * 3 * NV * s.threads * 16;                                                 \
        const cudaError_t e = attr_done.run([] {                                                                 \
            return cudaFuncSetAttribute(rms_norm_bwd_ahead_kernel<T, NV>,                                        \
                                        cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * 3 * NV * kBlockThreads * 16); \
        });                                                                                                      \
        if (e != cudaSuccess) return fail(GNNAGG_ERR_CUDA, "rms_norm_bwd: %s", cudaGetErrorString(e));           \
        const int wave = kNumSMs * resident<rms_norm_bwd_ahead_kernel<T, NV>>(s.threads, smem);                  \
        if (blocks > wave) blocks = wave;                                                                        \
        rms_norm_bwd_ahead_kernel<T, NV><<<blocks, s.threads, smem, st>>>(p);                                    \
    } while (0)
    if (VEC && s.lanes == 0 && s.nv == 1) RMS_AHEAD(1);
    else if (VEC && s.lanes == 0 && s.nv == 2) RMS_AHEAD(2);
    else if (VEC && s.lanes == 0 && s.nv == 4) RMS_AHEAD(4);
    else if (s.lanes == 16) RMS_LAUNCH(16, 1);
    else if (s.lanes == 32 && s.nv == 1) RMS_LAUNCH(32, 1);
    else if (s.lanes == 32 && s.nv == 2) RMS_LAUNCH(32, 2);
    else if (s.lanes == 32) RMS_LAUNCH(32, 4);
    else if (s.nv == 1) RMS_LAUNCH(0, 1);  // rows off 16 bytes
    else if (s.nv == 2) RMS_LAUNCH(0, 2);
    else if (s.nv == 4) RMS_LAUNCH(0, 4);
    else {
        static PerDeviceOnce attr_done;
        const cudaError_t e = attr_done.run([] {
            return cudaFuncSetAttribute(rms_norm_bwd_wide_kernel<T, VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        kMaxWidth * (int)sizeof(float));
        });
        if (e != cudaSuccess) return fail(GNNAGG_ERR_CUDA, "rms_norm_bwd: %s", cudaGetErrorString(e));
        const size_t smem = (size_t)div_up(p.F, Vec<T>::N) * Vec<T>::N * sizeof(float);
        rms_norm_bwd_wide_kernel<T, VEC><<<blocks, kWideThreads, smem, st>>>(p);
    }
#undef RMS_LAUNCH
#undef RMS_AHEAD
    return check_launch("rms_norm_bwd_kernel");
}

template <typename T>
int launch_dw(const float *partial, int blocks, int F, void *dw, cudaStream_t st) {
    column_sum_kernel<T><<<(unsigned)div_up(F, 32), dim3(32, 16), 0, st>>>(partial, blocks, F, static_cast<T *>(dw));
    return check_launch("column_sum_kernel");
}

// How many neighbouring elements all of a call's rows allow one access for.
struct Together {
    int F, size;
    uintptr_t bits = 0;  // of the addresses and strides in bytes, scaled to the rows' element size
    Together(int F, int size) : F(F), size(size) {}
    void add(const void *p, int64_t ld, int each) {
        bits |= reinterpret_cast<uintptr_t>(p) * size / each | (uintptr_t)(ld * size);
    }
    bool allow(int n) const { return F % n == 0 && bits % (uintptr_t)(n * size) == 0; }
};

int check_common(const char *what, int type, int w_type, int64_t rows, int F) {
    if (type_size(type) == 0) return fail(GNNAGG_ERR_ARG, "%s: unknown element type %d", what, type);
    if (w_type != kTypeF32 && w_type != type)
        return fail(GNNAGG_ERR_ARG, "%s: the weight is fp32 or of the rows' type", what);
    if (rows < 0 || F <= 0) return fail(GNNAGG_ERR_ARG, "%s: negative or zero size", what);
    if (F > kMaxWidth || rows > 0x7FFFFFFF)
        return fail(GNNAGG_ERR_UNSUPPORTED, "%s: at most %d columns and 2^31 - 1 rows", what, kMaxWidth);
    return GNNAGG_OK;
}

int fwd(const char *what, bool fp8, const void *x, int64_t ldx, const void *residual, int64_t ldr, const void *w,
        int w_type, int64_t rows, int F, int type, float eps, void *h, int64_t ldh, void *y, int64_t ldy, float *scales,
        int64_t lds, float *rstd, void *stream) {
    int rc = check_common(what, type, w_type, rows, F);
    if (rc != GNNAGG_OK) return rc;
    if (rows == 0) return GNNAGG_OK;
    if (x == nullptr || w == nullptr || y == nullptr || (fp8 && scales == nullptr))
        return fail(GNNAGG_ERR_ARG, "%s: null pointer", what);
    if ((residual == nullptr) != (h == nullptr))
        return fail(GNNAGG_ERR_ARG, "%s: the residual and the sum's output come together", what);
    if (ldx < F || ldy < F || (residual != nullptr && (ldr < F || ldh < F)) || (fp8 && lds < rows))
        return fail(GNNAGG_ERR_ARG, "%s: a stride is smaller than its rows", what);
    if (fp8 && (!aligned16(y) || ldy % 16 != 0))
        return fail(GNNAGG_ERR_UNSUPPORTED, "%s: code rows start on 16 bytes", what);
    const int size = type_size(type);
    Together rows_of(F, size);
    rows_of.add(x, ldx, size);
    rows_of.add(w, 0, w_type == kTypeF32 ? 4 : size);
    if (!fp8) rows_of.add(y, ldy, size);
    if (residual != nullptr) {
        rows_of.add(residual, ldr, size);
        rows_of.add(h, ldh, size);
    }
    const bool vec = rows_of.allow(16 / size), two = size == 2 && rows_of.allow(2);
    const FwdParams p{x, residual, w, h, y, scales, rstd, ldx, ldr, ldh, ldy, lds, rows, F, w_type == kTypeF32, eps};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
#define RMS_TYPE(T)                                                                                        \
    [&] {                                                                                                  \
        constexpr int V = Vec<T>::N, Two = sizeof(T) == 2 ? 2 : 1;                                         \
        return fp8 ? (vec ? launch_fwd<T, V, true>(p, st) : two ? launch_fwd<T, Two, true>(p, st)          \
                                                                : launch_fwd<T, 1, true>(p, st))           \
                   : (vec ? launch_fwd<T, V, false>(p, st) : two ? launch_fwd<T, Two, false>(p, st)        \
                                                                 : launch_fwd<T, 1, false>(p, st));        \
    }
    return by_type(type, RMS_TYPE(float), RMS_TYPE(__nv_bfloat16), RMS_TYPE(__half));
#undef RMS_TYPE
}

}  // namespace
}  // namespace gnnagg

using namespace gnnagg;

extern "C" int gnnagg_rms_norm_fwd(const void *x, int64_t ldx, const void *residual, int64_t ldr, const void *w,
                                   int32_t w_type, int64_t rows, int32_t F, int32_t type, float eps, void *h,
                                   int64_t ldh, void *y, int64_t ldy, float *rstd, void *stream) {
    return fwd("rms_norm_fwd", false, x, ldx, residual, ldr, w, w_type, rows, F, type, eps, h, ldh, y, ldy, nullptr, 0,
               rstd, stream);
}

extern "C" int gnnagg_rms_norm_fp8(const void *x, int64_t ldx, const void *residual, int64_t ldr, const void *w,
                                   int32_t w_type, int64_t rows, int32_t F, int32_t type, float eps, void *h,
                                   int64_t ldh, uint8_t *codes, int64_t ldc, float *scales, int64_t lds, void *stream) {
    return fwd("rms_norm_fp8", true, x, ldx, residual, ldr, w, w_type, rows, F, type, eps, h, ldh, codes, ldc, scales,
               lds, nullptr, stream);
}

extern "C" size_t gnnagg_rms_norm_partial_bytes(int64_t rows, int32_t F, int32_t type) {
    if (type_size(type) == 0 || rows < 0 || F <= 0 || F > kMaxWidth) return 0;
    return (size_t)bwd_blocks(rows, F, type_size(type)) * (size_t)F * sizeof(float);
}

extern "C" int gnnagg_rms_norm_bwd(const void *gy, int64_t ldgy, const void *gh, int64_t ldgh, const void *h, int64_t ldh,
                                   const float *rstd, const void *w, int32_t w_type, int64_t rows, int32_t F,
                                   int32_t type, void *gx, int64_t ldgx, void *dw, float *partial, size_t partial_bytes,
                                   void *stream) {
    int rc = check_common("rms_norm_bwd", type, w_type, rows, F);
    if (rc != GNNAGG_OK) return rc;
    if (dw == nullptr || w == nullptr || (rows > 0 && (gy == nullptr || h == nullptr || rstd == nullptr || gx == nullptr ||
                                                       partial == nullptr)))
        return fail(GNNAGG_ERR_ARG, "rms_norm_bwd: null pointer");
    if (rows > 0 && (ldgy < F || ldh < F || ldgx < F || (gh != nullptr && ldgh < F)))
        return fail(GNNAGG_ERR_ARG, "rms_norm_bwd: a stride is smaller than its rows");
    const int size = type_size(type);
    int blocks = bwd_blocks(rows, F, size);
    if (partial_bytes < gnnagg_rms_norm_partial_bytes(rows, F, type))
        return fail(GNNAGG_ERR_SCRATCH, "rms_norm_bwd: partial-sum scratch too small");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (rows > 0) {
        Together rows_of(F, size);
        rows_of.add(gy, ldgy, size);
        rows_of.add(h, ldh, size);
        rows_of.add(gx, ldgx, size);
        if (gh != nullptr) rows_of.add(gh, ldgh, size);
        rows_of.add(w, 0, w_type == kTypeF32 ? 4 : size);
        const bool vec = rows_of.allow(16 / size), two = size == 2 && rows_of.allow(2);
        const BwdParams p{gy, gh, h, w, rstd, gx, partial, ldgy, ldgh, ldh, ldgx, rows, F, w_type == kTypeF32};
#define RMS_TYPE(T)                                                                                  \
    [&] {                                                                                            \
        return vec   ? launch_bwd<T, Vec<T>::N>(p, blocks, st)                                       \
               : two ? launch_bwd<T, sizeof(T) == 2 ? 2 : 1>(p, blocks, st)                          \
                     : launch_bwd<T, 1>(p, blocks, st);                                              \
    }
        rc = by_type(type, RMS_TYPE(float), RMS_TYPE(__nv_bfloat16), RMS_TYPE(__half));
#undef RMS_TYPE
        if (rc != GNNAGG_OK) return rc;
    }
    return by_type(w_type, [&] { return launch_dw<float>(partial, blocks, F, dw, st); },
                   [&] { return launch_dw<__nv_bfloat16>(partial, blocks, F, dw, st); },
                   [&] { return launch_dw<__half>(partial, blocks, F, dw, st); });
}
