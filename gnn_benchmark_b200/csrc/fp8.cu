// Matrix product of e4m3 operands with a scale for each block of 128 along the sum, on the tensor cores (tcgen05 +
// TMEM + TMA), sm_100a:
//
//     C[m,n] = sum_kb  sa[m,kb] * sb[n,kb] * ( sum_{k in block kb} A[m,k] B[n,k] )   (+ bias[n]) (+ C[m,n])
//
// Scales are fp32, one per row or one per 128 rows of either operand.  The inner sum of a block is a chain of four
// MMAs into tensor memory; the outer one is taken in registers, one packed FMA per element and block, rounded to
// nearest.  Tensor memory holds several blocks' partial products, so the MMAs of the next block run under the FMAs
// of the last.
//
// One operand lies along the 128 lanes of tensor memory (P), the other along its columns (Q).  P is A and Q is B,
// except for few rows of A (SWAP): then the weight's rows fill the lanes and the few rows are the columns.
//
// One persistent CTA per SM, three warpgroups:
//   warp 0      lane 0 issues the TMA loads (a 128-byte wide k-block of both operands per stage);
//   warp 1      allocates tensor memory; lane 0 issues tcgen05.mma (kind::f8f6f4, 128 x BN x 32) and the commits;
//   warps 2-3   idle; their registers go to
//   warps 4-11  which read a block's product, scale and add it; after the last block, convert and store.  Warp w
//               reads lane quarter w % 4 and one half of the columns.
// A tile's sum may be split along k over several CTAs (few tiles, long sums): each writes an fp32 partial product
// to the workspace and a second kernel adds them in a fixed order.
// Every wait is bounded (about a second); on a time-out the kernel records a code in the library's status word,
// drains its own copies and MMAs, frees tensor memory and returns.
#include "lowp.cuh"
#include "tc.cuh"

namespace gnnagg {
namespace {

constexpr int BP = 128;                        // rows of P per tile = TMEM lanes
constexpr int BK = 128;                        // bytes = elements per k-block = one scale block = one swizzle row
constexpr int UMMA_K = 32;                     // elements per tcgen05.mma
constexpr int kThreads = 384;
// Registers per thread: 168 at launch (64,512 in all), then 56 for the first warpgroup and 216 for the other two
// (7,168 + 55,296).
constexpr int kRegsControl = 56, kRegsScaling = 216;
static_assert(128 * kRegsControl + 256 * kRegsScaling <= 168 * kThreads, "register split");
constexpr int kWarpsOut = 8;
constexpr int kTmemCols = 512;
constexpr int P_BYTES = BP * BK;
constexpr int kRowSpan = 128;                  // bytes of an output row that a warp stages at once
constexpr int kStaging = 32 * kRowSpan;        // per warp: the output of 32 rows, or two blocks' column scales
constexpr int kSmemLimit = 227 * 1024;

template <int BN>
struct Tile {
    static constexpr int kStageBytes = P_BYTES + BN * BK;
    static constexpr int kFit = (kSmemLimit - 1024 - 256 - kWarpsOut * kStaging) / kStageBytes;
    static constexpr int kStages = kFit > 10 ? 10 : kFit;
    static constexpr int kBufs = kTmemCols / BN > 4 ? 4 : kTmemCols / BN;  // partial products in tensor memory
    static constexpr int kCols = BN / 2;                                   // columns of a warp
    static constexpr int kSmem = 1024 + kStages * kStageBytes + kWarpsOut * kStaging + 256;
    static_assert(kSmem <= kSmemLimit && (2 * kStages + 2 * kBufs + 1) * 8 + 8 <= 256, "shared memory budget");
};

enum : int {
    kErrWaitEmpty = 1,    // TMA issuer waited for a free stage
    kErrWaitFull = 2,     // MMA issuer waited for a TMA load
    kErrWaitAccFree = 4,  // MMA issuer waited for a partial product to be read
    kErrWaitAccFull = 5,  // scaling warps waited for a partial product
    kErrDrain = 6,        // bounded drain after an abort ran out
};

// The code of the first wait that ran out on this device, 0 if none; sticky.
__device__ int g_status;

// fp32 scales of one operand: element (row or row block, k-block) at p[i * stride + kb * stride_k].
struct Scales {
    const float *p;
    int64_t stride, stride_k;
};

struct Params {
    void *C;             // output, or the workspace's partial products
    const float *bias;
    Scales sp, sq;
    int64_t rows_p, rows_q, ldc, split_stride;
    int p_block;         // P's scales are per 128 rows
    int kblocks, splits, kb_per_split;
    int tiles_p, tiles_q, items;
    int accumulate;
    int vec_out;         // 16-byte stores of the output's rows
    unsigned long long wait_ns;
    uint32_t tx_excess;
};

__device__ __forceinline__ void tc_mma_f8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                          uint32_t accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n"
        "}\n" ::"r"(tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// Instruction descriptor of kind::f8f6f4: fp32 accumulator, e4m3 A and B (format 0), both K-major, M = 128.
__host__ __device__ constexpr uint32_t f8_instr_desc(int n) {
    return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(BP >> 4) << 24);
}

// Two fp32 values in one 64-bit register pair.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
    return d;
}
__device__ __forceinline__ float2 unpair(uint64_t d) {
    float2 v;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(d));
    return v;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// A work item: one tile of the output and a range of its k-blocks.
struct Item {
    int tp, tq, split, kb0, kb1;
};
// Tiles of one column strip of 16 P-tiles are neighbours, so that concurrent CTAs share operand panels in L2.
__device__ __forceinline__ Item item_of(const Params &p, int i) {
    Item w;
    w.split = i % p.splits;
    const int t = i / p.splits;
    constexpr int kGroup = 16;
    const int per = kGroup * p.tiles_q, g = t / per, r = t - g * per;
    const int high = min(kGroup, p.tiles_p - g * kGroup);
    w.tq = r / high;
    w.tp = g * kGroup + (r - w.tq * high);
    w.kb0 = w.split * p.kb_per_split;
    w.kb1 = min(p.kblocks, w.kb0 + p.kb_per_split);
    return w;
}

// BN columns per tile; QROW: Q's scales are per row (per column of the tile); SWAP: the output is stored
// transposed, C[column][lane].
template <int BN, bool QROW, bool SWAP, typename TOut>
__global__ void __launch_bounds__(kThreads, 1)
fp8_matmul_kernel(const __grid_constant__ CUtensorMap map_p, const __grid_constant__ CUtensorMap map_q, const Params p) {
    using S = Tile<BN>;
    constexpr int kStages = S::kStages, kBufs = S::kBufs, kCols = S::kCols;
    extern __shared__ uint8_t smem_raw[];
    // 1024-byte alignment: the swizzle pattern and the descriptors assume it
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t *staging = smem + kStages * S::kStageBytes;
    uint64_t *bars = reinterpret_cast<uint64_t *>(staging + kWarpsOut * kStaging);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 2 * kStages + 2 * kBufs + 1);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const uint32_t bar0 = smem_u32(bars);
    auto bar_full = [&](int s) { return bar0 + 8u * (uint32_t)s; };
    auto bar_empty = [&](int s) { return bar0 + 8u * (uint32_t)(kStages + s); };
    auto bar_acc_full = [&](int b) { return bar0 + 8u * (uint32_t)(2 * kStages + b); };
    auto bar_acc_empty = [&](int b) { return bar0 + 8u * (uint32_t)(2 * kStages + kBufs + b); };
    const uint32_t bar_drain = bar0 + 8u * (uint32_t)(2 * kStages + 2 * kBufs);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(bar_full(s), 1);
            mbar_init(bar_empty(s), 1);
        }
        for (int b = 0; b < kBufs; ++b) {
            mbar_init(bar_acc_full(b), 1);
            mbar_init(bar_acc_empty(b), 32 * kWarpsOut);
        }
        mbar_init(bar_drain, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"((uint32_t)kTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsControl));
    if (warp == 0) {
        // ---------------- TMA issuer ----------------
        if (lane == 0) {
            uint32_t it = 0;
            bool ok = true;
            for (int i = blockIdx.x; i < p.items && ok; i += gridDim.x) {
                const Item w = item_of(p, i);
                for (int kb = w.kb0; kb < w.kb1; ++kb, ++it) {
                    const int s = it % kStages;
                    if (!mbar_wait(bar_empty(s), ((it / kStages) & 1u) ^ 1u, abort_flag, &g_status, kErrWaitEmpty,
                                   p.wait_ns)) {
                        ok = false;
                        break;
                    }
                    const uint32_t sp = smem_u32(smem + s * S::kStageBytes);
                    mbar_arrive_expect_tx(bar_full(s), (uint32_t)S::kStageBytes + p.tx_excess);
                    tma_load_2d(sp, &map_p, bar_full(s), kb * BK, w.tp * BP);
                    tma_load_2d(sp + P_BYTES, &map_q, bar_full(s), kb * BK, w.tq * BN);
                }
            }
            if (!ok) {
                // copies of the last k-blocks issued may still be landing: wait for them, bounded
                for (uint32_t back = 1; back <= (uint32_t)kStages && back <= it; ++back) {
                    const uint32_t j = it - back;
                    const unsigned long long t0 = globaltimer_ns();
                    while (!mbar_try_wait(bar_full(j % kStages), (j / kStages) & 1u)) {
                        if (globaltimer_ns() - t0 > p.wait_ns) {
                            atomicCAS(&g_status, 0, (int)kErrDrain);
                            break;
                        }
                    }
                }
            }
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer ----------------
        if (lane == 0) {
            uint32_t it = 0;
            bool ok = true;
            for (int i = blockIdx.x; i < p.items && ok; i += gridDim.x) {
                const Item w = item_of(p, i);
                for (int kb = w.kb0; kb < w.kb1; ++kb, ++it) {
                    const int s = it % kStages, b = it % kBufs;
                    if (!mbar_wait(bar_acc_empty(b), ((it / kBufs) & 1u) ^ 1u, abort_flag, &g_status, kErrWaitAccFree,
                                   p.wait_ns) ||
                        !mbar_wait(bar_full(s), (it / kStages) & 1u, abort_flag, &g_status, kErrWaitFull, p.wait_ns)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t sp = smem_u32(smem + s * S::kStageBytes);
                    const uint64_t dp = make_smem_desc(sp), dq = make_smem_desc(sp + P_BYTES);
#pragma unroll
                    for (int k = 0; k < BK / UMMA_K; ++k)  // 32 bytes further inside the swizzled row
                        tc_mma_f8(tmem_base + (uint32_t)(b * BN), dp + (uint64_t)(2 * k), dq + (uint64_t)(2 * k),
                                  f8_instr_desc(BN), k > 0 ? 1u : 0u);
                    tc_commit(bar_empty(s));
                    tc_commit(bar_acc_full(b));
                }
            }
            if (!ok) {
                // MMAs already issued still read shared memory and write tensor memory: drain, bounded
                tc_commit(bar_drain);
                const unsigned long long t0 = globaltimer_ns();
                while (!mbar_try_wait(bar_drain, 0)) {
                    if (globaltimer_ns() - t0 > p.wait_ns) {
                        atomicCAS(&g_status, 0, (int)kErrDrain);
                        break;
                    }
                }
            }
        }
    }
    } else {
        // ---------------- scaling warps ----------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsScaling));
        const int q = warp & 3, half = (warp - 4) >> 2;
        uint8_t *mine = staging + (warp - 4) * kStaging;
        constexpr int kChunk = kCols < 32 ? kCols : 32;
        constexpr int kQLoads = (kCols + 31) / 32;
        uint32_t it = 0;
        bool ok = true;
        for (int i = blockIdx.x; i < p.items && ok; i += gridDim.x) {
            const Item w = item_of(p, i);
            const int64_t row = (int64_t)w.tp * BP + q * 32 + lane;              // of P
            const int64_t col0 = (int64_t)w.tq * BN + half * kCols;              // of Q
            const bool row_ok = row < p.rows_p;
            const float *sp = p.sp.p + (p.p_block ? row / 128 : row) * p.sp.stride;
            const float *sq = p.sq.p + (QROW ? col0 + lane : col0 / 128) * p.sq.stride;
            float next_p = 0.0f, next_q[kQLoads] = {};
            auto fetch = [&](int kb) {
                next_p = row_ok ? __ldg(sp + kb * p.sp.stride_k) : 0.0f;
#pragma unroll
                for (int j = 0; j < kQLoads; ++j) {
                    const int64_t c = col0 + (QROW ? 32 * j + lane : 0);
                    next_q[j] = 0.0f;
                    if (c < p.rows_q && (!QROW || 32 * j + lane < kCols) && (QROW || j == 0))
                        next_q[j] = __ldg(sq + (QROW ? 32 * j * p.sq.stride : 0) + kb * p.sq.stride_k);
                }
            };
            uint64_t acc[kCols / 2];
#pragma unroll
            for (int j = 0; j < kCols / 2; ++j) acc[j] = 0;
            if (QROW) __syncwarp();  // the last item's column scales have been read
            if (w.kb0 < w.kb1) fetch(w.kb0);
            for (int kb = w.kb0; kb < w.kb1; ++kb, ++it) {
                const int b = it % kBufs;
                const float scale_p = next_p;
                uint64_t scale = pair(scale_p * next_q[0], scale_p * next_q[0]);
                const float *cols = reinterpret_cast<const float *>(mine) + (kb & 1) * kCols;
                if (QROW) {
                    scale = pair(scale_p, scale_p);
#pragma unroll
                    for (int j = 0; j < kQLoads; ++j)
                        if (32 * j + lane < kCols) const_cast<float *>(cols)[32 * j + lane] = next_q[j];
                    __syncwarp();
                }
                if (kb + 1 < w.kb1) fetch(kb + 1);
                // warp-uniform outcome: the tensor-memory loads below are warp-collective
                if (!__all_sync(kFullMask, mbar_wait(bar_acc_full(b), (it / kBufs) & 1u, abort_flag, &g_status,
                                                     kErrWaitAccFull, p.wait_ns))) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t taddr = tmem_base + (uint32_t)(b * BN + half * kCols) + ((uint32_t)(q * 32) << 16);
#pragma unroll
                for (int c = 0; c < kCols; c += kChunk) {
                    uint32_t r[kChunk];
                    TmemLoad<kChunk>::run(taddr + (uint32_t)c, r);
                    TmemLoad<kChunk>::wait(r);
#pragma unroll
                    for (int j = 0; j < kChunk; j += 2) {
                        const uint64_t v = pair(__uint_as_float(r[j]), __uint_as_float(r[j + 1]));
                        uint64_t f = scale;
                        if (QROW) {
                            const float2 cs = *reinterpret_cast<const float2 *>(cols + c + j);
                            f = mul2(scale, pair(cs.x, cs.y));
                        }
                        acc[(c + j) / 2] = fma2(v, f, acc[(c + j) / 2]);
                    }
                }
                tc_fence_before();
                mbar_arrive(bar_acc_empty(b));
            }
            if (!ok) break;
            TOut *out = static_cast<TOut *>(p.C) + w.split * p.split_stride;
            if (SWAP) {
                // lane = column of the output: 32 neighbouring columns of one output row per store
                const float bias = p.bias != nullptr && row_ok ? __ldg(p.bias + row) : 0.0f;
#pragma unroll
                for (int j = 0; j < kCols / 2; ++j) {
                    const float2 v = unpair(acc[j]);
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int64_t m = col0 + 2 * j + e;
                        if (row_ok && m < p.rows_q) {
                            TOut *dst = out + m * p.ldc + row;
                            float o = (e ? v.y : v.x) + bias;
                            if (p.accumulate) o += to_f32(*dst);
                            *dst = from_f32<TOut>(o);
                        }
                    }
                }
            } else {
                // 128 bytes of each of the warp's 32 rows at a time through shared memory (16-byte piece j of row r
                // sits at piece j ^ (r & 7)), then 8 lanes per row store them
                constexpr int kPiece = 16 / (int)sizeof(TOut);                       // columns per 16 bytes
                constexpr int kSpan = kCols < 8 * kPiece ? kCols : 8 * kPiece;       // columns per turn
                constexpr int kPieces = kSpan / kPiece;
                __syncwarp();
#pragma unroll
                for (int c = 0; c < kCols; c += kSpan) {
#pragma unroll
                    for (int j = 0; j < kPieces; ++j) {
                        float v[kPiece];
#pragma unroll
                        for (int e = 0; e < kPiece; e += 2) {
                            const float2 u = unpair(acc[(c + j * kPiece + e) / 2]);
                            v[e] = u.x, v[e + 1] = u.y;
                        }
                        if (p.bias != nullptr) {
#pragma unroll
                            for (int e = 0; e < kPiece; ++e) {
                                const int64_t n = col0 + c + j * kPiece + e;
                                if (n < p.rows_q) v[e] += __ldg(p.bias + n);
                            }
                        }
                        *reinterpret_cast<uint4 *>(mine + lane * kRowSpan + ((j ^ (lane & 7)) << 4)) = pack16<TOut>(v);
                    }
                    __syncwarp();
#pragma unroll
                    for (int t = 0; t < 8; ++t) {
                        const int r = 4 * t + (lane >> 3), j = lane & 7;
                        const int64_t m = (int64_t)w.tp * BP + q * 32 + r;
                        const int64_t n = col0 + c + j * kPiece;
                        if (j < kPieces && m < p.rows_p && n < p.rows_q) {
                            uint4 u = *reinterpret_cast<const uint4 *>(mine + r * kRowSpan + ((j ^ (r & 7)) << 4));
                            TOut *dst = out + m * p.ldc + n;
                            if (p.vec_out && n + kPiece <= p.rows_q && !p.accumulate) {
                                *reinterpret_cast<uint4 *>(dst) = u;
                            } else {
                                const TOut *e = reinterpret_cast<const TOut *>(&u);
#pragma unroll
                                for (int x = 0; x < kPiece; ++x)
                                    if (n + x < p.rows_q)
                                        dst[x] = p.accumulate ? from_f32<TOut>(to_f32(dst[x]) + to_f32(e[x])) : e[x];
                            }
                        }
                    }
                    __syncwarp();
                }
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((uint32_t)kTmemCols)
                     : "memory");
    }
}

// C[m,n] = sum of the splits' partial products in split order, plus bias, (plus C).  Four columns a thread.
template <typename TOut>
__global__ void __launch_bounds__(256)
fp8_join_kernel(const float *__restrict__ partial, int splits, int64_t split_stride, int64_t ldp, int64_t M, int64_t N,
                const float *__restrict__ bias, int accumulate, TOut *C, int64_t ldc) {
    const int64_t quads = ldp / 4, total = M * quads;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t m = i / quads, n = (i - m * quads) * 4;
        const float *src = partial + m * ldp + n;
        float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
        for (int s = 0; s < splits; ++s) {
            const float4 v = __ldcs(reinterpret_cast<const float4 *>(src + (int64_t)s * split_stride));
            a.x += v.x, a.y += v.y, a.z += v.z, a.w += v.w;
        }
        const float v[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (n + e < N) {
                TOut *dst = C + m * ldc + n + e;
                float o = v[e] + (bias != nullptr ? __ldg(bias + n + e) : 0.0f);
                if (accumulate) o += to_f32(*dst);
                *dst = from_f32<TOut>(o);
            }
    }
}

// What a call of these sizes runs: which operand lies along the lanes, the tile's columns, the splits of the sum.
struct Plan {
    bool swap;
    int bn, tiles_p, tiles_q, splits, kb_per_split, kblocks;
    int64_t ldp;  // row stride of a partial product
    size_t bytes() const { return splits > 1 ? (size_t)splits * rows * ldp * sizeof(float) : 0; }
    int64_t rows;
};

Plan plan_of(int64_t M, int64_t N, int64_t K) {
    Plan p;
    p.swap = M <= 64;
    const int64_t rp = p.swap ? N : M, rq = p.swap ? M : N;
    p.tiles_p = (int)div_up(rp, BP);
    p.bn = rq <= 16 ? 16 : rq <= 32 ? 32 : rq <= 64 ? 64 : 128;
    if (p.bn == 128 && (int64_t)p.tiles_p * div_up(rq, 256) >= kNumSMs / 2) p.bn = 256;
    p.tiles_q = (int)div_up(rq, p.bn);
    p.kblocks = (int)div_up(K, BK);
    const int64_t tiles = (int64_t)p.tiles_p * p.tiles_q;
    // a split has at least 4 k-blocks: below that the partial products' traffic outweighs the operands'
    int64_t splits = tiles > 0 ? kNumSMs / tiles : 1;
    if (splits > p.kblocks / 4) splits = p.kblocks / 4;
    if (splits < 1) splits = 1;
    p.kb_per_split = (int)div_up(p.kblocks, splits);
    p.splits = p.kb_per_split > 0 ? (int)div_up(p.kblocks, p.kb_per_split) : 1;
    p.rows = M;
    p.ldp = div_up(N, 4) * 4;
    return p;
}

int make_map_f8(CUtensorMap *map, const void *base, int64_t rows, int64_t cols, int64_t ld, int box_rows) {
    EncodeTiledFn fn = encode_fn();
    if (fn == nullptr) return fail(GNNAGG_ERR_CUDA, "fp8_matmul: cuTensorMapEncodeTiled is not available from the driver");
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)ld};
    const cuuint32_t box[2] = {(cuuint32_t)BK, (cuuint32_t)box_rows};
    const cuuint32_t estr[2] = {1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(base), dims, strides, box, estr,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(GNNAGG_ERR_CUDA, "fp8_matmul: cuTensorMapEncodeTiled failed with code %d", (int)r);
    return GNNAGG_OK;
}

template <int BN, bool QROW, bool SWAP, typename TOut>
int launch(const CUtensorMap &mp, const CUtensorMap &mq, const Params &p, cudaStream_t st) {
    static PerDeviceOnce attr_done;
    const cudaError_t e = attr_done.run([] {
        return cudaFuncSetAttribute(fp8_matmul_kernel<BN, QROW, SWAP, TOut>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    Tile<BN>::kSmem);
    });
    if (e != cudaSuccess)
        return fail(GNNAGG_ERR_CUDA, "fp8_matmul: cannot reserve %d bytes of shared memory: %s", Tile<BN>::kSmem,
                    cudaGetErrorString(e));
    const int grid = p.items < kNumSMs ? p.items : kNumSMs;
    fp8_matmul_kernel<BN, QROW, SWAP, TOut><<<grid, kThreads, Tile<BN>::kSmem, st>>>(mp, mq, p);
    return check_launch("fp8_matmul_kernel");
}

template <bool QROW, typename TOut>
int launch_tile(const Plan &plan, const CUtensorMap &mp, const CUtensorMap &mq, const Params &p, cudaStream_t st) {
    if (plan.swap)
        return plan.bn == 16   ? launch<16, QROW, true, TOut>(mp, mq, p, st)
               : plan.bn == 32 ? launch<32, QROW, true, TOut>(mp, mq, p, st)
                               : launch<64, QROW, true, TOut>(mp, mq, p, st);
    return plan.bn == 16    ? launch<16, QROW, false, TOut>(mp, mq, p, st)
           : plan.bn == 32  ? launch<32, QROW, false, TOut>(mp, mq, p, st)
           : plan.bn == 64  ? launch<64, QROW, false, TOut>(mp, mq, p, st)
           : plan.bn == 128 ? launch<128, QROW, false, TOut>(mp, mq, p, st)
                            : launch<256, QROW, false, TOut>(mp, mq, p, st);
}

template <typename TOut>
int launch_out(bool qrow, const Plan &plan, const CUtensorMap &mp, const CUtensorMap &mq, const Params &p, cudaStream_t st) {
    return qrow ? launch_tile<true, TOut>(plan, mp, mq, p, st) : launch_tile<false, TOut>(plan, mp, mq, p, st);
}

template <typename TOut>
int join(const Plan &plan, const float *partial, int splits, int64_t M, int64_t N, const float *bias, int accumulate,
         void *C, int64_t ldc, cudaStream_t st) {
    const int64_t want = div_up(M * (plan.ldp / 4), 256);
    const int64_t cap = (int64_t)kNumSMs * 8;
    fp8_join_kernel<TOut><<<(unsigned)(want < cap ? want : cap), 256, 0, st>>>(
        partial, splits, M * plan.ldp, plan.ldp, M, N, bias, accumulate, static_cast<TOut *>(C), ldc);
    return check_launch("fp8_join_kernel");
}

int join_out(int type, const Plan &plan, const float *partial, int splits, int64_t M, int64_t N, const float *bias,
             int accumulate, void *C, int64_t ldc, cudaStream_t st) {
    return type == kTypeF32    ? join<float>(plan, partial, splits, M, N, bias, accumulate, C, ldc, st)
           : type == kTypeBf16 ? join<__nv_bfloat16>(plan, partial, splits, M, N, bias, accumulate, C, ldc, st)
                               : join<__half>(plan, partial, splits, M, N, bias, accumulate, C, ldc, st);
}

}  // namespace
}  // namespace gnnagg

using namespace gnnagg;

extern "C" size_t gnnagg_fp8_matmul_workspace_bytes(int64_t M, int64_t N, int64_t K) {
    if (M <= 0 || N <= 0 || K <= 0 || M > 0x7FFFFFFF - 256 || N > 0x7FFFFFFF - 256 || K > 0x7FFFFFFF - 256) return 0;
    return plan_of(M, N, K).bytes();
}

extern "C" int gnnagg_fp8_matmul(const uint8_t *A, int64_t lda, const float *sa, int64_t sa_stride, int64_t sa_stride_k,
                                 int32_t a_block, const uint8_t *B, int64_t ldb, const float *sb, int64_t sb_stride,
                                 int64_t sb_stride_k, int32_t b_block, int64_t M, int64_t N, int64_t K,
                                 const float *bias, int32_t accumulate, void *C, int64_t ldc, int32_t out_type,
                                 void *workspace, size_t workspace_bytes, void *stream) {
    if (M < 0 || N < 0 || K < 0 || (accumulate != 0 && accumulate != 1))
        return fail(GNNAGG_ERR_ARG, "fp8_matmul: negative size or bad accumulate flag");
    if ((a_block != 1 && a_block != 128) || (b_block != 1 && b_block != 128))
        return fail(GNNAGG_ERR_ARG, "fp8_matmul: a scale covers 1 or 128 rows");
    if (type_size(out_type) == 0) return fail(GNNAGG_ERR_ARG, "fp8_matmul: unknown output type %d", out_type);
    if (accumulate && out_type != kTypeF32)
        return fail(GNNAGG_ERR_UNSUPPORTED, "fp8_matmul: accumulation needs an fp32 output");
    if (M == 0 || N == 0) return GNNAGG_OK;
    if (C == nullptr || (K > 0 && (A == nullptr || B == nullptr || sa == nullptr || sb == nullptr)))
        return fail(GNNAGG_ERR_ARG, "fp8_matmul: null pointer");
    if (M > 0x7FFFFFFF - 256 || N > 0x7FFFFFFF - 256 || K > 0x7FFFFFFF - 256)
        return fail(GNNAGG_ERR_UNSUPPORTED, "fp8_matmul: a size exceeds 2^31");
    if (ldc < N || (K > 0 && (lda < K || ldb < K))) return fail(GNNAGG_ERR_ARG, "fp8_matmul: a stride is smaller than its rows");
    if (K > 0 && (!aligned16(A) || !aligned16(B) || lda % 16 != 0 || ldb % 16 != 0))
        return fail(GNNAGG_ERR_UNSUPPORTED, "fp8_matmul: code rows must start on 16 bytes");
    if (sa_stride < 0 || sa_stride_k < 0 || sb_stride < 0 || sb_stride_k < 0)
        return fail(GNNAGG_ERR_ARG, "fp8_matmul: negative scale stride");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const Plan plan = plan_of(M, N, K);
    if (K == 0) return join_out(out_type, plan, nullptr, 0, M, N, bias, accumulate, C, ldc, st);
    const bool split = plan.splits > 1;
    if (split && (workspace == nullptr || !aligned16(workspace) || workspace_bytes < plan.bytes()))
        return fail(GNNAGG_ERR_SCRATCH, "fp8_matmul: workspace too small or misaligned (need %zu bytes)", plan.bytes());
    if ((int64_t)plan.tiles_p * plan.tiles_q * plan.splits > 0x7FFFFFFF)
        return fail(GNNAGG_ERR_UNSUPPORTED, "fp8_matmul: too many tiles");

    const Scales za{sa, sa_stride, sa_stride_k}, zb{sb, sb_stride, sb_stride_k};
    CUtensorMap map_p, map_q;
    int rc = plan.swap ? make_map_f8(&map_p, B, N, K, ldb, BP) : make_map_f8(&map_p, A, M, K, lda, BP);
    if (rc == GNNAGG_OK)
        rc = plan.swap ? make_map_f8(&map_q, A, M, K, lda, plan.bn) : make_map_f8(&map_q, B, N, K, ldb, plan.bn);
    if (rc != GNNAGG_OK) return rc;

    Params p;
    p.C = split ? workspace : C;
    p.bias = split ? nullptr : bias;
    p.sp = plan.swap ? zb : za;
    p.sq = plan.swap ? za : zb;
    p.rows_p = plan.swap ? N : M;
    p.rows_q = plan.swap ? M : N;
    p.ldc = split ? plan.ldp : ldc;
    p.split_stride = split ? M * plan.ldp : 0;
    p.p_block = (plan.swap ? b_block : a_block) == 128;
    p.kblocks = plan.kblocks;
    p.splits = plan.splits;
    p.kb_per_split = plan.kb_per_split;
    p.tiles_p = plan.tiles_p;
    p.tiles_q = plan.tiles_q;
    p.items = plan.tiles_p * plan.tiles_q * plan.splits;
    p.accumulate = split ? 0 : accumulate;
    p.vec_out = split || (aligned16(C) && (ldc * type_size(out_type)) % 16 == 0);
    p.wait_ns = g_stall.wait_ns;
    p.tx_excess = g_stall.tx_excess;
    const bool qrow = (plan.swap ? a_block : b_block) == 1;
    const int type = split ? (int)kTypeF32 : out_type;
    rc = type == kTypeF32    ? launch_out<float>(qrow, plan, map_p, map_q, p, st)
         : type == kTypeBf16 ? launch_out<__nv_bfloat16>(qrow, plan, map_p, map_q, p, st)
                             : launch_out<__half>(qrow, plan, map_p, map_q, p, st);
    if (rc != GNNAGG_OK || !split) return rc;
    return join_out(out_type, plan, static_cast<const float *>(workspace), plan.splits, M, N, bias, accumulate, C, ldc, st);
}

extern "C" int gnnagg_fp8_matmul_status(void *stream) {
    int code = 0;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t e = cudaMemcpyFromSymbolAsync(&code, g_status, sizeof(int), 0, cudaMemcpyDeviceToHost, st);
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
    if (e != cudaSuccess) return fail(GNNAGG_ERR_CUDA, "fp8_matmul_status: %s", cudaGetErrorString(e));
    return code;
}

extern "C" int gnnagg_fp8_matmul_status_clear(void *stream) {
    static const int zero = 0;
    const cudaError_t e =
        cudaMemcpyToSymbolAsync(g_status, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, static_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) return fail(GNNAGG_ERR_CUDA, "fp8_matmul_status_clear: %s", cudaGetErrorString(e));
    return GNNAGG_OK;
}
