// Matrix product of e4m3 operands with a scale for each block of 128 along the sum, on the tensor cores (tcgen05 +
// TMEM + TMA), sm_100a:
//
//     C[m,n] = sum_kb  sa[m,kb] * sb[n,kb] * ( sum_{k in block kb} A[m,k] B[n,k] )   (+ bias[n]) (+ C[m,n])
//
// Scales are fp32, one per row or one per 128 rows of either operand.  The inner sum of a block is a chain of four
// MMAs into tensor memory; the outer one is taken in registers, one FMA per element and block, rounded to nearest (two
// FMAs packed into one instruction are no faster: 258 cycles a block against 262).  Tensor memory holds several blocks'
// partial products, so the MMAs of the next block run under the FMAs of the last.
//
// One operand lies along the 128 lanes of tensor memory (P), the other along its columns (Q).  P is A and Q is B,
// except for few rows of A (SWAP): then the weight's rows fill the lanes and the few rows are the columns.
//
// One persistent CTA per SM:
//   warp 0      issues the TMA loads (a 128-byte wide k-block of both operands per stage);
//   warp 1      allocates tensor memory, issues tcgen05.mma (kind::f8f6f4) and the commits;
//   warps 2-3   take turns with a block's scales: bring them (cp.async, two turns ahead), multiply the two operands'
//               where one of Q's covers 128 columns, and lay them out beside the partial product, whose barrier
//               hands over both;
//   warps 4-11  read a block's product, scale and add it; after the last block, convert and store.  Warp w reads
//               lane quarter w % 4 and one half of the columns.
// What bounds a block is the scaling warps' chain: the wait, the tensor-memory reads, the FMAs, the release, over two
// partial products.  At 4096 x 4096 x 4096 a block takes 985 cycles, of which the MMAs fill 512; the schedulers issue in 55 %
// of them and the FMA pipe is busy in 31 %.  With row scales on both sides it takes 1525 (512, 60 %, 38 %).  No unit is
// full, so the scaling loop holds nothing that another warp can do.  8192 x 8192 x 8192 takes 500 us alone, 2.2 PFLOP/s, and
// 580 in a long run, where the power limit takes the clock from 1965 to about 1490 MHz (780 and 830 with row scales).
// Two CTAs that share a tile's operands were slower (the hand-over then goes through both), and so were tiles 128 wide
// with two CTAs an SM (644 us where this took 539 at the time), and sixteen scaling warps.
// Where one column of tiles and few k-blocks make up the product (tall activations, a small weight), Q stays in shared
// memory and only P's blocks go round: a third of the loads, and twice the blocks on their way (612500 x 256 x 100 in
// 82 us instead of 109; its bytes take 58).  A tile of one block then takes 3900 cycles, most of them in the chain from the
// product over the conversion to the stores: DRAM is at half its rate, the schedulers issue in 43 %.
// Output tiles leave through shared memory by TMA stores, which run under the next tile's MMAs; rows that TMA cannot
// address, and outputs that are added to, by plain stores (four bytes at a time: 612500 x 256 x 256 in fp32 takes 900 us
// with the addition and 141 without).
// The tiles of a last round that would leave SMs idle are shared out evenly instead: each CTA takes the same number of
// their k-blocks, a stretch that lies in one tile or two.  Whoever completes a tile (a count per tile and warp, no
// waiting) adds its parts in the order of k and stores it.
// A tile's sum may be split along k over several CTAs (few tiles, long sums): each writes an fp32 partial product
// to the workspace and a second kernel adds them in a fixed order (256 x 256 x 612500: 94 us, 19 of them that kernel); up
// to eight small ones (few rows) are CTAs of a cluster, and the first adds the others' from its own shared memory, which
// saves the second launch (8 x 4096 x 4096: 10 us a call).
// Every wait is bounded (about a second); on a time-out the kernel records a code in the library's status word,
// drains its own copies and MMAs, frees tensor memory and returns.
#include "lowp.cuh"
#include "tc.cuh"

namespace gnnagg {
namespace {

constexpr int BP = 128;                        // rows of P per CTA and tile = TMEM lanes
constexpr int BK = 128;                        // bytes = elements per k-block = one scale block = one swizzle row
constexpr int UMMA_K = 32;                     // elements per tcgen05.mma
constexpr int kTmemCols = 512;
constexpr int P_BYTES = BP * BK;
constexpr int kPanel = 32 * 128;               // 32 rows of 128 bytes of the output, as a warp stages them
constexpr int kRing = 3;                       // a scale warp's blocks: in use and on their way
constexpr int kMaxStages = 10;
constexpr int kBarBytes = 256;
constexpr int kSmemLimit = 227 * 1024;
// Registers per thread of the widest tiles after the launch: the control warpgroup gives up what the scaling ones
// take (sums up to what the block was launched with; launch() checks that before the first run).
constexpr int kRegsControl = 72, kRegsScaling = 216;

// BN columns per tile; QROW: Q's scales are per row.
template <int BN, bool QROW>
struct Tile {
    static constexpr int kParts = BN >= 32 ? 2 : 1;                        // shares of the columns
    static constexpr int kCols = BN / kParts;                              // columns of a warp: 16 to 128
    static constexpr int kWarps = 4 * kParts;                              // scaling warps
    static constexpr int kThreads = 128 + 32 * kWarps;
    static constexpr int kStageBytes = P_BYTES + BN * BK;
    static constexpr int kBufs = kTmemCols / BN > 4 ? 4 : kTmemCols / BN;  // partial products in tensor memory
    static constexpr int kSets = (BN + 127) / 128;                         // scales of Q, when one covers 128 columns
    static constexpr int kRaw = BP + (QROW ? BN : 4);                      // floats: scales as loaded, of a block
    static constexpr int kSlot = QROW ? BP + BN : BP * kSets;              // floats: scales as used, of a block
    static constexpr int kPanels = kCols == 128 ? 2 : 1;                   // staged panels per warp
    static constexpr int kWarpBytes = kPanels * kPanel + kCols * 4;
    static constexpr int kFixed = 1024 + kBarBytes + kWarps * kWarpBytes + (2 * kRing * kRaw + kBufs * kSlot) * 4;
    static constexpr int kFit = (kSmemLimit - kFixed) / kStageBytes;
    static constexpr int kStages = kFit > kMaxStages ? kMaxStages : kFit;
    static constexpr int kSmem = kFixed + kStages * kStageBytes;
    static constexpr int kBarriers = 2 * kMaxStages + 2 * kBufs + 2;
    static_assert(kSmem <= kSmemLimit && kStages >= 3 && kBarriers * 8 + 8 <= kBarBytes, "shared memory budget");
    static constexpr bool kSplitRegs = BN == 256;
    static constexpr int kRegsNeeded = 128 * kRegsControl + 32 * kWarps * kRegsScaling;
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
    const void *bias;
    int bias_type;
    Scales sp, sq;
    int64_t rows_p, rows_q, ldc, split_stride;
    int p_block;         // P's scales are per 128 rows
    int kblocks, splits, kb_per_split;
    int tiles_p, tiles_q, items;
    int stages;          // of the ring; with keep_q they hold P alone, behind Q's k-blocks
    int keep_q;
    int accumulate;
    int vec_out;         // 16-byte stores of the output's rows
    int tma_out;         // the output leaves by TMA
    unsigned long long wait_ns;
    uint32_t tx_excess;
    float *parts;        // sums of shared tiles' parts, two places a CTA
    int *counts;         // parts of a shared tile that are there, for each scaling warp
    int full, tail, per; // tiles that have a CTA of their own, tiles that are shared, k-blocks of these for each CTA
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

__device__ __forceinline__ void cluster_sync() {
    __syncwarp();  // the barrier's aligned form wants whole warps
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Stores to the shared memory of the cluster's first CTA, at the place of this CTA's address `addr`.
__device__ __forceinline__ void st_first(uint32_t addr, float v) {
    asm volatile(
        "{\n"
        ".reg .b32 r;\n"
        "mapa.shared::cluster.u32 r, %0, 0;\n"
        "st.shared::cluster.f32 [r], %1;\n"
        "}\n" ::"r"(addr), "f"(v)
        : "memory");
}

// 4 bytes global -> shared, or zero when !ok.
__device__ __forceinline__ void cp_async_4_or_zero(uint32_t dst, const float *src, bool ok) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(ok ? 4 : 0) : "memory");
}

// 16 bytes, of which the first `bytes` (0 to 16) are read and the others zero.
__device__ __forceinline__ void cp_async_16_or_less(uint32_t dst, const float *src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// The warp's copies of N scales of block kb, of the rows from row0 on (zero behind `rows`): 16 bytes a lane where the
// rows' scales lie side by side, a quarter of the instructions (4-byte copies kept the scale warps at 900 cycles a block).
template <int N>
__device__ __forceinline__ void fetch_scales(uint32_t dst, const Scales &s, int64_t row0, int64_t rows, int rows_each, int kb,
                                             int lane) {
    const float *base = s.p + kb * s.stride_k;
    if (s.stride == 1 && rows_each == 1 && (reinterpret_cast<uintptr_t>(base) & 15u) == 0) {
#pragma unroll
        for (int j = 0; j < N; j += 128) {
            const int64_t r = row0 + j + 4 * lane;
            const int left = (int)(rows - r < 4 ? (rows - r < 0 ? 0 : rows - r) : 4);
            if (j + 4 * lane < N) cp_async_16_or_less(dst + (j + 4 * lane) * 4, left > 0 ? base + r : base, 4 * left);
        }
    } else {
#pragma unroll 1
        for (int j = lane; j < N; j += 32) {
            const int64_t r = row0 + j;
            cp_async_4_or_zero(dst + j * 4, r < rows ? base + (rows_each == 1 ? r : r / 128) * s.stride : s.p, r < rows);
        }
    }
}

// Instruction descriptor of kind::f8f6f4: fp32 accumulator, e4m3 A and B (format 0), both K-major, M = 128.
__host__ __device__ constexpr uint32_t f8_instr_desc(int n) {
    return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(BP >> 4) << 24);
}

// A work item: one tile of the output and a range of its k-blocks.  Of a shared tile: its number among them, and the
// CTAs that have a part of it.
struct Item {
    int tp, tq, split, kb0, kb1;
    int shared, cta0, ctas;
};
// The shared tiles' k-blocks lie one behind the other, CTA c has [c per, (c + 1) per); per is less than a tile's.
__device__ __forceinline__ int shared_first(const Params &p, int cta) { return cta * p.per / p.kblocks; }
// Tiles of one column strip of 16 P-tiles are neighbours, so that concurrent CTAs share operand panels in L2.
template <bool TAIL>
__device__ __forceinline__ Item item_of(const Params &p, int i) {
    Item w;
    int t = i;
    w.split = 0, w.tq = 0;
    if (TAIL) w.ctas = 1;
    w.kb0 = 0, w.kb1 = p.kblocks;
    if (TAIL && i >= p.full) {
        const int second = i - p.full >= kNumSMs ? 1 : 0, cta = i - p.full - second * kNumSMs;
        const int a = cta * p.per, e = min(a + p.per, p.tail * p.kblocks);
        w.shared = shared_first(p, cta) + second;
        const int begin = w.shared * p.kblocks;
        w.kb0 = max(a - begin, 0);
        w.kb1 = min(e - begin, p.kblocks);  // not above kb0: this CTA has no such part
        w.cta0 = begin / p.per;
        w.ctas = (begin + p.kblocks - 1) / p.per - w.cta0 + 1;
        w.tp = 0;
        if (w.kb0 >= w.kb1) return w;
        t = p.full + w.shared;
    }
    if (!TAIL && p.splits > 1) {
        t = i / p.splits;
        w.split = i - t * p.splits;
        w.kb0 = w.split * p.kb_per_split;
        w.kb1 = min(p.kblocks, w.kb0 + p.kb_per_split);
    }
    w.tp = t;
    if (p.tiles_q > 1) {
        constexpr int kGroup = 16;
        const int per = kGroup * p.tiles_q, g = t / per, r = t - g * per;
        const int high = min(kGroup, p.tiles_p - g * kGroup);
        w.tq = r / high;
        w.tp = g * kGroup + (r - w.tq * high);
    }
    return w;
}

// Place and phase parity in a ring of n barriers.
struct Ring {
    int n;
    int i = 0;
    uint32_t phase = 0;
    __device__ __forceinline__ explicit Ring(int size) : n(size) {}
    __device__ __forceinline__ void next() {
        if (++i == n) i = 0, phase ^= 1u;
    }
};

// SWAP: the output is stored transposed, C[column][lane].  SHARE: with SWAP the splits of a tile are a cluster, without
// the last round's tiles are shared out (a variant of its own: the others lose 2 to 5 % to its code).
template <int BN, bool QROW, bool SWAP, bool SHARE, typename TOut>
__global__ void __launch_bounds__((Tile<BN, QROW>::kThreads), 1)
fp8_matmul_kernel(const __grid_constant__ CUtensorMap map_p, const __grid_constant__ CUtensorMap map_q,
                  const __grid_constant__ CUtensorMap map_c, const Params p) {
    using S = Tile<BN, QROW>;
    constexpr bool JOIN = SWAP && SHARE, TAIL = !SWAP && SHARE;
    constexpr int kBufs = S::kBufs, kCols = S::kCols, kWarps = S::kWarps;
    extern __shared__ uint8_t smem_raw[];
    // 1024-byte alignment: the swizzle pattern and the descriptors assume it
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t *staging = smem + S::kStages * S::kStageBytes;
    float *bias_s = reinterpret_cast<float *>(staging + kWarps * S::kPanels * kPanel);  // kCols per warp
    float *raw = bias_s + kWarps * kCols;                                                // kRing * kRaw per scale warp
    float *slots = raw + 2 * kRing * S::kRaw;                                                // one per partial product
    uint64_t *bars = reinterpret_cast<uint64_t *>(slots + kBufs * S::kSlot);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + S::kBarriers);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const uint32_t bar0 = smem_u32(bars);
    auto bar_full = [&](int s) { return bar0 + 8u * (uint32_t)s; };
    auto bar_empty = [&](int s) { return bar0 + 8u * (uint32_t)(kMaxStages + s); };
    auto bar_acc_full = [&](int b) { return bar0 + 8u * (uint32_t)(2 * kMaxStages + b); };
    auto bar_acc_empty = [&](int b) { return bar0 + 8u * (uint32_t)(2 * kMaxStages + kBufs + b); };
    const uint32_t bar_drain = bar0 + 8u * (uint32_t)(2 * kMaxStages + 2 * kBufs);
    const uint32_t bar_q = bar_drain + 8u;  // Q has landed, where it stays
    // where a stage's P and Q begin
    const uint32_t stage0 = smem_u32(smem) + (p.keep_q ? (uint32_t)(p.kblocks * BN * BK) : 0u);
    const uint32_t stage_step = p.keep_q ? P_BYTES : S::kStageBytes;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(bar_full(s), 1);
            mbar_init(bar_empty(s), 1);
        }
        for (int b = 0; b < kBufs; ++b) {
            mbar_init(bar_acc_full(b), 2);  // the product, the scales
            mbar_init(bar_acc_empty(b), kWarps);
        }
        mbar_init(bar_drain, 1);
        mbar_init(bar_q, 1);
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
        if (S::kSplitRegs) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsControl));
        if (warp == 0) {
            // ---------------- TMA issuer ----------------
            Ring st(p.stages);
            uint32_t it = 0;
            bool ok = true;
            if (p.keep_q && elect_one()) {
                mbar_arrive_expect_tx(bar_q, (uint32_t)(p.kblocks * BN * BK));
                for (int kb = 0; kb < p.kblocks; ++kb)
                    tma_load_2d(smem_u32(smem) + (uint32_t)(kb * BN * BK), &map_q, bar_q, kb * BK, 0);
            }
            __syncwarp();
            for (int i = blockIdx.x; i < p.items && ok; i += gridDim.x) {
                const Item w = item_of<TAIL>(p, i);
                for (int kb = w.kb0; kb < w.kb1; ++kb, ++it, st.next()) {
                    if (!mbar_wait(bar_empty(st.i), st.phase ^ 1u, abort_flag, &g_status, kErrWaitEmpty, p.wait_ns)) {
                        ok = false;
                        break;
                    }
                    if (elect_one()) {
                        const uint32_t sp = stage0 + (uint32_t)st.i * stage_step;
                        mbar_arrive_expect_tx(bar_full(st.i), stage_step + p.tx_excess);
                        tma_load_2d(sp, &map_p, bar_full(st.i), kb * BK, w.tp * BP);
                        if (!p.keep_q) tma_load_2d(sp + P_BYTES, &map_q, bar_full(st.i), kb * BK, w.tq * BN);
                    }
                    __syncwarp();
                }
            }
            if (!ok) {
                // copies of the last k-blocks issued may still be landing: wait for them, bounded
                const uint32_t n = (uint32_t)p.stages;
                for (uint32_t back = 0; back <= n && back <= it; ++back) {
                    if (back == 0 && !p.keep_q) continue;
                    const uint32_t j = it - back, bar = back == 0 ? bar_q : bar_full((int)(j % n));
                    const unsigned long long t0 = globaltimer_ns();
                    while (!mbar_try_wait(bar, back == 0 ? 0u : (j / n) & 1u)) {
                        if (globaltimer_ns() - t0 > p.wait_ns) {
                            atomicCAS(&g_status, 0, (int)kErrDrain);
                            break;
                        }
                    }
                }
            }
        } else if (warp == 1) {
            // ---------------- MMA issuer ----------------
            Ring st(p.stages);
            Ring ac(kBufs);
            bool ok = !p.keep_q || mbar_wait(bar_q, 0, abort_flag, &g_status, kErrWaitFull, p.wait_ns);
            for (int i = blockIdx.x; i < p.items && ok; i += gridDim.x) {
                const Item w = item_of<TAIL>(p, i);
                for (int kb = w.kb0; kb < w.kb1; ++kb, st.next(), ac.next()) {
                    if (!mbar_wait(bar_full(st.i), st.phase, abort_flag, &g_status, kErrWaitFull, p.wait_ns) ||
                        !mbar_wait(bar_acc_empty(ac.i), ac.phase ^ 1u, abort_flag, &g_status, kErrWaitAccFree, p.wait_ns)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    if (elect_one()) {
                        const uint32_t sp = stage0 + (uint32_t)st.i * stage_step;
                        const uint32_t sq = p.keep_q ? smem_u32(smem) + (uint32_t)(kb * BN * BK) : sp + P_BYTES;
                        const uint64_t dp = make_smem_desc(sp), dq = make_smem_desc(sq);
                        const uint32_t d = tmem_base + (uint32_t)(ac.i * BN);
#pragma unroll
                        for (int k = 0; k < BK / UMMA_K; ++k)  // 32 bytes further inside the swizzled row
                            tc_mma_f8(d, dp + (uint64_t)(2 * k), dq + (uint64_t)(2 * k), f8_instr_desc(BN), k > 0 ? 1u : 0u);
                        tc_commit(bar_acc_full(ac.i));
                        tc_commit(bar_empty(st.i));
                    }
                    __syncwarp();
                }
            }
            if (!ok) {
                // MMAs already issued still read shared memory and write tensor memory: drain, bounded
                __syncwarp();
                if (elect_one()) tc_commit(bar_drain);
                __syncwarp();
                const unsigned long long t0 = globaltimer_ns();
                while (!mbar_try_wait(bar_drain, 0)) {
                    if (globaltimer_ns() - t0 > p.wait_ns) {
                        atomicCAS(&g_status, 0, (int)kErrDrain);
                        break;
                    }
                }
            }
        } else {
            // ---------------- scales ----------------
            float *mine = raw + (warp - 2) * kRing * S::kRaw;
            Ring ac(kBufs);
            uint32_t it = 0;  // of all blocks; this warp has every second
            bool ok = true;
            for (int i = blockIdx.x; i < p.items && ok; i += gridDim.x) {
                const Item w = item_of<TAIL>(p, i);
                if (TAIL && w.kb0 >= w.kb1) continue;
                const int64_t row0 = (int64_t)w.tp * BP, col0 = (int64_t)w.tq * BN;
                const int first = w.kb0 + (int)((it ^ (uint32_t)(warp - 2)) & 1u);
                auto fetch = [&](int kb) {
                    if (kb < w.kb1) {
                        const uint32_t dst = smem_u32(mine) + (uint32_t)((kb - first) / 2 % kRing * S::kRaw) * 4;
                        fetch_scales<BP>(dst, p.sp, row0, p.rows_p, p.p_block ? 128 : 1, kb, lane);
                        if (QROW)
                            fetch_scales<BN>(dst + BP * 4, p.sq, col0, p.rows_q, 1, kb, lane);
                        else if (lane < S::kSets)
                            cp_async_4_or_zero(dst + (BP + lane) * 4,
                                               p.sq.p + min(col0 / 128 + lane, (p.rows_q - 1) / 128) * p.sq.stride +
                                                   kb * p.sq.stride_k,
                                               true);
                    }
                    cp_async_commit();
                };
                for (int a = 0; a + 1 < kRing; ++a) fetch(first + 2 * a);
                for (int kb = w.kb0; kb < w.kb1; ++kb, ++it, ac.next()) {
                    if (((kb - first) & 1) != 0) continue;
                    cp_async_wait<kRing - 2>();
                    // the scaling warps have read what this slot held
                    if (!__all_sync(kFullMask, mbar_wait(bar_acc_empty(ac.i), ac.phase ^ 1u, abort_flag, &g_status,
                                                         kErrWaitAccFree, p.wait_ns))) {
                        ok = false;
                        break;
                    }
                    __syncwarp();  // other lanes' copies are read: each lane has waited for its own, the barrier orders them
                    const float *src = mine + (kb - first) / 2 % kRing * S::kRaw;
                    float *dst = slots + ac.i * S::kSlot;
                    const float4 a = *reinterpret_cast<const float4 *>(src + 4 * lane);
                    if (QROW) {
                        *reinterpret_cast<float4 *>(dst + 4 * lane) = a;
#pragma unroll
                        for (int j = 0; j < BN; j += 128)
                            if (j + 4 * lane < BN)
                                *reinterpret_cast<float4 *>(dst + BP + j + 4 * lane) =
                                    *reinterpret_cast<const float4 *>(src + BP + j + 4 * lane);
                    } else {
#pragma unroll
                        for (int j = 0; j < S::kSets; ++j) {
                            const float b = src[BP + j];
                            *reinterpret_cast<float4 *>(dst + j * BP + 4 * lane) = make_float4(a.x * b, a.y * b, a.z * b, a.w * b);
                        }
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar_acc_full(ac.i));
                    fetch(kb + 2 * (kRing - 1));
                }
                cp_async_wait<0>();
                __syncwarp();
            }
        }
        if (JOIN) {  // the two barriers of the scaling warps
            cluster_sync();
            cluster_sync();
        }
    } else {
        // ---------------- scaling warps ----------------
        if (S::kSplitRegs) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsScaling));
        const int q = warp & 3, part = (warp - 4) >> 2;
        uint8_t *mine = staging + (warp - 4) * S::kPanels * kPanel;
        auto release = [&](uint32_t bar) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);
        };
        constexpr int kChunk = kCols > 32 ? (QROW ? 8 : 16) : kCols;
        Ring ac(kBufs);
        float *bias = bias_s + (warp - 4) * kCols;
        int64_t bias_at = -1;  // first column of the bias that is there
        uint32_t limit = 1u << 22;
        for (int i = blockIdx.x; i < p.items; i += gridDim.x) {
            const Item w = item_of<TAIL>(p, i);
            if (TAIL && w.kb0 >= w.kb1) continue;
            const int64_t row0 = (int64_t)w.tp * BP + q * 32;                    // of P
            const int64_t col0 = (int64_t)w.tq * BN + part * kCols;              // of Q
            float acc[kCols];
#pragma unroll
            for (int j = 0; j < kCols; ++j) acc[j] = 0.0f;
            for (int kb = w.kb0; kb < w.kb1; ++kb, ac.next()) {
                // a wait that is counted in polls (up to about a second) and leaves the loop alone (a vote of the warp to
                // leave it costs 1 % of the time): after a time-out the sums are not used, and later waits poll once
                uint32_t polls = 0;
                while (!mbar_try_wait(bar_acc_full(ac.i), ac.phase))
                    if (limit == 0 || ((++polls & 1023u) == 0 && (polls > limit || *abort_flag != 0))) {
                        limit = 0;
                        break;
                    }
                __syncwarp();  // the tensor-memory loads are warp-collective
                const float *slot = slots + ac.i * S::kSlot;
                const float scale = slot[(QROW ? 0 : part * kCols / 128 * BP) + q * 32 + lane];
                const float *col = slot + BP + part * kCols;
                tc_fence_after();
                const uint32_t taddr = tmem_base + (uint32_t)(ac.i * BN + part * kCols) + ((uint32_t)(q * 32) << 16);
                // the next columns are on their way while the FMAs of the last ones run
                uint32_t r[2][kChunk];
                TmemLoad<kChunk>::run(taddr, r[0]);
#pragma unroll
                for (int c0 = 0; c0 < kCols; c0 += kChunk) {
                    uint32_t(&now)[kChunk] = r[c0 / kChunk & 1];
                    TmemLoad<kChunk>::wait(now);
                    if (c0 + kChunk < kCols) {
                        TmemLoad<kChunk>::run(taddr + (uint32_t)(c0 + kChunk), r[(c0 / kChunk + 1) & 1]);
                    } else if (!QROW) {  // all of the partial product is in registers
                        release(bar_acc_empty(ac.i));
                    }
#pragma unroll
                    for (int j = 0; j < kChunk; j += 4) {
                        if (QROW) {
                            const float4 cs = *reinterpret_cast<const float4 *>(col + c0 + j);
                            acc[c0 + j] = fmaf(__uint_as_float(now[j]), scale * cs.x, acc[c0 + j]);
                            acc[c0 + j + 1] = fmaf(__uint_as_float(now[j + 1]), scale * cs.y, acc[c0 + j + 1]);
                            acc[c0 + j + 2] = fmaf(__uint_as_float(now[j + 2]), scale * cs.z, acc[c0 + j + 2]);
                            acc[c0 + j + 3] = fmaf(__uint_as_float(now[j + 3]), scale * cs.w, acc[c0 + j + 3]);
                        } else {
#pragma unroll
                            for (int e = j; e < j + 4; ++e) acc[c0 + e] = fmaf(__uint_as_float(now[e]), scale, acc[c0 + e]);
                        }
                    }
                }
                if (QROW) release(bar_acc_empty(ac.i));  // the column scales have been read too
            }
            if (__any_sync(kFullMask, limit == 0)) {
                *abort_flag = 1;
                atomicCAS(&g_status, 0, (int)kErrWaitAccFull);
                if (JOIN) {
                    cluster_sync();
                    cluster_sync();
                }
                break;
            }
            if (JOIN) {
                // one tile per cluster: its CTAs' sums go to the first one, into stages that its MMAs have left, and
                // are added there in rank order
                cluster_sync();
                float *sums = reinterpret_cast<float *>(smem) + (warp - 4) * kCols * 32 + lane;
                if (w.split > 0) {
#pragma unroll
                    for (int j = 0; j < kCols; ++j)
                        st_first(smem_u32(sums + ((w.split - 1) * kWarps * kCols + j) * 32), acc[j]);
                }
                cluster_sync();
                if (w.split > 0) break;
                for (int r = 1; r < p.splits; ++r)
#pragma unroll
                    for (int j = 0; j < kCols; ++j) acc[j] += sums[((r - 1) * kWarps * kCols + j) * 32];
            }
            if (TAIL && w.ctas > 1) {
                auto place = [&](int cta) {  // of this warp's share of the tile's part
                    const int second = shared_first(p, cta) != w.shared;
                    return p.parts + ((int64_t)((cta * 2 + second) * kWarps + (warp - 4)) * kCols) * 32 + lane;
                };
                float *own = place((int)blockIdx.x);
#pragma unroll
                for (int j = 0; j < kCols; ++j) __stcg(own + j * 32, acc[j]);
                __threadfence();
                __syncwarp();
                int there = 0;
                if (lane == 0) there = atomicAdd(p.counts + w.shared * kWarps + (warp - 4), 1) + 1;
                there = __shfl_sync(kFullMask, there, 0);
                if (there < w.ctas) continue;  // another one completes the tile
                __threadfence();
#pragma unroll
                for (int j = 0; j < kCols; ++j) acc[j] = 0.0f;
                for (int c = w.cta0; c < w.cta0 + w.ctas; ++c) {
                    const float *src = place(c);
#pragma unroll
                    for (int j = 0; j < kCols; ++j) acc[j] += __ldcg(src + j * 32);
                }
            }
            if (SWAP) {
                // lane = column of the output: 32 neighbouring columns of one output row per store
                const int64_t row = row0 + lane;
                const float bias = p.bias != nullptr && row < p.rows_p ? load_as_f32(p.bias, p.bias_type, row) : 0.0f;
                TOut *dst = static_cast<TOut *>(p.C) + (JOIN ? 0 : w.split * p.split_stride) + col0 * p.ldc + row;
#pragma unroll
                for (int j = 0; j < kCols; ++j, dst += p.ldc) {
                    if (row < p.rows_p && col0 + j < p.rows_q) {
                        float o = acc[j] + bias;
                        if (p.accumulate) o += to_f32(*dst);
                        *dst = from_f32<TOut>(o);
                    }
                }
            } else {
                // panels of 128 bytes of each of the warp's 32 rows in shared memory; 16-byte piece j of row r sits at
                // piece j ^ (r & 7), the 128-byte swizzle of the output's tensor map
                constexpr int kPiece = 16 / (int)sizeof(TOut);                       // columns per 16 bytes
                constexpr int kSpan = kCols < 8 * kPiece ? kCols : 8 * kPiece;       // columns per panel
                constexpr int kPieces = kSpan / kPiece;
                const int valid = (int)(p.rows_q - col0 < kCols ? p.rows_q - col0 : kCols);
                if (col0 != bias_at) {  // zeros where there is no bias
                    __syncwarp();
                    for (int j = lane; j < kCols; j += 32)
                        bias[j] = p.bias != nullptr && j < valid ? load_as_f32(p.bias, p.bias_type, col0 + j) : 0.0f;
                    __syncwarp();
                    bias_at = col0;
                }
#pragma unroll
                for (int c0 = 0; c0 < kCols; c0 += kSpan * S::kPanels) {
                    if (p.tma_out) {
                        if (lane == 0) tma_store_wait_read<0>();  // the stores that last read the panels are done
                        __syncwarp();
                    }
#pragma unroll
                    for (int c = c0; c < c0 + kSpan * S::kPanels && c < kCols; c += kSpan) {
                        uint8_t *panel = mine + (c - c0) / kSpan * kPanel;
#pragma unroll
                        for (int j = 0; j < kPieces; ++j) {
                            float v[kPiece];
#pragma unroll
                            for (int e = 0; e < kPiece; e += 4) {
                                const float4 u = *reinterpret_cast<const float4 *>(bias + c + j * kPiece + e);
                                const float *a = acc + c + j * kPiece + e;
                                v[e] = a[0] + u.x, v[e + 1] = a[1] + u.y, v[e + 2] = a[2] + u.z, v[e + 3] = a[3] + u.w;
                            }
                            *reinterpret_cast<uint4 *>(panel + lane * 128 + ((j ^ (lane & 7)) << 4)) = pack16<TOut>(v);
                        }
                    }
                    if (p.tma_out) {
                        fence_generic_to_async_smem();
                        __syncwarp();
                        if (lane == 0) {
#pragma unroll
                            for (int c = c0; c < c0 + kSpan * S::kPanels && c < kCols; c += kSpan)
                                if (c < valid)
                                    tma_store_3d(&map_c, smem_u32(mine) + (uint32_t)((c - c0) / kSpan * kPanel), (int)col0 + c,
                                                 (int)row0, w.split);
                            tma_store_commit();
                        }
                        continue;
                    }
                    __syncwarp();
#pragma unroll
                    for (int c = c0; c < c0 + kSpan * S::kPanels && c < kCols; c += kSpan) {
                        const uint8_t *panel = mine + (c - c0) / kSpan * kPanel;
                        const int j0 = lane & 7, left = valid - (c + j0 * kPiece);  // columns of this lane's piece that exist
                        TOut *dst = static_cast<TOut *>(p.C) + w.split * p.split_stride + (row0 + (lane >> 3)) * p.ldc + col0 + c +
                                    j0 * kPiece;
#pragma unroll
                        for (int t = 0; t < 8; ++t, dst += 4 * p.ldc) {
                            const int r = 4 * t + (lane >> 3);
                            if (j0 < kPieces && left > 0 && row0 + r < p.rows_p) {
                                const uint4 u = *reinterpret_cast<const uint4 *>(panel + r * 128 + ((j0 ^ (r & 7)) << 4));
                                if (p.vec_out && left >= kPiece) {
                                    *reinterpret_cast<uint4 *>(dst) = u;
                                } else {
                                    const TOut *e = reinterpret_cast<const TOut *>(&u);
#pragma unroll
                                    for (int x = 0; x < kPiece; ++x)
                                        if (x < left)
                                            dst[x] = p.accumulate ? from_f32<TOut>(to_f32(dst[x]) + to_f32(e[x])) : e[x];
                                }
                            }
                        }
                    }
                    __syncwarp();
                }
            }
        }
        if (!SWAP && p.tma_out && lane == 0) tma_store_wait_all();  // shared memory stays valid until TMA has read it
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
                const void *bias, int bias_type, int accumulate, TOut *C, int64_t ldc) {
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
                float o = v[e] + (bias != nullptr ? load_as_f32(bias, bias_type, n + e) : 0.0f);
                if (accumulate) o += to_f32(*dst);
                *dst = from_f32<TOut>(o);
            }
    }
}

constexpr int64_t kSharedOperands = 180000000;  // bytes of both operands, up to which a last round is shared out
constexpr size_t kCountBytes = 8192;  // counts of shared tiles: fewer than the SMs, eight warps each
static_assert(kNumSMs * 8 * sizeof(int) <= kCountBytes, "counts of shared tiles");

// What a call of these sizes runs: which operand lies along the lanes, the tile's columns, the splits of the sum.
struct Plan {
    bool swap;
    int bn, tiles_p, tiles_q, splits, kb_per_split, kblocks;
    int64_t ldp;  // row stride of a partial product
    size_t bytes() const {
        if (tail > 0) return kCountBytes + (size_t)2 * kNumSMs * BP * bn * sizeof(float);
        return splits > 1 && !join ? (size_t)splits * rows * ldp * sizeof(float) : 0;
    }
    int64_t rows;
    int tail, per;  // tiles that are shared, k-blocks of these for each CTA
    bool join;    // the splits of a tile are a cluster
};

// Shared memory of the stages of a tile of few rows.
int stage_bytes(int bn) {
    return bn == 16   ? Tile<16, true>::kStages * Tile<16, true>::kStageBytes
           : bn == 32 ? Tile<32, true>::kStages * Tile<32, true>::kStageBytes
                      : Tile<64, true>::kStages * Tile<64, true>::kStageBytes;
}

Plan plan_of(int64_t M, int64_t N, int64_t K) {
    Plan p;
    p.swap = M <= 64;
    const int64_t rp = p.swap ? N : M, rq = p.swap ? M : N;
    p.bn = rq <= 16 ? 16 : rq <= 32 ? 32 : rq <= 64 ? 64 : 128;
    if (rp > BP && rq > 128) p.bn = 256;
    p.tiles_p = (int)div_up(rp, BP);
    p.tiles_q = (int)div_up(rq, p.bn);
    p.kblocks = (int)div_up(K, BK);
    const int64_t tiles = (int64_t)p.tiles_p * p.tiles_q;
    // a split has at least 4 k-blocks: below that the partial products' traffic outweighs the operands'
    int64_t splits = tiles > 0 ? kNumSMs / tiles : 1;
    if (splits > p.kblocks / 4) splits = p.kblocks / 4;
    if (splits < 1) splits = 1;
    p.kb_per_split = (int)div_up(p.kblocks, splits);
    p.splits = p.kb_per_split > 0 ? (int)div_up(p.kblocks, p.kb_per_split) : 1;
    // a cluster has at most eight CTAs; their tiles' sums have to fit behind one another in the first one's stages
    p.join = p.swap && p.splits > 1 && p.splits <= 8 && (p.splits - 1) * BP * p.bn * 4 <= stage_bytes(p.bn);
    p.rows = M;
    p.ldp = div_up(N, 4) * 4;
    // A last round of fewer tiles than SMs is shared out where that shortens it by 40 k-blocks or more (a block takes
    // 0.5 us, 0.8 with row scales on both sides; the parts' way through memory and the cleared counts 12 to 14 us in all).
    // 2048 x 2560 x 8192: 73 -> 66 us, with row scales 116 -> 91; 4096 x 4096 x 4096, 17 blocks shorter: 80 -> 86.  CTAs
    // that share a tile are at different k at a time, so the operands have to stay in L2 in the main: at 168 MB (8192 x
    // 2048 x 16384) 275 -> 262 and 424 -> 391, at 210 MB (1500 x 2000 x 60000) 263 -> 352.  At most nine CTAs have a part
    // of a tile.
    p.tail = 0, p.per = 0;
    const int64_t rest = tiles % kNumSMs;
    if (!p.swap && p.bn >= 128 && p.splits == 1 && rest > 0 && K > 0 && M + N <= kSharedOperands / K) {
        int64_t per = div_up(rest * p.kblocks, kNumSMs);
        if (per < div_up(p.kblocks, 8)) per = div_up(p.kblocks, 8);
        if (per < 4) per = 4;
        if (p.kblocks - per >= 40) p.tail = (int)rest, p.per = (int)per;
    }
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

// The output as `splits` matrices of M x N one behind the other, in boxes of 128 bytes x 32 rows; a tile's part
// outside its matrix is not written, but for what completes a row's last 16 bytes.
int make_map_out(CUtensorMap *map, void *base, int type, int splits, int64_t M, int64_t N, int64_t ld) {
    EncodeTiledFn fn = encode_fn();
    const int size = type_size(type);
    const cuuint64_t dims[3] = {(cuuint64_t)N, (cuuint64_t)M, (cuuint64_t)splits};
    const cuuint64_t strides[2] = {(cuuint64_t)(ld * size), (cuuint64_t)(M * ld * size)};
    const cuuint32_t box[3] = {(cuuint32_t)(128 / size), 32, 1};
    const cuuint32_t estr[3] = {1, 1, 1};
    const CUtensorMapDataType dt = type == kTypeF32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : type == kTypeBf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                       : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const CUresult r = fn(map, dt, 3, base, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(GNNAGG_ERR_CUDA, "fp8_matmul: cuTensorMapEncodeTiled failed with code %d", (int)r);
    return GNNAGG_OK;
}

// Stages of P alone that `bytes` hold beside all of Q's k-blocks, 0 for fewer than three.  In 64 bits: Q may be long.
constexpr int stages_beside_q(int64_t kblocks, int bn, int64_t bytes) {
    const int64_t left = bytes - kblocks * bn * BK;
    return left < 3 * P_BYTES ? 0 : left / P_BYTES < kMaxStages ? (int)(left / P_BYTES) : kMaxStages;
}
static_assert(stages_beside_q(1, 256, 5 * P_BYTES) == 3 && stages_beside_q(1, 16, 64 * P_BYTES) == kMaxStages, "Q that stays");
static_assert(stages_beside_q(2, 256, 5 * P_BYTES) == 0 && stages_beside_q(1 << 16, 256, 5 * P_BYTES) == 0 &&
                  stages_beside_q(1 << 17, 256, 5 * P_BYTES) == 0 && stages_beside_q((1 << 24) - 2, 256, 5 * P_BYTES) == 0,
              "Q that does not fit, up to the longest sum");

template <int BN, bool QROW, bool SWAP, bool SHARE, typename TOut>
int launch(const CUtensorMap &mp, const CUtensorMap &mq, const CUtensorMap &mc, Params p, cudaStream_t st) {
    using S = Tile<BN, QROW>;
    static PerDeviceOnce attr_done;
    const cudaError_t e = attr_done.run([] {
        cudaFuncAttributes a;
        const cudaError_t r = cudaFuncGetAttributes(&a, fp8_matmul_kernel<BN, QROW, SWAP, SHARE, TOut>);
        if (r != cudaSuccess) return r;
        // a register split above what the launch allocates would wait forever
        if (S::kSplitRegs && (a.numRegs > kRegsScaling || a.numRegs * S::kThreads < S::kRegsNeeded))
            return cudaErrorInvalidConfiguration;
        return cudaFuncSetAttribute(fp8_matmul_kernel<BN, QROW, SWAP, SHARE, TOut>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    S::kSmem);
    });
    if (e != cudaSuccess)
        return fail(GNNAGG_ERR_CUDA, "fp8_matmul: cannot reserve %d bytes of shared memory and the registers: %s", S::kSmem,
                    cudaGetErrorString(e));
    const int grid = p.items < kNumSMs ? p.items : kNumSMs;
    // Q stays where every CTA has several tiles of one column, and all of its k-blocks and three of P's fit
    const int beside = stages_beside_q(p.kblocks, BN, S::kStages * S::kStageBytes);
    p.keep_q = p.tiles_q == 1 && p.splits == 1 && p.tiles_p > grid && beside > 0;
    p.stages = p.keep_q ? beside : S::kStages;
    if (SWAP && SHARE) {  // one item per CTA: all of them are resident
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)p.items);
        cfg.blockDim = dim3(S::kThreads);
        cfg.dynamicSmemBytes = S::kSmem;
        cfg.stream = st;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = (unsigned)p.splits;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        const cudaError_t le = cudaLaunchKernelEx(&cfg, fp8_matmul_kernel<BN, QROW, SWAP, SHARE, TOut>, mp, mq, mc, p);
        if (le != cudaSuccess) return fail(GNNAGG_ERR_CUDA, "fp8_matmul_kernel: %s", cudaGetErrorString(le));
    } else {
        fp8_matmul_kernel<BN, QROW, SWAP, SHARE, TOut><<<grid, S::kThreads, S::kSmem, st>>>(mp, mq, mc, p);
    }
    return check_launch("fp8_matmul_kernel");
}

template <bool QROW, typename TOut>
int launch_tile(const Plan &plan, const CUtensorMap &mp, const CUtensorMap &mq, const CUtensorMap &mc, const Params &p,
                cudaStream_t st) {
    if (plan.join)
        return plan.bn == 16   ? launch<16, QROW, true, true, TOut>(mp, mq, mc, p, st)
               : plan.bn == 32 ? launch<32, QROW, true, true, TOut>(mp, mq, mc, p, st)
                               : launch<64, QROW, true, true, TOut>(mp, mq, mc, p, st);
    if (plan.swap)
        return plan.bn == 16   ? launch<16, QROW, true, false, TOut>(mp, mq, mc, p, st)
               : plan.bn == 32 ? launch<32, QROW, true, false, TOut>(mp, mq, mc, p, st)
                               : launch<64, QROW, true, false, TOut>(mp, mq, mc, p, st);
    if (plan.tail > 0)
        return plan.bn == 128 ? launch<128, QROW, false, true, TOut>(mp, mq, mc, p, st)
                              : launch<256, QROW, false, true, TOut>(mp, mq, mc, p, st);
    return plan.bn == 16    ? launch<16, QROW, false, false, TOut>(mp, mq, mc, p, st)
           : plan.bn == 32  ? launch<32, QROW, false, false, TOut>(mp, mq, mc, p, st)
           : plan.bn == 64  ? launch<64, QROW, false, false, TOut>(mp, mq, mc, p, st)
           : plan.bn == 128 ? launch<128, QROW, false, false, TOut>(mp, mq, mc, p, st)
                            : launch<256, QROW, false, false, TOut>(mp, mq, mc, p, st);
}

template <typename TOut>
int launch_out(bool qrow, const Plan &plan, const CUtensorMap &mp, const CUtensorMap &mq, const CUtensorMap &mc,
               const Params &p, cudaStream_t st) {
    return qrow ? launch_tile<true, TOut>(plan, mp, mq, mc, p, st) : launch_tile<false, TOut>(plan, mp, mq, mc, p, st);
}

template <typename TOut>
int join(const Plan &plan, const float *partial, int splits, int64_t M, int64_t N, const void *bias,
         int bias_type, int accumulate, void *C, int64_t ldc, cudaStream_t st) {
    const int64_t want = div_up(M * (plan.ldp / 4), 256);
    const int64_t cap = (int64_t)kNumSMs * 8;
    fp8_join_kernel<TOut><<<(unsigned)(want < cap ? want : cap), 256, 0, st>>>(
        partial, splits, M * plan.ldp, plan.ldp, M, N, bias, bias_type, accumulate, static_cast<TOut *>(C), ldc);
    return check_launch("fp8_join_kernel");
}

int join_out(int type, const Plan &plan, const float *partial, int splits, int64_t M, int64_t N, const void *bias,
             int bias_type, int accumulate, void *C, int64_t ldc, cudaStream_t st) {
    return type == kTypeF32    ? join<float>(plan, partial, splits, M, N, bias, bias_type, accumulate, C, ldc, st)
           : type == kTypeBf16 ? join<__nv_bfloat16>(plan, partial, splits, M, N, bias, bias_type, accumulate, C, ldc, st)
                               : join<__half>(plan, partial, splits, M, N, bias, bias_type, accumulate, C, ldc, st);
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
                                 const void *bias, int32_t bias_type, int32_t accumulate, void *C, int64_t ldc, int32_t out_type,
                                 void *workspace, size_t workspace_bytes, void *stream) {
    if (M < 0 || N < 0 || K < 0 || (accumulate != 0 && accumulate != 1))
        return fail(GNNAGG_ERR_ARG, "fp8_matmul: negative size or bad accumulate flag");
    if ((a_block != 1 && a_block != 128) || (b_block != 1 && b_block != 128))
        return fail(GNNAGG_ERR_ARG, "fp8_matmul: a scale covers 1 or 128 rows");
    if (bias != nullptr && type_size(bias_type) == 0)
        return fail(GNNAGG_ERR_ARG, "fp8_matmul: unknown bias type %d", bias_type);
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
    if (K == 0) return join_out(out_type, plan, nullptr, 0, M, N, bias, bias_type, accumulate, C, ldc, st);
    const bool split = plan.splits > 1 && !plan.join;  // through the workspace
    if (plan.bytes() > 0 && (workspace == nullptr || !aligned16(workspace) || workspace_bytes < plan.bytes()))
        return fail(GNNAGG_ERR_SCRATCH, "fp8_matmul: workspace too small or misaligned (need %zu bytes)", plan.bytes());
    if ((int64_t)plan.tiles_p * plan.tiles_q * plan.splits > 0x7FFFFFFF)
        return fail(GNNAGG_ERR_UNSUPPORTED, "fp8_matmul: too many tiles");

    const Scales za{sa, sa_stride, sa_stride_k}, zb{sb, sb_stride, sb_stride_k};
    CUtensorMap map_p, map_q;
    int rc = plan.swap ? make_map_f8(&map_p, B, N, K, ldb, BP) : make_map_f8(&map_p, A, M, K, lda, BP);
    if (rc == GNNAGG_OK)
        rc = plan.swap ? make_map_f8(&map_q, A, M, K, lda, plan.bn) : make_map_f8(&map_q, B, N, K, ldb, plan.bn);
    if (rc != GNNAGG_OK) return rc;
    const int type = split ? (int)kTypeF32 : out_type;
    const int64_t ldo = split ? plan.ldp : ldc;
    void *out = split ? workspace : C;
    const bool vec_out = aligned16(out) && (ldo * type_size(type)) % 16 == 0 && !(accumulate && !split);
    // wide tiles leave by TMA where it can address the rows; it ends a row on 16 bytes, so a row that ends between them
    // would have what lies behind it written over (padding in the workspace, the caller's own in an output)
    const bool tma_out = vec_out && !plan.swap && plan.bn >= 128 && (split || N * type_size(type) % 16 == 0);
    CUtensorMap map_c = map_p;  // not used without tma_out
    if (tma_out) rc = make_map_out(&map_c, out, type, plan.splits, M, N, ldo);
    if (rc != GNNAGG_OK) return rc;

    Params p;
    p.C = out;
    p.bias = split ? nullptr : bias;
    p.bias_type = bias_type;
    p.sp = plan.swap ? zb : za;
    p.sq = plan.swap ? za : zb;
    p.rows_p = plan.swap ? N : M;
    p.rows_q = plan.swap ? M : N;
    p.ldc = ldo;
    p.split_stride = split ? M * plan.ldp : 0;
    p.p_block = (plan.swap ? b_block : a_block) == 128;
    p.kblocks = plan.kblocks;
    p.splits = plan.splits;
    p.kb_per_split = plan.kb_per_split;
    p.tiles_p = plan.tiles_p;
    p.tiles_q = plan.tiles_q;
    p.items = plan.tiles_p * plan.tiles_q * plan.splits;
    p.tail = plan.tail, p.per = plan.per, p.full = p.items - plan.tail;
    p.counts = static_cast<int *>(workspace);
    p.parts = reinterpret_cast<float *>(static_cast<uint8_t *>(workspace) + (plan.tail > 0 ? kCountBytes : 0));
    if (plan.tail > 0) {
        p.items = p.full + 2 * kNumSMs;
        const cudaError_t e = cudaMemsetAsync(p.counts, 0, kCountBytes, st);
        if (e != cudaSuccess) return fail(GNNAGG_ERR_CUDA, "fp8_matmul: %s", cudaGetErrorString(e));
    }
    p.accumulate = split ? 0 : accumulate;
    p.vec_out = vec_out;
    p.tma_out = tma_out;
    p.wait_ns = g_stall.wait_ns;
    p.tx_excess = g_stall.tx_excess;
    const bool qrow = (plan.swap ? a_block : b_block) == 1;
    rc = type == kTypeF32    ? launch_out<float>(qrow, plan, map_p, map_q, map_c, p, st)
         : type == kTypeBf16 ? launch_out<__nv_bfloat16>(qrow, plan, map_p, map_q, map_c, p, st)
                             : launch_out<__half>(qrow, plan, map_p, map_q, map_c, p, st);
    if (rc != GNNAGG_OK || !split) return rc;
    return join_out(out_type, plan, static_cast<const float *>(workspace), plan.splits, M, N, bias, bias_type, accumulate, C, ldc, st);
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
