// e4m3 codes and block scales of a matrix, along its rows, along its columns (transposed codes), or both from one
// read: the operands of the 8-bit product.
//
// A block of the grid holds a 128 x 128 tile in registers, as it lies in memory: 256 threads, each V neighbouring
// columns (16 bytes of input) of a run of neighbouring rows.  Largest magnitudes are maxima of bit patterns, by shuffles along a row and
// by shared-memory atomics along columns (a maximum does not depend on the order).  Transposed codes go through a
// 16 KB shared tile: 8 rows of a column are one 8-byte piece, at piece index XOR (column / V) so that a warp's
// stores meet different banks, and leave as 16-byte stores.
// Bound by memory: per element its bytes in and one byte out for each orientation.
#include "lowp.cuh"

namespace gnnagg {
namespace {

constexpr int kTile = 128;
constexpr int kThreads = 256;

struct QuantParams {
    const void *x;
    int64_t ldx, rows, cols;
    uint8_t *codes, *codes_t;      // [rows][ldc], [cols][ldt]
    int64_t ldc, ldt;
    float *scales, *scales_t;      // scale of (row or row block i, column group j) at i + j * lds, likewise for the
    int64_t lds, lds_t;            // transpose
    float *column_sums;            // [row blocks][cols] sums of x over a tile's rows, or null
};

// BLOCK: one scale for the whole tile; otherwise one per row (ROWS) and one per column (COLS) of the tile.
template <typename T, bool VEC, bool BLOCK, bool ROWS, bool COLS>
__global__ void __launch_bounds__(kThreads) fp8_quantize_kernel(const QuantParams p) {
    constexpr int V = Vec<T>::N;
    constexpr int kLanes = kTile / V;             // threads along a row: 16 or 32
    constexpr int kRun = kTile * kLanes / kThreads;  // neighbouring rows of a thread: 8 or 16
    __shared__ uint32_t top[kTile];
    __shared__ __align__(16) uint8_t tile[COLS ? kTile * kTile : 16];
    const int ch = threadIdx.x % kLanes, rg = threadIdx.x / kLanes;
    const int64_t row0 = (int64_t)blockIdx.x * kTile, col0 = (int64_t)blockIdx.y * kTile;
    const int64_t col = col0 + ch * V;
    const int valid = (int)(p.cols - col < V ? p.cols - col : V);
    if (threadIdx.x < kTile) top[threadIdx.x] = 0;
    __syncthreads();
    uint4 raw[kRun];
    auto at = [&](int i, int e) { return to_f32(reinterpret_cast<const T *>(&raw[i])[e]); };
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
        const int64_t row = row0 + rg * kRun + i;
        raw[i] = make_uint4(0, 0, 0, 0);
        if (row < p.rows && valid > 0) raw[i] = load_raw<T, VEC>(static_cast<const T *>(p.x) + row * p.ldx + col, valid);
    }
    if (p.column_sums != nullptr) {
        constexpr int kRuns = kTile / kRun;
        __shared__ float red[kRuns][kTile];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            float s = at(0, e);
#pragma unroll
            for (int i = 1; i < kRun; ++i) s += at(i, e);
            red[rg][ch * V + e] = s;
        }
        __syncthreads();
        if (threadIdx.x < kTile && col0 + threadIdx.x < p.cols) {
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < kRuns; ++i) s += red[i][threadIdx.x];
            p.column_sums[blockIdx.x * p.cols + col0 + threadIdx.x] = s;
        }
    }
    uint32_t whole = 0;
    if (BLOCK) {
#pragma unroll
        for (int i = 0; i < kRun; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) whole = max(whole, abs_bits(at(i, e)));
        whole = __reduce_max_sync(kFullMask, whole);
        if ((threadIdx.x & 31) == 0) atomicMax(&top[0], whole);
        __syncthreads();
        whole = top[0];
        if (threadIdx.x == 0) {
            const float s = block_scale(block_amax(whole));
            if (ROWS) p.scales[blockIdx.x + blockIdx.y * p.lds] = s;
            if (COLS) p.scales_t[blockIdx.y + blockIdx.x * p.lds_t] = s;
        }
    }
    if (ROWS) {
#pragma unroll
        for (int i = 0; i < kRun; ++i) {
            const int64_t row = row0 + rg * kRun + i;
            uint32_t m = whole;
            if (!BLOCK) {
#pragma unroll
                for (int e = 0; e < V; ++e) m = max(m, abs_bits(at(i, e)));
#pragma unroll
                for (int off = kLanes / 2; off > 0; off >>= 1) m = max(m, __shfl_xor_sync(kFullMask, m, off));
            }
            const float a = block_amax(m), f = block_factor(a);
            if (row < p.rows && valid > 0) {
                uint32_t c[V / 4];
#pragma unroll
                for (int k = 0; k < V / 4; ++k)
                    c[k] = e4m3x4(__fmul_rn(at(i, 4 * k), f), __fmul_rn(at(i, 4 * k + 1), f), __fmul_rn(at(i, 4 * k + 2), f),
                                  __fmul_rn(at(i, 4 * k + 3), f));
                // code rows are padded to 16 bytes, so a whole chunk always fits
                uint32_t *dst = reinterpret_cast<uint32_t *>(p.codes + row * p.ldc + col);
                if (V == 8)
                    *reinterpret_cast<uint2 *>(dst) = make_uint2(c[0], c[V / 4 - 1]);
                else
                    *dst = c[0];
                if (!BLOCK && ch == 0) p.scales[row + blockIdx.y * p.lds] = block_scale(a);
            }
        }
    }
    if (COLS) {
        if (!BLOCK) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                uint32_t m = 0;
#pragma unroll
                for (int i = 0; i < kRun; ++i) m = max(m, abs_bits(at(i, e)));
                if (V == 8) m = max(m, __shfl_xor_sync(kFullMask, m, 16));  // the warp's other run of rows
                if (V == 4 || (threadIdx.x & 16) == 0) atomicMax(&top[ch * V + e], m);
            }
            __syncthreads();
        }
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float f = block_factor(block_amax(BLOCK ? whole : top[ch * V + e]));
#pragma unroll
            for (int k = 0; k < kRun / 8; ++k) {
                uint2 u;
                u.x = e4m3x4(__fmul_rn(at(8 * k, e), f), __fmul_rn(at(8 * k + 1, e), f), __fmul_rn(at(8 * k + 2, e), f),
                             __fmul_rn(at(8 * k + 3, e), f));
                u.y = e4m3x4(__fmul_rn(at(8 * k + 4, e), f), __fmul_rn(at(8 * k + 5, e), f), __fmul_rn(at(8 * k + 6, e), f),
                             __fmul_rn(at(8 * k + 7, e), f));
                const int piece = (rg * (kRun / 8) + k) ^ (ch & 15);
                *reinterpret_cast<uint2 *>(tile + (ch * V + e) * kTile + piece * 8) = u;
            }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < kTile * 8; i += kThreads) {
            const int c = i >> 3, j = i & 7, key = (c / V) & 15;
            const int64_t out = col0 + c, r = row0 + 16 * j;
            if (out < p.cols && r < p.rows) {
                const uint2 a = *reinterpret_cast<const uint2 *>(tile + c * kTile + ((2 * j) ^ key) * 8);
                const uint2 b = *reinterpret_cast<const uint2 *>(tile + c * kTile + ((2 * j + 1) ^ key) * 8);
                *reinterpret_cast<uint4 *>(p.codes_t + out * p.ldt + r) = make_uint4(a.x, a.y, b.x, b.y);
            }
        }
        if (!BLOCK && threadIdx.x < kTile && col0 + threadIdx.x < p.cols)
            p.scales_t[col0 + threadIdx.x + blockIdx.x * p.lds_t] = block_scale(block_amax(top[threadIdx.x]));
    }
}

template <typename T, bool VEC, bool BLOCK>
int launch(const QuantParams &p, cudaStream_t st) {
    const dim3 grid((unsigned)div_up(p.rows, kTile), (unsigned)div_up(p.cols, kTile));
    if (p.codes != nullptr && p.codes_t != nullptr)
        fp8_quantize_kernel<T, VEC, BLOCK, true, true><<<grid, kThreads, 0, st>>>(p);
    else if (p.codes != nullptr)
        fp8_quantize_kernel<T, VEC, BLOCK, true, false><<<grid, kThreads, 0, st>>>(p);
    else
        fp8_quantize_kernel<T, VEC, BLOCK, false, true><<<grid, kThreads, 0, st>>>(p);
    return check_launch("fp8_quantize_kernel");
}

template <typename T>
int launch_type(const QuantParams &p, bool block, cudaStream_t st) {
    const bool vec = aligned16(p.x) && (p.ldx * sizeof(T)) % 16 == 0 && p.cols % Vec<T>::N == 0;
    if (block) return vec ? launch<T, true, true>(p, st) : launch<T, false, true>(p, st);
    return vec ? launch<T, true, false>(p, st) : launch<T, false, false>(p, st);
}

}  // namespace
}  // namespace gnnagg

using namespace gnnagg;

extern "C" int gnnagg_fp8_quantize(const void *x, int64_t ldx, int64_t rows, int64_t cols, int32_t type, int32_t block_rows,
                                   uint8_t *codes, int64_t ldc, float *scales, int64_t lds, uint8_t *codes_t, int64_t ldt,
                                   float *scales_t, int64_t lds_t, float *column_sums, void *stream) {
    if (rows < 0 || cols < 0) return fail(GNNAGG_ERR_ARG, "fp8_quantize: negative size");
    if (type_size(type) == 0) return fail(GNNAGG_ERR_ARG, "fp8_quantize: unknown element type %d", type);
    if (block_rows != 1 && block_rows != 128) return fail(GNNAGG_ERR_ARG, "fp8_quantize: blocks are 1 x 128 or 128 x 128");
    if (rows == 0 || cols == 0) return GNNAGG_OK;
    if (codes == nullptr && codes_t == nullptr) return fail(GNNAGG_ERR_ARG, "fp8_quantize: no output");
    if (x == nullptr || (codes != nullptr && scales == nullptr) || (codes_t != nullptr && scales_t == nullptr))
        return fail(GNNAGG_ERR_ARG, "fp8_quantize: null pointer");
    if (rows > 0x7FFFFFFF - 256 || cols > (int64_t)65535 * kTile)
        return fail(GNNAGG_ERR_UNSUPPORTED, "fp8_quantize: more than 2^31 rows or %d columns", 65535 * kTile);
    if (ldx < cols || (codes != nullptr && ldc < cols) || (codes_t != nullptr && ldt < rows))
        return fail(GNNAGG_ERR_ARG, "fp8_quantize: a stride is smaller than its rows");
    if ((codes != nullptr && (!aligned16(codes) || ldc % 16 != 0)) ||
        (codes_t != nullptr && (!aligned16(codes_t) || ldt % 16 != 0)))
        return fail(GNNAGG_ERR_UNSUPPORTED, "fp8_quantize: code rows must start on 16 bytes");
    const int64_t r = block_rows == 1 ? rows : div_up(rows, kTile), c = block_rows == 1 ? cols : div_up(cols, kTile);
    if ((codes != nullptr && lds < r) || (codes_t != nullptr && lds_t < c))
        return fail(GNNAGG_ERR_ARG, "fp8_quantize: a stride of the scales is too small");
    const QuantParams p{x, ldx, rows, cols, codes, codes_t, ldc, ldt, scales, scales_t, lds, lds_t, column_sums};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool block = block_rows == 128;
    return type == kTypeF32    ? launch_type<float>(p, block, st)
           : type == kTypeBf16 ? launch_type<__nv_bfloat16>(p, block, st)
                               : launch_type<__half>(p, block, st);
}
