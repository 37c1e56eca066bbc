// e4m3 codes and block scales of a matrix, along its rows, along its columns (transposed codes), or both from one
// read: the operands of the 8-bit product.
//
// A block of the grid holds a 128 x 128 tile in registers, as it lies in memory: 256 threads, each V neighbouring
// columns (16 bytes of input) of a run of neighbouring rows.  Largest magnitudes are maxima of bit patterns, two 16-bit
// elements an instruction; a run's rows are reduced across their 16 (32) threads by halving exchanges, so that a row's
// reciprocal is taken once, and columns through a shared table of the runs' maxima.  Transposed codes go through a 16 KB
// shared tile: 8 rows of a column are one 8-byte piece, at piece index XOR (column / V) so that a warp's stores meet
// different banks, and leave as 16-byte stores.
// Its floor is memory: per element its bytes in and one byte out for each orientation.  16384 x 8192 bf16 in both
// orientations take 106 us, 5.1 TB/s, at 16 instructions an element (195 us with a shuffle reduction per row and a reciprocal
// per thread and column); the schedulers issue in 62 % of the cycles, and the 24 warps that the registers allow an SM wait
// for loads in most of the others.  fp32 158 us, 5.1 TB/s.  Rows off 16 bytes are loaded element by element: 612500 x 100 bf16
// take 117 us, 2.1 TB/s, and 30000 x 1501 78 us.
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
    uint32_t col_tiles;
    float *column_sums;            // [row blocks][cols] sums of x over a tile's rows, or null
};

// Magnitudes of a 32-bit word's elements (one fp32, or two 16-bit ones side by side) and their maxima, as bits.
template <typename T>
__device__ __forceinline__ uint32_t word_abs(uint32_t w) {
    return sizeof(T) == 4 ? w & 0x7FFFFFFFu : w & 0x7FFF7FFFu;
}
template <typename T>
__device__ __forceinline__ uint32_t word_max(uint32_t a, uint32_t b) {
    return sizeof(T) == 4 ? max(a, b) : __vmaxu2(a, b);
}
// A word's larger magnitude as fp32 bits.
template <typename T>
__device__ __forceinline__ uint32_t word_amax(uint32_t w) {
    if (sizeof(T) == 4) return w;
    const uint16_t m = (uint16_t)max(w & 0xFFFFu, w >> 16);
    return __float_as_uint(to_f32(*reinterpret_cast<const T *>(&m)));
}

// BLOCK: one scale for the whole tile; otherwise one per row (ROWS) and one per column (COLS) of the tile.
template <typename T, bool VEC, bool BLOCK, bool ROWS, bool COLS>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 2 ? 3 : 2) fp8_quantize_kernel(const QuantParams p) {
    constexpr int V = Vec<T>::N;
    constexpr int kLanes = kTile / V;                // threads along a row: 16 or 32
    constexpr int kRun = kTile * kLanes / kThreads;  // neighbouring rows of a thread: 8 or 16
    constexpr int kRuns = kTile / kRun;
    __shared__ __align__(16) uint8_t tile[COLS ? kTile * kTile : 16];
    __shared__ __align__(16) float factors[COLS && !BLOCK ? kTile : 4];
    __shared__ uint32_t top;
    const int ch = threadIdx.x % kLanes, rg = threadIdx.x / kLanes;
    // neighbouring blocks read neighbouring columns of the same rows
    const int64_t rt = blockIdx.x / p.col_tiles, ct = blockIdx.x - rt * p.col_tiles;
    const int64_t row0 = rt * kTile, col0 = ct * kTile;
    const int64_t col = col0 + ch * V;
    const int valid = (int)(p.cols - col < V ? p.cols - col : V);
    uint4 raw[kRun];
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
        const int64_t row = row0 + rg * kRun + i;
        raw[i] = make_uint4(0, 0, 0, 0);
        if (row < p.rows && valid > 0) raw[i] = load_raw<T, VEC>(static_cast<const T *>(p.x) + row * p.ldx + col, valid);
    }
    auto at = [&raw](int i, int e) {
        const uint32_t words[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
        if (sizeof(T) == 4) return __uint_as_float(words[e]);
        const uint32_t w = words[e / 2 % 4];
        if (std::is_same<T, __nv_bfloat16>::value) return __uint_as_float(e % 2 ? w & 0xFFFF0000u : w << 16);
        const uint16_t h = (uint16_t)(e % 2 ? w >> 16 : w);
        return to_f32(*reinterpret_cast<const T *>(&h));
    };
    if (BLOCK) {
        if (threadIdx.x == 0) top = 0;
        __syncthreads();
    }
    if (p.column_sums != nullptr) {
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
            p.column_sums[rt * p.cols + col0 + threadIdx.x] = s;
        }
    }
    // maxima of the thread's rows (m) and columns (cm)
    uint32_t m[kRun], cm[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
        const uint32_t w[4] = {word_abs<T>(raw[i].x), word_abs<T>(raw[i].y), word_abs<T>(raw[i].z), word_abs<T>(raw[i].w)};
        m[i] = word_max<T>(word_max<T>(w[0], w[1]), word_max<T>(w[2], w[3]));
        if (COLS && !BLOCK) {
#pragma unroll
            for (int k = 0; k < 4; ++k) cm[k] = word_max<T>(cm[k], w[k]);
        }
    }
    float whole = 0.0f;  // BLOCK: the tile's factor
    if (BLOCK) {
        uint32_t a = 0;
#pragma unroll
        for (int i = 0; i < kRun; ++i) a = word_max<T>(a, m[i]);
        a = __reduce_max_sync(kFullMask, word_amax<T>(a));
        if ((threadIdx.x & 31) == 0) atomicMax(&top, a);
        __syncthreads();
        const float amax = block_amax(top);
        whole = block_factor(amax);
        if (threadIdx.x == 0) {
            if (ROWS) p.scales[rt + ct * p.lds] = block_scale(amax);
            if (COLS) p.scales_t[ct + rt * p.lds_t] = block_scale(amax);
        }
    }
    if (COLS && !BLOCK) {
        // the runs' column maxima side by side (in the tile's memory), then one thread a column
        uint32_t *table = reinterpret_cast<uint32_t *>(tile);  // [kRuns][kTile / elements per word]
        *reinterpret_cast<uint4 *>(table + rg * kLanes * 4 + ch * 4) = make_uint4(cm[0], cm[1], cm[2], cm[3]);
        __syncthreads();
        if (threadIdx.x < kTile) {
            const T *column = reinterpret_cast<const T *>(tile) + threadIdx.x;
            uint32_t a = 0;
#pragma unroll
            for (int i = 0; i < kRuns; ++i) a = max(a, __float_as_uint(to_f32(column[i * kTile])));
            const float amax = block_amax(a);
            factors[threadIdx.x] = block_factor(amax);
            if (col0 + threadIdx.x < p.cols) p.scales_t[col0 + threadIdx.x + rt * p.lds_t] = block_scale(amax);
        }
        __syncthreads();
    }
    if (ROWS) {
        float f = whole;
        if (!BLOCK) {
            // halving exchange: after each step a thread holds half as many rows, with twice the columns in each
#pragma unroll
            for (int n = kRun / 2, off = kLanes / 2; n > 0; n /= 2, off /= 2) {
                const bool upper = (ch & off) != 0;
#pragma unroll
                for (int k = 0; k < n; ++k) {
                    const uint32_t other = __shfl_xor_sync(kFullMask, upper ? m[k] : m[k + n], off);
                    m[k] = word_max<T>(upper ? m[k + n] : m[k], other);
                }
            }
            const uint32_t a = word_max<T>(m[0], __shfl_xor_sync(kFullMask, m[0], 1));
            const float amax = block_amax(word_amax<T>(a));  // of row ch / 2 of the run
            f = block_factor(amax);
            const int64_t row = row0 + rg * kRun + ch / 2;
            if ((ch & 1) == 0 && row < p.rows) p.scales[row + ct * p.lds] = block_scale(amax);
        }
#pragma unroll
        for (int i = 0; i < kRun; ++i) {
            const int64_t row = row0 + rg * kRun + i;
            const float fi = BLOCK ? whole : __shfl_sync(kFullMask, f, 2 * i, kLanes);
            if (row < p.rows && valid > 0) {
                uint32_t c[V / 4];
#pragma unroll
                for (int k = 0; k < V / 4; ++k)
                    c[k] = e4m3x4(__fmul_rn(at(i, 4 * k), fi), __fmul_rn(at(i, 4 * k + 1), fi), __fmul_rn(at(i, 4 * k + 2), fi),
                                  __fmul_rn(at(i, 4 * k + 3), fi));
                // code rows are padded to 16 bytes, so a whole chunk always fits
                uint32_t *dst = reinterpret_cast<uint32_t *>(p.codes + row * p.ldc + col);
                if (V == 8)
                    *reinterpret_cast<uint2 *>(dst) = make_uint2(c[0], c[V / 4 - 1]);
                else
                    *dst = c[0];
            }
        }
    }
    if (COLS) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float f = BLOCK ? whole : factors[ch * V + e];
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
    }
}

template <typename T, bool VEC, bool BLOCK>
int launch(const QuantParams &p, cudaStream_t st) {
    const unsigned grid = (unsigned)(div_up(p.rows, kTile) * p.col_tiles);
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
    if (rows > 0x7FFFFFFF - 256 || cols > 0x7FFFFFFF - 256 || div_up(rows, kTile) * div_up(cols, kTile) > 0x7FFFFFFF)
        return fail(GNNAGG_ERR_UNSUPPORTED, "fp8_quantize: more than 2^31 rows, columns or tiles");
    if (ldx < cols || (codes != nullptr && ldc < cols) || (codes_t != nullptr && ldt < rows))
        return fail(GNNAGG_ERR_ARG, "fp8_quantize: a stride is smaller than its rows");
    if ((codes != nullptr && (!aligned16(codes) || ldc % 16 != 0)) ||
        (codes_t != nullptr && (!aligned16(codes_t) || ldt % 16 != 0)))
        return fail(GNNAGG_ERR_UNSUPPORTED, "fp8_quantize: code rows must start on 16 bytes");
    const int64_t r = block_rows == 1 ? rows : div_up(rows, kTile), c = block_rows == 1 ? cols : div_up(cols, kTile);
    if ((codes != nullptr && lds < r) || (codes_t != nullptr && lds_t < c))
        return fail(GNNAGG_ERR_ARG, "fp8_quantize: a stride of the scales is too small");
    const QuantParams p{x, ldx, rows, cols, codes, codes_t, ldc, ldt, scales, scales_t, lds, lds_t, (uint32_t)div_up(cols, kTile), column_sums};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool block = block_rows == 128;
    return type == kTypeF32    ? launch_type<float>(p, block, st)
           : type == kTypeBf16 ? launch_type<__nv_bfloat16>(p, block, st)
                               : launch_type<__half>(p, block, st);
}
