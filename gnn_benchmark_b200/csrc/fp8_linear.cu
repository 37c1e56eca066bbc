// The 8-bit linear layer as one call each way: quantise both operands (each read once, in both orientations where
// the backward needs the other), multiply, and keep the backward's operands as codes.  No kernels of its own but the
// join of the bias gradient's column sums.
#include "lowp.cuh"

namespace gnnagg {
namespace {

inline int64_t up(int64_t v, int64_t m) { return div_up(v, m) * m; }

// A piece of a buffer: codes [rows][ld], scales [groups][lds] (one per row and group, or per 128 x 128 block).
struct Piece {
    int64_t rows, cols, ld, lds, groups;
    uint8_t *codes;
    float *scales;
};

// Lays pieces one behind the other, each part on 256 bytes; `base` null: only counts.
struct Layout {
    uint8_t *base;
    size_t at = 0;
    void *take(size_t bytes) {
        uint8_t *p = base == nullptr ? nullptr : base + at;
        at += (bytes + 255) / 256 * 256;
        return p;
    }
    Piece piece(int64_t rows, int64_t cols, bool block) {
        Piece p;
        p.rows = rows, p.cols = cols;
        p.ld = up(cols, 16);
        p.lds = up(block ? div_up(rows, 128) : rows, 4);  // 16-byte rows of scales
        p.groups = div_up(cols, 128);
        p.codes = static_cast<uint8_t *>(take((size_t)(p.rows * p.ld)));
        p.scales = static_cast<float *>(take((size_t)(p.lds * p.groups) * sizeof(float)));
        return p;
    }
};

struct Kept {
    Piece xt, wt;  // x^T in blocks of 1 x 128, w^T of 128 x 128
    size_t bytes;
    Kept(void *base, int64_t M, int64_t N, int64_t K, bool need_x, bool need_w) : xt(), wt() {
        Layout l{static_cast<uint8_t *>(base)};
        if (need_w) xt = l.piece(K, M, false);
        if (need_x) wt = l.piece(K, N, true);
        bytes = l.at;
    }
};

struct Forward {
    Piece x, w;
    void *ws;
    size_t ws_bytes, bytes;
    Forward(void *base, int64_t M, int64_t N, int64_t K) {
        Layout l{static_cast<uint8_t *>(base)};
        x = l.piece(M, K, false);
        w = l.piece(N, K, true);
        ws_bytes = gnnagg_fp8_matmul_workspace_bytes(M, N, K);
        ws = l.take(ws_bytes);
        bytes = l.at;
    }
};

struct Backward {
    Piece g, gt;
    float *sums;
    void *ws;
    size_t ws_bytes, bytes;
    Backward(void *base, int64_t M, int64_t N, int64_t K) {
        Layout l{static_cast<uint8_t *>(base)};
        g = l.piece(M, N, false);
        gt = l.piece(N, M, false);
        sums = static_cast<float *>(l.take((size_t)(div_up(M, 128) * N) * sizeof(float)));
        const size_t a = gnnagg_fp8_matmul_workspace_bytes(M, K, N), b = gnnagg_fp8_matmul_workspace_bytes(N, K, M);
        ws_bytes = a > b ? a : b;  // the two products follow one another
        ws = l.take(ws_bytes);
        bytes = l.at;
    }
};

int multiply(const Piece &a, bool a_block, const Piece &b, bool b_block, int64_t M, int64_t N, int64_t K, const void *bias,
             int bias_type, void *out, int out_type, void *ws, size_t ws_bytes, void *stream) {
    return gnnagg_fp8_matmul(a.codes, a.ld, a.scales, 1, a.lds, a_block ? 128 : 1, b.codes, b.ld, b.scales, 1, b.lds,
                             b_block ? 128 : 1, M, N, K, bias, bias_type, 0, out, N, out_type, ws, ws_bytes, stream);
}

int check(const char *what, int64_t M, int64_t N, int64_t K, const void *kept, size_t kept_bytes, size_t kept_need,
          const void *scratch, size_t scratch_bytes, size_t scratch_need) {
    if (M > 0x7FFFFFFF - 256 || N > 0x7FFFFFFF - 256 || K > 0x7FFFFFFF - 256)
        return fail(GNNAGG_ERR_UNSUPPORTED, "%s: a size exceeds 2^31", what);
    if (kept_need > 0 && (kept == nullptr || !aligned16(kept) || kept_bytes < kept_need))
        return fail(GNNAGG_ERR_SCRATCH, "%s: the buffer that is kept is too small or misaligned (need %zu bytes)", what, kept_need);
    if (scratch_need > 0 && (scratch == nullptr || !aligned16(scratch) || scratch_bytes < scratch_need))
        return fail(GNNAGG_ERR_SCRATCH, "%s: scratch too small or misaligned (need %zu bytes)", what, scratch_need);
    return GNNAGG_OK;
}

template <typename T>
int join_sums(const float *sums, int64_t blocks, int64_t N, void *gb, cudaStream_t st) {
    column_sum_kernel<T><<<(unsigned)div_up(N, 32), dim3(32, 16), 0, st>>>(sums, blocks, N, static_cast<T *>(gb));
    return check_launch("column_sum_kernel");
}

}  // namespace
}  // namespace gnnagg

using namespace gnnagg;

extern "C" size_t gnnagg_fp8_linear_kept_bytes(int64_t M, int64_t N, int64_t K, int32_t need_x, int32_t need_w) {
    if (M < 0 || N < 0 || K < 0) return 0;
    return Kept(nullptr, M, N, K, need_x != 0, need_w != 0).bytes;
}

extern "C" size_t gnnagg_fp8_linear_scratch_bytes(int64_t M, int64_t N, int64_t K, int32_t backward) {
    if (M < 0 || N < 0 || K < 0) return 0;
    return backward ? Backward(nullptr, M, N, K).bytes : Forward(nullptr, M, N, K).bytes;
}

extern "C" int gnnagg_fp8_linear_fwd(const void *x, int64_t ldx, int32_t x_type, const void *w, int64_t ldw, int32_t w_type,
                                     const void *bias, int32_t bias_type, int64_t M, int64_t N, int64_t K, void *y,
                                     int32_t y_type, int32_t need_x, int32_t need_w, void *kept, size_t kept_bytes,
                                     void *scratch, size_t scratch_bytes, void *stream) {
    if (M < 0 || N < 0 || K < 0) return fail(GNNAGG_ERR_ARG, "fp8_linear_fwd: negative size");
    const Kept k(kept, M, N, K, need_x != 0, need_w != 0);
    const Forward f(scratch, M, N, K);
    int rc = check("fp8_linear_fwd", M, N, K, kept, kept_bytes, k.bytes, scratch, scratch_bytes, f.bytes);
    if (rc != GNNAGG_OK) return rc;
    rc = gnnagg_fp8_quantize(x, ldx, M, K, x_type, 1, f.x.codes, f.x.ld, f.x.scales, f.x.lds, k.xt.codes, k.xt.ld, k.xt.scales,
                             k.xt.lds, nullptr, stream);
    if (rc == GNNAGG_OK)
        rc = gnnagg_fp8_quantize(w, ldw, N, K, w_type, 128, f.w.codes, f.w.ld, f.w.scales, f.w.lds, k.wt.codes, k.wt.ld,
                                 k.wt.scales, k.wt.lds, nullptr, stream);
    if (rc != GNNAGG_OK) return rc;
    return multiply(f.x, false, f.w, true, M, N, K, bias, bias_type, y, y_type, f.ws, f.ws_bytes, stream);
}

extern "C" int gnnagg_fp8_linear_bwd(const void *g, int64_t ldg, int32_t g_type, int64_t M, int64_t N, int64_t K,
                                     int32_t need_x, int32_t need_w, const void *kept, size_t kept_bytes, void *gx,
                                     int32_t x_type, void *gw, int32_t w_type, void *gb, int32_t b_type, void *scratch,
                                     size_t scratch_bytes, void *stream) {
    if (M < 0 || N < 0 || K < 0) return fail(GNNAGG_ERR_ARG, "fp8_linear_bwd: negative size");
    if ((gx != nullptr && !need_x) || (gw != nullptr && !need_w))
        return fail(GNNAGG_ERR_ARG, "fp8_linear_bwd: a gradient whose operand was not kept");
    if (gb != nullptr && type_size(b_type) == 0) return fail(GNNAGG_ERR_ARG, "fp8_linear_bwd: unknown bias type %d", b_type);
    const Kept k(const_cast<void *>(kept), M, N, K, need_x != 0, need_w != 0);
    const Backward b(scratch, M, N, K);
    int rc = check("fp8_linear_bwd", M, N, K, kept, kept_bytes, k.bytes, scratch, scratch_bytes, b.bytes);
    if (rc != GNNAGG_OK) return rc;
    const bool rows = gx != nullptr || gw == nullptr;  // for the sums alone the codes are made and not used
    if (gx == nullptr && gw == nullptr && gb == nullptr) return GNNAGG_OK;
    rc = gnnagg_fp8_quantize(g, ldg, M, N, g_type, 1, rows ? b.g.codes : nullptr, b.g.ld, b.g.scales, b.g.lds,
                             gw != nullptr ? b.gt.codes : nullptr, b.gt.ld, b.gt.scales, b.gt.lds,
                             gb != nullptr ? b.sums : nullptr, stream);
    if (rc != GNNAGG_OK) return rc;
    if (gb != nullptr && N > 0) {
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        const int64_t blocks = div_up(M, 128);
        rc = b_type == kTypeF32    ? join_sums<float>(b.sums, blocks, N, gb, st)
             : b_type == kTypeBf16 ? join_sums<__nv_bfloat16>(b.sums, blocks, N, gb, st)
                                   : join_sums<__half>(b.sums, blocks, N, gb, st);
        if (rc != GNNAGG_OK) return rc;
    }
    if (gx != nullptr)
        rc = multiply(b.g, false, k.wt, true, M, K, N, nullptr, 0, gx, x_type, b.ws, b.ws_bytes, stream);
    if (rc == GNNAGG_OK && gw != nullptr)
        rc = multiply(b.gt, false, k.xt, false, N, K, M, nullptr, 0, gw, w_type, b.ws, b.ws_bytes, stream);
    return rc;
}
