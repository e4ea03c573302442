// gsd_capi.cpp — the extern "C" entry points of libgsrdecoder.so (declared in
// include/gsrdecoder.h): argument checks, workspace layout and the launches.
// Nothing here allocates, throws or waits.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdarg>
#include <cstdint>
#include <cstdio>

#include "gsd_internal.h"

namespace {

thread_local char g_err[256] = "";

int fail(int code, const char* format, ...) {
    va_list args;
    va_start(args, format);
    std::vsnprintf(g_err, sizeof g_err, format, args);
    va_end(args);
    return code;
}

#define GSD_HIP(expr, what)                                                            \
    do {                                                                               \
        const hipError_t gsd_e_ = (expr);                                              \
        if (gsd_e_ != hipSuccess)                                                      \
            return fail(GSR_ERR_HIP, "%s: %s", what, hipGetErrorString(gsd_e_));       \
    } while (0)

#define GSD_REQUIRE(cond, ...)                                                   \
    do {                                                                         \
        if (!(cond)) return fail(GSR_ERR_INVALID_ARGUMENT, __VA_ARGS__);         \
    } while (0)

inline hipStream_t as_stream(void* s) { return static_cast<hipStream_t>(s); }

inline size_t align_up(size_t x) { return (x + 255) / 256 * 256; }

constexpr int64_t kMaxCount = INT64_C(1) << 31;  // of any one dimension
constexpr int64_t kMaxListSpan = (INT64_C(1) << 30) - 1024;  // elements
// a launch holds fewer than 2^32 work-items: work-groups of 256, and of 1024 (one per batch)
// where a mask is listed
constexpr int64_t kMaxGroups = (INT64_C(1) << 24) - 1;
constexpr int64_t kMaxListed = (INT64_C(1) << 22) - 1;

inline bool dtype_ok(int d) { return d == GSD_F32 || d == GSD_BF16 || d == GSD_F16; }
inline int dtype_size(int d) { return d == GSD_F32 ? 4 : 2; }

inline bool aligned(const void* p, int size) {
    return reinterpret_cast<uintptr_t>(p) % (uintptr_t)size == 0;
}

// a * b * c >= 0 stays below 2^62
inline bool product_fits(int64_t a, int64_t b, int64_t c = 1) {
    const __int128 p = (__int128)a * b * c;
    return p < ((__int128)1 << 62);
}

int check_norm(const gsd_norm* a) {
    GSD_REQUIRE(a, "null pointer");
    GSD_REQUIRE(dtype_ok(a->dtype), "unknown dtype %d", a->dtype);
    GSD_REQUIRE(a->rows >= 0 && a->rows < kMaxCount, "rows must lie in [0, 2^31)");
    GSD_REQUIRE(a->width >= 1 && a->width <= GSD_MAX_NORM_WIDTH, "width must lie in [1, %d]",
                GSD_MAX_NORM_WIDTH);
    GSD_REQUIRE(a->eps >= 0.0 && std::isfinite(a->eps), "eps must be finite and not negative");
    if (a->rows == 0) return GSR_OK;
    GSD_REQUIRE(a->x && a->weight, "null pointer");
    const int e = dtype_size(a->dtype);
    GSD_REQUIRE(aligned(a->x, e) && aligned(a->residual, e) && aligned(a->weight, e) &&
                    aligned(a->h, e) && aligned(a->rstd, 4),
                "a pointer is not aligned to its elements");
    return GSR_OK;
}

int check_attention(const gsd_attention* a) {
    GSD_REQUIRE(a, "null pointer");
    GSD_REQUIRE(a->dtype == GSD_BF16 || a->dtype == GSD_F16,
                "attention takes 16-bit types: dtype must be GSD_BF16 or GSD_F16");
    GSD_REQUIRE(a->batch >= 0 && a->batch < kMaxCount && a->queries >= 0 &&
                    a->queries < kMaxCount && a->keys >= 0 && a->keys < kMaxCount,
                "batch, queries and keys must lie in [0, 2^31)");
    GSD_REQUIRE(a->heads >= 1 && a->heads < 65536 && a->kv_heads >= 1 &&
                    a->heads % a->kv_heads == 0,
                "heads must be a positive multiple of kv_heads, below 65536");
    GSD_REQUIRE(a->dim >= 8 && a->dim <= GSD_MAX_HEAD_DIM && a->dim % 8 == 0,
                "dim must be a multiple of 8 in [8, %d]", GSD_MAX_HEAD_DIM);
    GSD_REQUIRE(a->scale > 0.0f && std::isfinite(a->scale), "scale must be positive and finite");
    GSD_REQUIRE(a->queries * (a->heads / a->kv_heads) < kMaxCount - 1024 &&
                    a->keys < kMaxCount - 1024,
                "queries x heads / kv_heads and keys must lie below 2^31 - 1024");
    GSD_REQUIRE(a->k_stride_l >= 0 && a->k_stride_l <= GSD_MAX_ATTENTION_STRIDE &&
                    a->v_stride_l >= 0 && a->v_stride_l <= GSD_MAX_ATTENTION_STRIDE,
                "the strides of keys and values must lie in [0, %d]", GSD_MAX_ATTENTION_STRIDE);
    GSD_REQUIRE(!a->key_mask || (a->keys * a->k_stride_l < kMaxListSpan &&
                                 a->keys * a->v_stride_l < kMaxListSpan),
                "with a mask, keys x their stride must lie below 2^30");
    GSD_REQUIRE(!a->key_mask || a->batch <= kMaxListed, "with a mask, batch must lie below 2^22");
    GSD_REQUIRE(product_fits(a->batch, a->queries, a->heads * a->dim * 4) &&
                    product_fits(a->batch, a->keys, a->kv_heads * a->dim * 4),
                "the tensors are too large");
    return GSR_OK;
}

int check_attention_pointers(const gsd_attention* a) {
    const bool any_q = a->batch > 0 && a->queries > 0, any_k = a->batch > 0 && a->keys > 0;
    GSD_REQUIRE(!any_q || (a->q && a->o), "null pointer");
    GSD_REQUIRE(!any_k || (a->k && a->v), "null pointer");
    GSD_REQUIRE(aligned(a->q, 2) && aligned(a->k, 2) && aligned(a->v, 2) && aligned(a->o, 2) &&
                    aligned(a->o_low, 2) && aligned(a->lse, 4) && aligned(a->key_lengths, 4),
                "a pointer is not aligned to its elements");
    return GSR_OK;
}

bool grid_fits(const gsd_attention& a, const gsd::AttentionSplit& s) {
    const __int128 p = (__int128)s.blocks * s.parts * a.batch * a.kv_heads;
    return p <= kMaxGroups;
}

size_t rows_of(const gsd_attention& a) {
    return (size_t)a.batch * (size_t)a.queries * (size_t)a.heads;
}
size_t key_rows_of(const gsd_attention& a) {
    return (size_t)a.batch * (size_t)a.keys * (size_t)a.kv_heads;
}

// A tile's rows are reached by 31-bit offsets from its first query.
bool row_strides_fit(const gsd_attention& a, int64_t l, int64_t h) {
    return l >= 0 && h >= 0 && l < (INT64_C(1) << 30) && h < (INT64_C(1) << 30) &&
           65 * l + a.heads / a.kv_heads * h + a.dim <= (INT64_C(1) << 30);
}

// a mask's valid keys, batch by batch, then their counts
size_t list_bytes(const gsd_attention& a) {
    return a.key_mask ? 4 * (size_t)a.batch * ((size_t)a.keys + 1) : 0;
}

struct ForwardLayout {
    size_t o, lse, list, end;
};
ForwardLayout forward_layout(const gsd_attention& a, const gsd::AttentionSplit& s) {
    const size_t rows = s.parts > 1 ? 4 * (size_t)s.parts * rows_of(a) : 0;
    ForwardLayout l;
    l.o = 0;
    l.lse = align_up(rows * (size_t)a.dim);
    l.list = l.lse + align_up(rows);
    l.end = l.list + align_up(list_bytes(a));
    return l;
}

struct BackwardLayout {
    size_t stat, top, value_top, dq, dk, dv, list, end;
};
BackwardLayout backward_layout(const gsd_attention& a, const gsd::AttentionSplit& sq,
                               const gsd::AttentionSplit& sk) {
    BackwardLayout l;
    size_t off = 0;
    auto take = [&](size_t bytes) {
        const size_t at = off;
        off += align_up(bytes);
        return at;
    };
    l.stat = take(8 * rows_of(a));
    const size_t tops = a.dtype == GSD_F16 ? 4 * (size_t)a.batch * (size_t)a.kv_heads : 0;
    l.top = take(2 * tops * (size_t)gsd::attention_top_blocks(a));
    l.value_top = take(tops * (size_t)gsd::attention_value_blocks(a));
    l.dq = take(sq.parts > 1 ? 4 * (size_t)sq.parts * rows_of(a) * (size_t)a.dim : 0);
    const size_t keys = sk.parts > 1 ? 4 * (size_t)sk.parts * key_rows_of(a) * (size_t)a.dim : 0;
    l.dk = take(keys);
    l.dv = take(keys);
    l.list = take(list_bytes(a));
    l.end = off;
    return l;
}

template <typename T>
T* at(void* ws, size_t off) {
    return ws ? reinterpret_cast<T*>(static_cast<char*>(ws) + off) : nullptr;
}

}  // namespace

extern "C" {

const char* gsd_last_error(void) { return g_err; }
const char* gsd_version(void) { return "gsrdecoder 1.0 (gfx950)"; }

int gsd_rotary_axes(const gsd_rotary* a, void* stream) {
    GSD_REQUIRE(a, "null pointer");
    GSD_REQUIRE(dtype_ok(a->dtype), "unknown dtype %d", a->dtype);
    GSD_REQUIRE(a->positions_type == GSD_POS_F32 || a->positions_type == GSD_POS_I32 ||
                    a->positions_type == GSD_POS_I64,
                "unknown type of positions %d", a->positions_type);
    GSD_REQUIRE(a->batch >= 0 && a->batch < kMaxCount && a->length >= 0 && a->length < kMaxCount,
                "batch and length must lie in [0, 2^31)");
    GSD_REQUIRE(a->heads >= 1 && a->heads < 65536 && a->dim >= 1 && a->dim <= 65536,
                "heads must lie in [1, 65536), dim in [1, 65536]");
    GSD_REQUIRE(a->axes >= 1 && a->axes <= GSD_MAX_AXES, "axes must lie in [1, %d]", GSD_MAX_AXES);
    int64_t pairs = 0;
    for (int i = 0; i < a->axes; ++i) {
        GSD_REQUIRE(a->sections[i] >= 0 && a->sections[i] <= a->dim, "section %d is out of range",
                    i);
        pairs += a->sections[i];
    }
    GSD_REQUIRE(2 * pairs <= a->dim, "the sections turn %lld channels of %lld",
                (long long)(2 * pairs), (long long)a->dim);
    // a thread takes four values at least, in 32-bit counts
    const __int128 n = (__int128)a->batch * a->length * a->heads * a->dim;
    GSD_REQUIRE((__int128)a->batch * a->length * a->heads * (a->dim / 4 + 2) <= 256 * kMaxGroups,
                "the tensor is too large");
    if (n == 0) return GSR_OK;
    GSD_REQUIRE(a->x && a->y && (pairs == 0 || (a->positions && a->inv_freq)), "null pointer");
    const int e = dtype_size(a->dtype), p = a->positions_type == GSD_POS_I64 ? 8 : 4;
    GSD_REQUIRE(aligned(a->x, e) && aligned(a->y, e) && aligned(a->positions, p) &&
                    aligned(a->inv_freq, 4),
                "a pointer is not aligned to its elements");
    GSD_HIP(gsd::launch_rotary(*a, as_stream(stream)), "rotary_axes");
    return GSR_OK;
}

int gsd_rms_norm(const gsd_norm* a, void* y, void* stream) {
    if (int rc = check_norm(a)) return rc;
    if (a->rows == 0) return GSR_OK;
    GSD_REQUIRE(y, "null pointer");
    GSD_REQUIRE(aligned(y, dtype_size(a->dtype)), "a pointer is not aligned to its elements");
    GSD_HIP(gsd::launch_rms_norm(*a, y, nullptr, nullptr, as_stream(stream)), "rms_norm");
    return GSR_OK;
}

int gsd_rms_norm_fp8(const gsd_norm* a, uint8_t* y8, float* scale, void* stream) {
    if (int rc = check_norm(a)) return rc;
    if (a->rows == 0) return GSR_OK;
    GSD_REQUIRE(y8 && scale, "null pointer");
    GSD_REQUIRE(aligned(scale, 4), "a pointer is not aligned to its elements");
    GSD_HIP(gsd::launch_rms_norm(*a, nullptr, y8, scale, as_stream(stream)), "rms_norm_fp8");
    return GSR_OK;
}

size_t gsd_rms_norm_backward_workspace_bytes(int64_t rows, int64_t width) {
    if (rows <= 0 || rows >= kMaxCount || width < 1 || width > GSD_MAX_NORM_WIDTH) return 0;
    return 4 * (size_t)gsd::norm_backward_groups(rows, width) * (size_t)width;
}

int gsd_rms_norm_backward(int dtype, int64_t rows, int64_t width, const void* h,
                          const float* rstd, const void* weight, const void* dy,
                          int64_t dy_stride, const void* dh, int64_t dh_stride, void* dx,
                          void* dweight, void* ws, size_t ws_bytes, void* stream) {
    GSD_REQUIRE(dtype_ok(dtype), "unknown dtype %d", dtype);
    GSD_REQUIRE(rows >= 0 && rows < kMaxCount, "rows must lie in [0, 2^31)");
    GSD_REQUIRE(width >= 1 && width <= GSD_MAX_NORM_WIDTH, "width must lie in [1, %d]",
                GSD_MAX_NORM_WIDTH);
    if (!dx && !dweight) return GSR_OK;
    GSD_REQUIRE(rows == 0 || (h && rstd && weight && dy), "null pointer");
    const int e = dtype_size(dtype);
    GSD_REQUIRE(aligned(h, e) && aligned(rstd, 4) && aligned(weight, e) && aligned(dy, e) &&
                    aligned(dh, e) && aligned(dx, e) && aligned(dweight, e) && aligned(ws, 4),
                "a pointer is not aligned to its elements");
    if (dweight && ws_bytes < gsd_rms_norm_backward_workspace_bytes(rows, width))
        return fail(GSR_ERR_WORKSPACE, "workspace of %zu bytes is too small", ws_bytes);
    GSD_REQUIRE(!dweight || rows == 0 || ws, "null pointer");
    GSD_HIP(gsd::launch_rms_norm_backward(dtype, rows, width, h, rstd, weight, dy, dy_stride, dh,
                                          dh_stride, dx, dweight, static_cast<float*>(ws),
                                          as_stream(stream)),
            "rms_norm_backward");
    return GSR_OK;
}

size_t gsd_attention_workspace_bytes(const gsd_attention* a) {
    if (check_attention(a)) return 0;
    return forward_layout(*a, gsd::attention_split_rows(*a)).end;
}

int gsd_cross_attention(const gsd_attention* a, void* ws, size_t ws_bytes, void* stream) {
    if (int rc = check_attention(a)) return rc;
    if (int rc = check_attention_pointers(a)) return rc;
    if (a->batch == 0 || a->queries == 0) return GSR_OK;
    const gsd::AttentionSplit s = gsd::attention_split_rows(*a);
    GSD_REQUIRE(grid_fits(*a, s), "too many rows");
    const ForwardLayout l = forward_layout(*a, s);
    if (ws_bytes < l.end || (l.end && !ws))
        return fail(GSR_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", ws_bytes, l.end);
    GSD_REQUIRE(aligned(ws, 16), "the workspace must be 16-byte aligned");
    GSD_HIP(gsd::launch_attention(*a, s, at<float>(ws, l.o), at<float>(ws, l.lse),
                                  a->key_mask ? at<int32_t>(ws, l.list) : nullptr,
                                  as_stream(stream)),
            "cross_attention");
    return GSR_OK;
}

size_t gsd_attention_backward_workspace_bytes(const gsd_attention* a) {
    if (check_attention(a)) return 0;
    return backward_layout(*a, gsd::attention_split_dq(*a), gsd::attention_split_dkdv(*a)).end;
}

int gsd_cross_attention_backward(const gsd_attention* a, const gsd_attention_grad* g, void* ws,
                                 size_t ws_bytes, void* stream) {
    if (int rc = check_attention(a)) return rc;
    if (int rc = check_attention_pointers(a)) return rc;
    GSD_REQUIRE(g, "null pointer");
    if (a->batch == 0) return GSR_OK;
    GSD_REQUIRE(a->queries == 0 || (a->lse && g->d_o), "null pointer");
    GSD_REQUIRE(!g->dk == !g->dv, "dk and dv go together");
    GSD_REQUIRE(row_strides_fit(*a, a->q_stride_l, a->q_stride_h) &&
                    row_strides_fit(*a, g->do_stride_l, g->do_stride_h),
                "the strides of q and do must not be negative, nor 64 queries or the heads of a "
                "group span 2^30 elements");
    GSD_REQUIRE(aligned(g->d_o, 2) && aligned(g->dq, 2) && aligned(g->dk, 2) && aligned(g->dv, 2),
                "a pointer is not aligned to its elements");
    const gsd::AttentionSplit sq = gsd::attention_split_dq(*a);
    const gsd::AttentionSplit sk = gsd::attention_split_dkdv(*a);
    GSD_REQUIRE(grid_fits(*a, sq) && grid_fits(*a, sk), "too many rows or keys");
    // delta's work-groups: of rows, of values, of zeros (2048 values each)
    GSD_REQUIRE((__int128)a->batch * a->kv_heads *
                        (gsd::attention_top_blocks(*a) + gsd::attention_value_blocks(*a) +
                         (__int128)a->keys * a->dim / 2048 + 2) <= kMaxGroups,
                "too many rows or keys");
    const BackwardLayout l = backward_layout(*a, sq, sk);
    if (ws_bytes < l.end || (l.end && !ws))
        return fail(GSR_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", ws_bytes, l.end);
    GSD_REQUIRE(aligned(ws, 16), "the workspace must be 16-byte aligned");
    const gsd::AttentionBackwardBuffers buf{at<float>(ws, l.stat), at<float>(ws, l.top),
                                            at<float>(ws, l.value_top), at<float>(ws, l.dq),
                                            at<float>(ws, l.dk), at<float>(ws, l.dv),
                                            a->key_mask ? at<int32_t>(ws, l.list) : nullptr};
    GSD_HIP(gsd::launch_attention_backward(*a, *g, sq, sk, buf, as_stream(stream)),
            "cross_attention_backward");
    return GSR_OK;
}

}  // extern "C"
