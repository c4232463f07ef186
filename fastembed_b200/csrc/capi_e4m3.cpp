// capi_e4m3.cpp — extern "C" entry points of the 8-bit (e4m3) operators: argument validation,
// then the launchers.  No counterpart in the reference, whose arithmetic is fp32.
#include <cuda_runtime.h>

#include <cmath>
#include <string>

#include "fe_internal.h"

using fe::fail;

namespace {

inline cudaStream_t cs(fe_stream_t s) { return reinterpret_cast<cudaStream_t>(s); }

inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

fe_status bad(const char *name, const char *what) { return fail(FE_ERR_INVALID_ARGUMENT, std::string(name) + ": " + what); }

fe_status unsupported(const char *name, const char *what) { return fail(FE_ERR_UNSUPPORTED, std::string(name) + ": " + what); }

fe_status check_rows(const char *name, fe_dtype dtype, int64_t rows, int32_t dim)
{
    if (rows < 0 || dim <= 0) return bad(name, "bad shape");
    if (rows > 0x7fffffff || dim > 1 << 30) return unsupported(name, "too many rows or columns");
    if (dtype != FE_DTYPE_F32 && dtype != FE_DTYPE_BF16) return bad(name, "unknown input dtype");
    return FE_OK;
}

// The geometry that the cache's write and its attention share.
fe_status check_cache(const char *name, int32_t batch, int32_t max_len, int64_t total, int32_t q_heads, int32_t kv_heads,
                      int32_t head_dim, int32_t width, int32_t pages, int32_t page)
{
    if (batch < 0 || max_len < 0 || total < 0 || q_heads <= 0 || kv_heads <= 0 || width < 0 || pages < 0)
        return bad(name, "bad shape");
    if (q_heads % kv_heads != 0) return bad(name, "q_heads must be a multiple of kv_heads");
    if (head_dim != 64 && head_dim != 128 && head_dim != 256) return unsupported(name, "head_dim must be 64, 128 or 256");
    if (page != 16 && page != 32 && page != 64 && page != 128) return unsupported(name, "pages hold 16, 32, 64 or 128 tokens");
    if (batch > 65535 || q_heads > 1024 || max_len > 1 << 20 || total > 0x7fffffff || width > 1 << 26)
        return unsupported(name, "batch, heads, max_len or table too large");
    // CTAs of one launch: row tiles of 8 (token, head of a group) rows, or reached pages, per sequence
    if (static_cast<int64_t>(batch) * ((static_cast<int64_t>(max_len) * (q_heads / kv_heads) + 7) / 8 + max_len / 16 + 2) >
        0x7fffffff)
        return unsupported(name, "batch x max_len too large");
    return FE_OK;
}

// Tiles of 128 or 256 rows of a sequence's key-value head are a launch's z extent.
fe_status check_rows_per_head(const char *name, int32_t max_len, int32_t q_heads, int32_t kv_heads)
{
    if (static_cast<int64_t>(max_len) * (q_heads / kv_heads) > 65535 * 128)
        return unsupported(name, "max_len x q_heads / kv_heads too large");
    return FE_OK;
}

// What a call that has work to do needs of the pool: TMA coordinates count its rows in 32 bits.
fe_status check_pool(const char *name, int32_t pages, int32_t kv_heads, int32_t page)
{
    if (pages == 0) return bad(name, "a pool without pages");
    if (static_cast<int64_t>(pages) * kv_heads * page > 0x7ffffff0) return unsupported(name, "pages x kv_heads x page_size past 2^31");
    return FE_OK;
}

}  // namespace

extern "C" {

fe_status fe_quantize_rows_e4m3(const void *x, fe_dtype x_dtype, int64_t rows, int32_t dim, void *q, float *scale,
                                fe_stream_t stream)
{
    const char *name = "fe_quantize_rows_e4m3";
    FE_TRY(check_rows(name, x_dtype, rows, dim));
    if (rows == 0) return FE_OK;
    if (!x || !q || !scale) return bad(name, "null pointer");
    return fe::check_cuda(fe::launch_quantize_rows_e4m3(x, x_dtype, rows, dim, q, scale, cs(stream)), name);
}

fe_status fe_add_rmsnorm_e4m3(const void *y, fe_dtype y_dtype, float *h32, const float *w, int32_t one_plus, float eps,
                              int64_t rows, int32_t dim, void *q, float *scale, fe_stream_t stream)
{
    const char *name = "fe_add_rmsnorm_e4m3";
    FE_TRY(check_rows(name, y_dtype, rows, dim));
    if (!(eps >= 0.f)) return bad(name, "eps must be >= 0");
    if (rows == 0) return FE_OK;
    if (!h32 || !w || !q || !scale) return bad(name, "null pointer");
    return fe::check_cuda(
        fe::launch_add_rmsnorm_e4m3(y, y_dtype, h32, w, one_plus != 0, eps, rows, dim, q, scale, cs(stream)), name);
}

fe_status fe_linear_e4m3(const void *x, const float *x_scale, const void *w, const float *w_scale, const float *bias,
                         const float *residual, void *y, int64_t m, int64_t n, int64_t k, fe_epilogue epilogue,
                         fe_dtype y_dtype, fe_stream_t stream)
{
    const char *name = "fe_linear_e4m3";
    if (m < 0 || n <= 0 || k <= 0) return bad(name, "bad shape");
    if (k % 16 != 0 || n % 8 != 0) return bad(name, "k must be a multiple of 16 and n of 8");
    if (m > 0x7fffffff - 255 || n > 0x7fffffff - 255 || k > 0x7fffffff - 127 ||
        (m + 127) / 128 * ((n + 63) / 64) > 0x7fffffff)
        return unsupported(name, "size too large");
    if (epilogue < FE_EPI_NONE || epilogue > FE_EPI_GEGLU) return bad(name, "unknown epilogue");
    if (y_dtype != FE_DTYPE_F32 && y_dtype != FE_DTYPE_BF16) return bad(name, "unknown output dtype");
    const bool glu = epilogue == FE_EPI_SWIGLU || epilogue == FE_EPI_GEGLU;
    const bool act = epilogue == FE_EPI_BIAS_GELU || epilogue == FE_EPI_BIAS_RELU || epilogue == FE_EPI_BIAS_SWISH;
    if ((glu || act) && y_dtype != FE_DTYPE_BF16) return bad(name, "activations write bf16");
    if (glu && n % 128 != 0) return bad(name, "gated epilogues need n % 128 == 0");
    if (epilogue == FE_EPI_BIAS_RESIDUAL && y_dtype != FE_DTYPE_F32) return bad(name, "the residual epilogue writes fp32");
    if (m == 0) return FE_OK;
    if (!x || !x_scale || !w || !w_scale || !y) return bad(name, "null pointer");
    if (epilogue != FE_EPI_NONE && !glu && !bias) return bad(name, "epilogue needs a bias");
    if (epilogue == FE_EPI_BIAS_RESIDUAL && !residual) return bad(name, "residual epilogue needs a residual");
    if (!aligned16(x) || !aligned16(w) || !aligned16(y) || !aligned16(w_scale) || (bias && !aligned16(bias)) ||
        (residual && !aligned16(residual)))
        return bad(name, "pointers must be 16-byte aligned");
    fe_status st = FE_OK;
    cudaError_t e = fe::launch_linear_e4m3(x, x_scale, w, w_scale, bias, residual, y, m, n, k, epilogue, y_dtype, cs(stream), &st);
    if (st != FE_OK) return st;
    return fe::check_cuda(e, name);
}

fe_status fe_kv_cache_append_e4m3(const void *qkv, const int32_t *cu_seqlens, int32_t batch, int32_t max_len,
                                  int64_t total_tokens, int32_t q_heads, int32_t kv_heads, int32_t head_dim,
                                  const int32_t *past_lens, const int32_t *page_table, int32_t table_width, void *k_pages,
                                  void *v_pages, float *k_scales, float *v_scales, int32_t pages, int32_t page_size,
                                  fe_stream_t stream)
{
    const char *name = "fe_kv_cache_append_e4m3";
    FE_TRY(check_cache(name, batch, max_len, total_tokens, q_heads, kv_heads, head_dim, table_width, pages, page_size));
    if (batch == 0 || total_tokens == 0 || max_len == 0) return FE_OK;
    FE_TRY(check_pool(name, pages, kv_heads, page_size));
    if (!qkv || !cu_seqlens || !past_lens || !page_table || !k_pages || !v_pages || !k_scales || !v_scales)
        return bad(name, "null pointer");
    if (!aligned16(qkv) || !aligned16(k_pages) || !aligned16(v_pages)) return bad(name, "pointers must be 16-byte aligned");
    return fe::check_cuda(
        fe::launch_kv_cache_append_e4m3(qkv, cu_seqlens, batch, max_len, total_tokens, q_heads, kv_heads, head_dim, past_lens,
                                        page_table, table_width, k_pages, v_pages, k_scales, v_scales, pages, page_size,
                                        cs(stream)),
        name);
}

fe_status fe_attention_cache_workspace_bytes(int32_t batch, int32_t max_len, int64_t total_tokens, int32_t max_kv_len,
                                             int32_t q_heads, int32_t kv_heads, int32_t head_dim, size_t *bytes)
{
    const char *name = "fe_attention_cache_workspace_bytes";
    if (!bytes) return bad(name, "null pointer");
    FE_TRY(check_cache(name, batch, max_len, total_tokens, q_heads, kv_heads, head_dim, 0, 0, 16));
    FE_TRY(check_rows_per_head(name, max_len, q_heads, kv_heads));
    if (max_kv_len < 0) return bad(name, "bad shape");
    *bytes = batch == 0 || total_tokens == 0 || max_len == 0
                 ? 0
                 : fe::attention_cache_workspace_bytes(batch, max_len, total_tokens, max_kv_len, q_heads, kv_heads, head_dim);
    return FE_OK;
}

fe_status fe_attention_cache_e4m3(const void *qkv, const int32_t *cu_seqlens, int32_t batch, int32_t max_len,
                                  int64_t total_tokens, int32_t q_heads, int32_t kv_heads, int32_t head_dim,
                                  const int32_t *past_lens, int32_t max_kv_len, const int32_t *page_table,
                                  int32_t table_width, const void *k_pages, const void *v_pages, const float *k_scales,
                                  const float *v_scales, int32_t pages, int32_t page_size, int32_t causal, float scale,
                                  void *out, void *workspace, size_t workspace_bytes, fe_stream_t stream)
{
    const char *name = "fe_attention_cache_e4m3";
    FE_TRY(check_cache(name, batch, max_len, total_tokens, q_heads, kv_heads, head_dim, table_width, pages, page_size));
    FE_TRY(check_rows_per_head(name, max_len, q_heads, kv_heads));
    if (max_kv_len < 0 || !std::isfinite(scale)) return bad(name, "bad max_kv_len or scale");
    if (batch == 0 || total_tokens == 0 || max_len == 0) return FE_OK;
    FE_TRY(check_pool(name, pages, kv_heads, page_size));
    if (!qkv || !cu_seqlens || !past_lens || !page_table || !k_pages || !v_pages || !k_scales || !v_scales || !out)
        return bad(name, "null pointer");
    if (!aligned16(qkv) || !aligned16(k_pages) || !aligned16(v_pages) || !aligned16(out))
        return bad(name, "pointers must be 16-byte aligned");
    const size_t need =
        fe::attention_cache_workspace_bytes(batch, max_len, total_tokens, max_kv_len, q_heads, kv_heads, head_dim);
    if (need > 0 && (!workspace || workspace_bytes < need || !aligned16(workspace)))
        return bad(name, "workspace missing, too small or not 16-byte aligned");
    fe_status st = FE_OK;
    cudaError_t e = fe::launch_attention_cache_e4m3(qkv, cu_seqlens, batch, max_len, total_tokens, q_heads, kv_heads, head_dim,
                                                    past_lens, max_kv_len, page_table, table_width, k_pages, v_pages, k_scales,
                                                    v_scales, pages, page_size, causal != 0, scale, out, workspace, cs(stream),
                                                    &st);
    if (st != FE_OK) return st;
    return fe::check_cuda(e, name);
}

}  // extern "C"
