// Checks that the attention entry points over a vaa_kv_view share.
#pragma once

#include "common.h"

namespace vaa {

inline int check_view(const char* what, const vaa_attn_params* p, const vaa_kv_view* view) {
  if (!p || !view) return fail(VAA_ERR_INVALID_ARG, "%s: null params", what);
  const bool q8 = view->cache_type == VAA_CACHE_E4M3;
  if (!q8 && view->cache_type != VAA_CACHE_16BIT)
    return fail(VAA_ERR_UNSUPPORTED, "%s: cache_type=%d", what, view->cache_type);
  if (!head_size_ok(p->head_size) || (q8 && p->head_size % 16))
    return fail(VAA_ERR_UNSUPPORTED, "%s: head_size=%d (a multiple of %d up to 128)", what,
                p->head_size, q8 ? 16 : 8);
  if (!valid_dtype(p->dtype))
    return fail(VAA_ERR_UNSUPPORTED, "%s: dtype=%d (VAA_DTYPE_F16 or VAA_DTYPE_BF16)", what,
                p->dtype);
  // The running maximum is taken over the products, before the scale.
  if (!(p->scale > 0.f && p->scale < 3.0e38f))
    return fail(VAA_ERR_INVALID_ARG, "%s: scale=%g must be positive and finite", what,
                static_cast<double>(p->scale));
  if (p->block_size <= 0)
    return fail(VAA_ERR_INVALID_ARG, "%s: block_size=%d must be positive", what, p->block_size);
  if (p->num_kv_heads <= 0 || p->num_query_heads <= 0 ||
      p->num_query_heads % p->num_kv_heads != 0 ||
      p->queries_per_kv != p->num_query_heads / p->num_kv_heads)
    return fail(VAA_ERR_INVALID_ARG, "%s: heads %d/%d, queries_per_kv=%d", what,
                p->num_query_heads, p->num_kv_heads, p->queries_per_kv);
  if (p->num_blocks <= 0)
    return fail(VAA_ERR_INVALID_ARG, "%s: num_blocks=%lld", what, (long long)p->num_blocks);
  if (view->window < 0 || view->first_tokens < 0)
    return fail(VAA_ERR_INVALID_ARG, "%s: window=%d first_tokens=%d", what, view->window,
                view->first_tokens);
  if (q8 && (!view->key_exps || !view->value_exps))
    return fail(VAA_ERR_INVALID_ARG, "%s: null exponents", what);
  const int64_t unit = q8 ? 16 : 8;
  const int64_t cache[] = {p->k_stride_block, p->k_stride_head, p->k_stride_token,
                           p->v_stride_block, p->v_stride_head, p->v_stride_token};
  for (int64_t s : cache)
    if (s < 0 || s % unit)
      return fail(VAA_ERR_INVALID_ARG, "%s: cache strides must be non-negative multiples of %d",
                  what, (int)unit);
  const int64_t rows[] = {p->q_stride_token, p->q_stride_head, p->o_stride_token,
                          p->o_stride_head};
  for (int64_t s : rows)
    if (s < 0 || s % 8)
      return fail(VAA_ERR_INVALID_ARG,
                  "%s: query and output strides must be non-negative multiples of 8", what);
  if (q8) {
    const int64_t exps[] = {view->ke_stride_block, view->ke_stride_head, view->ke_stride_token,
                            view->ve_stride_block, view->ve_stride_head, view->ve_stride_token};
    for (int64_t s : exps)
      if (s < 0) return fail(VAA_ERR_INVALID_ARG, "%s: negative exponent stride", what);
    if (view->ke_stride_token >= (int64_t{1} << 24) || view->ve_stride_token >= (int64_t{1} << 24))
      return fail(VAA_ERR_INVALID_ARG, "%s: exponent token stride too large", what);
  }
  // Offsets inside a block are 32-bit bytes.
  if (p->k_stride_block >= (int64_t{1} << 31) || p->v_stride_block >= (int64_t{1} << 31) ||
      p->k_stride_token * p->block_size >= (int64_t{1} << 31) ||
      p->v_stride_token * p->block_size >= (int64_t{1} << 31))
    return fail(VAA_ERR_UNSUPPORTED, "%s: a cache block of 2^31 values or more", what);
  if (p->k_stride_token >= (int64_t{1} << 24) || p->v_stride_token >= (int64_t{1} << 24))
    return fail(VAA_ERR_INVALID_ARG, "%s: token stride too large", what);
  return VAA_OK;
}

}  // namespace vaa
