// Quantised KV cache: the write that rounds 16-bit K/V rows to e4m3 codes with
// one exponent byte a row, and the read that gives them back.
//
// A row x (one token, one kv head) is held as
//   z = x with its magnitudes held to T,  T = 61440 (fp16), 15/16 * 2^128 (bf16)
//   e = the least integer with max|z| <= 448 * 2^e, at least -126
//   codes = z * 2^-e rounded to nearest even e4m3,  byte = e + 127
// The scale is a power of two because e4m3 is itself a floating format: within
// its 18 binades another factor would give the same relative step, while this
// one makes z * 2^-e exact (one rounding per value, the same on any machine) and
// the dequantised value exact in bf16.  T keeps what the row stands for finite
// in the row's type: values above 15/16 of the range would round up to its end,
// and go to T instead, at most 6.2 % off against the 6.25 % of e4m3's half step.
// NaN keeps a NaN code and does not count in the maximum.
//
// Bound by memory: 256 B in and 129 B out per row of 128 bf16 values.  LANES
// lanes share a row (8 values each, K and V alike), so a wave reads whole rows
// with 16-byte loads, and the maximum is two to four DPP steps in the VALU.  Measured
// (8 kv heads of 128, a call): the write of 24573 tokens, 150 MB, 30.2 us, 5.0 TB/s (a
// large copy 5.1); of 32 tokens 4.5 us, a launch; the read of 65536 tokens, 404 MB,
// 84.8 us, 4.8 TB/s.
#include "fp8.h"
#include "kv_slots.h"

namespace vaa {
namespace {

constexpr int kThreadsQ = 256;

struct QuantCache {
  uint8_t* k;
  uint8_t* v;
  uint8_t* ke;
  uint8_t* ve;
  int64_t k_sb, k_sh, k_st, v_sb, v_sh, v_st;
  int64_t ke_sb, ke_sh, ke_st, ve_sb, ve_sh, ve_st;
};

struct Rows16 {
  uint16_t* k;
  uint16_t* v;
  int64_t s_tok, s_head;
};

// Slots below 2^31: division in 32 bits, or a shift where the block size is a power
// of two (SlotResolver divides in 64).
template <typename IdxT>
struct NarrowSlots {
  const IdxT* slots;
  int block_size, shift;  // shift < 0: not a power of two
  uint32_t capacity;
  __device__ bool operator()(int t, int64_t& block, int64_t& off) const {
    const int64_t s = static_cast<int64_t>(slots[t]);
    if (static_cast<uint64_t>(s) >= capacity) return false;
    const uint32_t u = static_cast<uint32_t>(s);
    const uint32_t b = shift >= 0 ? u >> shift : u / static_cast<uint32_t>(block_size);
    block = b;
    off = u - b * static_cast<uint32_t>(block_size);
    return true;
  }
};

// Magnitudes are compared as bit patterns, which order like them: a NaN x, quiet or
// signalling (bf16 rows can hold both), does not count.
__device__ __forceinline__ uint32_t count_in(uint32_t m, float x) {
  const uint32_t u = __float_as_uint(x) & 0x7FFFFFFFu;
  return max(m, u > 0x7F800000u ? 0u : u);
}

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_max(uint32_t x) {
  return max(x, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(x), CTRL, 0xF, 0xF,
                                                               true)));
}

// The maximum over each aligned group of LANES lanes, in all of them: quad_perm
// by 1 and 2, then mirrors of 8 and of 16 lanes, whose sources hold the
// maximum of the other half.
template <int LANES>
__device__ __forceinline__ uint32_t group_max(uint32_t x) {
  x = dpp_max<0xB1>(x);
  x = dpp_max<0x4E>(x);
  if constexpr (LANES >= 8) x = dpp_max<0x141>(x);
  if constexpr (LANES >= 16) x = dpp_max<0x140>(x);
  return x;
}

template <typename T>
constexpr float kTop = 61440.f;
template <>
constexpr float kTop<bf16> = 0x1.Ep127f;

// e for a row whose magnitudes reach u (a bit pattern), held to T: 448 = 1.75 * 2^8,
// so 1.f * 2^E needs e = E - 8 up to a fraction of 1.75 and E - 7 above it.
template <typename T>
__device__ __forceinline__ int row_exponent(uint32_t u) {
  u = min(u, __builtin_bit_cast(uint32_t, kTop<T>));
  const int e = static_cast<int>(u >> 23) - 127 - 8 + ((u & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return max(e, -126);  // zero and the smallest rows of bf16
}

// |x| to T; NaN stays (the comparison is false).
__device__ __forceinline__ float hold(float x, float top) {
  return fabsf(x) > top ? copysignf(top, x) : x;
}

template <typename T>
__device__ __forceinline__ u32x2 quant8(const float* x, float scale) {
  float z[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) z[i] = hold(x[i], kTop<T>) * scale;
  u32x2 r;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    int p = __builtin_amdgcn_cvt_pk_fp8_f32(z[4 * w], z[4 * w + 1], 0, false);
    r[w] = __builtin_amdgcn_cvt_pk_fp8_f32(z[4 * w + 2], z[4 * w + 3], p, true);
  }
  return r;
}

template <typename T, int LANES>
__device__ __forceinline__ void quant_row(u32x4 raw, uint8_t* codes, uint8_t* exp, bool mine,
                                          bool first) {
  const auto h = __builtin_bit_cast(typename Elem<T>::x8, raw);
  float x[8];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = Elem<T>::to_f(h[i]);
    m = count_in(m, x[i]);
  }
  const int e = row_exponent<T>(group_max<LANES>(m));
  const u32x2 c = quant8<T>(x, __uint_as_float(static_cast<uint32_t>(127 - e) << 23));
  if (mine) *reinterpret_cast<u32x2*>(codes) = c;
  if (first) *exp = static_cast<uint8_t>(e + 127);
}

// LANES lanes a row (4, 8 or 16), lane c of them the values 8c .. 8c + 7.
template <typename T, int LANES, typename Resolver>
__global__ void __launch_bounds__(kThreadsQ)
kv_quant_kernel(QuantCache d, Rows16 s, Resolver resolve, int num_tokens, int num_kv_heads,
                int chunks) {
  const int c = threadIdx.x % LANES;
  const int64_t rows = static_cast<int64_t>(num_tokens) * num_kv_heads;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (kThreadsQ / LANES);
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreadsQ / LANES) + threadIdx.x / LANES;
       row < rows; row += step) {
    const int h = static_cast<int>(row % num_kv_heads);
    const int t = static_cast<int>(row / num_kv_heads);
    const bool in = c < chunks;
    const int64_t so = t * s.s_tok + h * s.s_head + 8 * c;
    // The rows are read before the slot is known: one round trip.
    u32x4 k = {0u, 0u, 0u, 0u}, v = k;
    if (in) {
      k = ld16_stream(s.k + so);
      v = ld16_stream(s.v + so);
    }
    int64_t block, off;
    if (!resolve(t, block, off)) continue;  // the same for the row's lanes
    quant_row<T, LANES>(k, d.k + block * d.k_sb + h * d.k_sh + off * d.k_st + 8 * c,
                        d.ke + block * d.ke_sb + h * d.ke_sh + off * d.ke_st, in, c == 0);
    quant_row<T, LANES>(v, d.v + block * d.v_sb + h * d.v_sh + off * d.v_st + 8 * c,
                        d.ve + block * d.ve_sb + h * d.ve_sh + off * d.ve_st, in, c == 0);
  }
}

// Rows that are not made of aligned 16-byte pieces: 16 lanes a row, one value at
// a time, in two passes.
template <typename T>
__device__ __forceinline__ void quant_row1(const uint16_t* x, uint8_t* codes, uint8_t* exp, int hd,
                                           int c) {
  const T* xs = reinterpret_cast<const T*>(x);
  uint32_t m = 0;
  for (int i = c; i < hd; i += 16) m = count_in(m, Elem<T>::to_f(xs[i]));
  const int e = row_exponent<T>(group_max<16>(m));
  const float scale = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
  for (int i = c; i < hd; i += 16) {
    const float z = hold(Elem<T>::to_f(xs[i]), kTop<T>) * scale;
    codes[i] = static_cast<uint8_t>(__builtin_amdgcn_cvt_pk_fp8_f32(z, z, 0, false));
  }
  if (c == 0) *exp = static_cast<uint8_t>(e + 127);
}

template <typename T, typename Resolver>
__global__ void __launch_bounds__(kThreadsQ)
kv_quant_kernel1(QuantCache d, Rows16 s, Resolver resolve, int num_tokens, int num_kv_heads,
                 int hd) {
  const int c = threadIdx.x % 16;
  const int64_t rows = static_cast<int64_t>(num_tokens) * num_kv_heads;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (kThreadsQ / 16);
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreadsQ / 16) + threadIdx.x / 16;
       row < rows; row += step) {
    const int h = static_cast<int>(row % num_kv_heads);
    const int t = static_cast<int>(row / num_kv_heads);
    int64_t block, off;
    if (!resolve(t, block, off)) continue;
    const int64_t so = t * s.s_tok + h * s.s_head;
    quant_row1<T>(s.k + so, d.k + block * d.k_sb + h * d.k_sh + off * d.k_st,
                  d.ke + block * d.ke_sb + h * d.ke_sh + off * d.ke_st, hd, c);
    quant_row1<T>(s.v + so, d.v + block * d.v_sb + h * d.v_sh + off * d.v_st,
                  d.ve + block * d.ve_sb + h * d.ve_sh + off * d.ve_st, hd, c);
  }
}

// The read: a lane takes eight codes of K and the same eight of V.  A token
// without a slot gets zeros.
template <typename T, typename Resolver>
__global__ void __launch_bounds__(kThreadsQ)
kv_dequant_kernel(QuantCache d, Rows16 s, Resolver resolve, int num_tokens, int num_kv_heads,
                  int chunks) {
  const int64_t total = static_cast<int64_t>(num_tokens) * num_kv_heads * chunks;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreadsQ + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * kThreadsQ) {
    const int c = static_cast<int>(i % chunks);
    const int64_t th = i / chunks;
    const int h = static_cast<int>(th % num_kv_heads);
    const int t = static_cast<int>(th / num_kv_heads);
    const int64_t so = t * s.s_tok + h * s.s_head + 8 * c;
    u32x4 k = {0u, 0u, 0u, 0u}, v = k;
    int64_t block, off;
    if (resolve(t, block, off)) {
      const u32x2 kc = *reinterpret_cast<const u32x2*>(d.k + block * d.k_sb + h * d.k_sh +
                                                       off * d.k_st + 8 * c);
      const u32x2 vc = *reinterpret_cast<const u32x2*>(d.v + block * d.v_sb + h * d.v_sh +
                                                       off * d.v_st + 8 * c);
      const uint32_t ke = d.ke[block * d.ke_sb + h * d.ke_sh + off * d.ke_st];
      const uint32_t ve = d.ve[block * d.ve_sb + h * d.ve_sh + off * d.ve_st];
      k = deq8<T>(kc[0], kc[1], scale_of(ke));
      v = deq8<T>(vc[0], vc[1], scale_of(ve));
    }
    st16(s.k + so, k);
    st16(s.v + so, v);
  }
}

// The same a value at a time, for rows that are not made of aligned pieces.
template <typename T, typename Resolver>
__global__ void __launch_bounds__(kThreadsQ)
kv_dequant_kernel1(QuantCache d, Rows16 s, Resolver resolve, int num_tokens, int num_kv_heads,
                   int hd) {
  const int64_t total = static_cast<int64_t>(num_tokens) * num_kv_heads * hd;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreadsQ + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * kThreadsQ) {
    const int c = static_cast<int>(i % hd);
    const int64_t th = i / hd;
    const int h = static_cast<int>(th % num_kv_heads);
    const int t = static_cast<int>(th / num_kv_heads);
    const int64_t so = t * s.s_tok + h * s.s_head + c;
    uint32_t k = 0, v = 0;
    int64_t block, off;
    if (resolve(t, block, off)) {
      k = deq2<T, false>(d.k[block * d.k_sb + h * d.k_sh + off * d.k_st + c],
                         scale_of(d.ke[block * d.ke_sb + h * d.ke_sh + off * d.ke_st]));
      v = deq2<T, false>(d.v[block * d.v_sb + h * d.v_sh + off * d.v_st + c],
                         scale_of(d.ve[block * d.ve_sb + h * d.ve_sh + off * d.ve_st]));
    }
    s.k[so] = static_cast<uint16_t>(k);
    s.v[so] = static_cast<uint16_t>(v);
  }
}

bool pieces_aligned(const QuantCache& d, const Rows16& s, int hd) {
  const int64_t bytes[] = {d.k_sb, d.k_sh, d.k_st, d.v_sb, d.v_sh, d.v_st, s.s_tok, s.s_head, hd};
  for (int64_t b : bytes)
    if (b % 8) return false;
  return aligned16(s.k) && aligned16(s.v) && reinterpret_cast<uintptr_t>(d.k) % 8 == 0 &&
         reinterpret_cast<uintptr_t>(d.v) % 8 == 0;
}

unsigned blocks_for(int64_t items, int per_block) {
  const int64_t n = (items + per_block - 1) / per_block;
  return static_cast<unsigned>(n < 65536 ? n : 65536);
}

template <typename T, typename Resolver>
int launch_quant(const QuantCache& d, const Rows16& s, const Resolver& r, int n, int kvh, int hd,
                 hipStream_t stream) {
  const int64_t rows = static_cast<int64_t>(n) * kvh;
  if (!pieces_aligned(d, s, hd) || hd > 128) {
    hipLaunchKernelGGL((kv_quant_kernel1<T, Resolver>), dim3(blocks_for(rows, kThreadsQ / 16)),
                       dim3(kThreadsQ), 0, stream, d, s, r, n, kvh, hd);
    return check_launch("kv_quant_kernel1");
  }
  const int chunks = hd / 8;
#define VAA_QUANT(LANES)                                                                        \
  hipLaunchKernelGGL((kv_quant_kernel<T, LANES, Resolver>),                                     \
                     dim3(blocks_for(rows, kThreadsQ / LANES)), dim3(kThreadsQ), 0, stream, d, \
                     s, r, n, kvh, chunks)
  if (chunks <= 4)
    VAA_QUANT(4);
  else if (chunks <= 8)
    VAA_QUANT(8);
  else
    VAA_QUANT(16);
#undef VAA_QUANT
  return check_launch("kv_quant_kernel");
}

template <typename T, typename Resolver>
int launch_dequant(const QuantCache& d, const Rows16& s, const Resolver& r, int n, int kvh, int hd,
                   hipStream_t stream) {
  const int64_t rows = static_cast<int64_t>(n) * kvh;
  if (!pieces_aligned(d, s, hd)) {
    hipLaunchKernelGGL((kv_dequant_kernel1<T, Resolver>), dim3(blocks_for(rows * hd, kThreadsQ)),
                       dim3(kThreadsQ), 0, stream, d, s, r, n, kvh, hd);
    return check_launch("kv_dequant_kernel1");
  }
  hipLaunchKernelGGL((kv_dequant_kernel<T, Resolver>),
                     dim3(blocks_for(rows * (hd / 8), kThreadsQ)), dim3(kThreadsQ), 0, stream, d,
                     s, r, n, kvh, hd / 8);
  return check_launch("kv_dequant_kernel");
}

// The checks that the three entry points share.
int check_quant(const char* what, const vaa_attn_params* p, const vaa_kv_view* view,
                const void* k, const void* v, const void* sk, const void* sv, int num_tokens) {
  if (!p || !view) return fail(VAA_ERR_INVALID_ARG, "%s: null params", what);
  if (!valid_dtype(p->dtype)) return fail(VAA_ERR_UNSUPPORTED, "%s: dtype=%d", what, p->dtype);
  if (view->cache_type != VAA_CACHE_E4M3)
    return fail(VAA_ERR_UNSUPPORTED, "%s: cache_type=%d (VAA_CACHE_E4M3)", what,
                view->cache_type);
  if (num_tokens < 0) return fail(VAA_ERR_INVALID_ARG, "%s: num_tokens=%d", what, num_tokens);
  if (p->num_kv_heads <= 0 || p->head_size <= 0 || p->block_size <= 0 || p->num_blocks < 0)
    return fail(VAA_ERR_INVALID_ARG, "%s: num_kv_heads=%d head_size=%d block_size=%d", what,
                p->num_kv_heads, p->head_size, p->block_size);
  if (num_tokens > 0 && (!k || !v || !sk || !sv || !view->key_exps || !view->value_exps))
    return fail(VAA_ERR_INVALID_ARG, "%s: null cache, exponent or row pointer", what);
  return VAA_OK;
}

QuantCache cache_of(const vaa_attn_params* p, const vaa_kv_view* c, uint8_t* k, uint8_t* v) {
  return QuantCache{k, v, c->key_exps, c->value_exps,
                    p->k_stride_block, p->k_stride_head, p->k_stride_token,
                    p->v_stride_block, p->v_stride_head, p->v_stride_token,
                    c->ke_stride_block, c->ke_stride_head, c->ke_stride_token,
                    c->ve_stride_block, c->ve_stride_head, c->ve_stride_token};
}

// Calls f with the resolver for these slots.
template <typename F>
int with_slots(const vaa_attn_params* p, const void* slots, int index_type, F f) {
  const int64_t cap = p->num_blocks * p->block_size;
  const bool wide = index_type == VAA_INDEX_I64;
  const int bs = p->block_size;
  if (cap >= (int64_t{1} << 31))
    return wide ? f(SlotResolver<int64_t>{static_cast<const int64_t*>(slots), bs, cap})
                : f(SlotResolver<int32_t>{static_cast<const int32_t*>(slots), bs, cap});
  const int shift = (bs & (bs - 1)) == 0 ? __builtin_ctz(bs) : -1;
  const uint32_t c = static_cast<uint32_t>(cap);
  return wide ? f(NarrowSlots<int64_t>{static_cast<const int64_t*>(slots), bs, shift, c})
              : f(NarrowSlots<int32_t>{static_cast<const int32_t*>(slots), bs, shift, c});
}

template <typename Resolver>
int quantise(const vaa_attn_params* p, const QuantCache& d, const Rows16& s, const Resolver& r,
             int n, void* stream) {
  hipStream_t st = static_cast<hipStream_t>(stream);
  return p->dtype == VAA_DTYPE_BF16
             ? launch_quant<bf16>(d, s, r, n, p->num_kv_heads, p->head_size, st)
             : launch_quant<f16>(d, s, r, n, p->num_kv_heads, p->head_size, st);
}

template <typename Resolver>
int dequantise(const vaa_attn_params* p, const QuantCache& d, const Rows16& s, const Resolver& r,
               int n, void* stream) {
  hipStream_t st = static_cast<hipStream_t>(stream);
  return p->dtype == VAA_DTYPE_BF16
             ? launch_dequant<bf16>(d, s, r, n, p->num_kv_heads, p->head_size, st)
             : launch_dequant<f16>(d, s, r, n, p->num_kv_heads, p->head_size, st);
}

}  // namespace
}  // namespace vaa

using namespace vaa;

extern "C" int vaa_kv_write_slots_q8(const vaa_attn_params* p, const vaa_kv_view* view,
                                     uint8_t* key_cache, uint8_t* value_cache,
                                     const void* slot_mapping, int slot_index_type,
                                     const uint16_t* new_keys, const uint16_t* new_values,
                                     int num_tokens, void* stream) {
  const char* what = "vaa_kv_write_slots_q8";
  int st = check_quant(what, p, view, key_cache, value_cache, new_keys, new_values, num_tokens);
  if (st) return st;
  if (slot_index_type != VAA_INDEX_I32 && slot_index_type != VAA_INDEX_I64)
    return fail(VAA_ERR_INVALID_ARG, "%s: slot_index_type=%d", what, slot_index_type);
  if (num_tokens == 0) return VAA_OK;
  if (!slot_mapping) return fail(VAA_ERR_INVALID_ARG, "%s: null slot_mapping", what);
  const QuantCache d = cache_of(p, view, key_cache, value_cache);
  const Rows16 s{const_cast<uint16_t*>(new_keys), const_cast<uint16_t*>(new_values),
                 p->new_kv_stride_token, p->new_kv_stride_head};
  return with_slots(p, slot_mapping, slot_index_type, [&](const auto& r) {
    return quantise(p, d, s, r, num_tokens, stream);
  });
}

extern "C" int vaa_kv_write_decode_q8(const vaa_attn_params* p, const vaa_kv_view* view,
                                      uint8_t* key_cache, uint8_t* value_cache,
                                      const int32_t* block_table, const int32_t* seq_lens,
                                      const uint16_t* new_keys, const uint16_t* new_values,
                                      void* stream) {
  const char* what = "vaa_kv_write_decode_q8";
  int st = check_quant(what, p, view, key_cache, value_cache, new_keys, new_values,
                       p ? p->num_seqs : 0);
  if (st) return st;
  if (p->max_blocks_per_seq <= 0)
    return fail(VAA_ERR_INVALID_ARG, "%s: max_blocks_per_seq=%d", what, p->max_blocks_per_seq);
  if (p->num_seqs == 0) return VAA_OK;
  if (!block_table || !seq_lens)
    return fail(VAA_ERR_INVALID_ARG, "%s: null block_table or seq_lens", what);
  const QuantCache d = cache_of(p, view, key_cache, value_cache);
  const Rows16 s{const_cast<uint16_t*>(new_keys), const_cast<uint16_t*>(new_values),
                 p->new_kv_stride_token, p->new_kv_stride_head};
  return quantise(p, d, s, DecodeResolver{block_table, seq_lens, p->max_blocks_per_seq,
                                          p->block_size, p->num_blocks}, p->num_seqs, stream);
}

extern "C" int vaa_kv_read_slots_q8(const vaa_attn_params* p, const vaa_kv_view* view,
                                    const uint8_t* key_cache, const uint8_t* value_cache,
                                    const void* slot_mapping, int slot_index_type, uint16_t* keys,
                                    uint16_t* values, int num_tokens, void* stream) {
  const char* what = "vaa_kv_read_slots_q8";
  int st = check_quant(what, p, view, key_cache, value_cache, keys, values, num_tokens);
  if (st) return st;
  if (slot_index_type != VAA_INDEX_I32 && slot_index_type != VAA_INDEX_I64)
    return fail(VAA_ERR_INVALID_ARG, "%s: slot_index_type=%d", what, slot_index_type);
  if (num_tokens == 0) return VAA_OK;
  if (!slot_mapping) return fail(VAA_ERR_INVALID_ARG, "%s: null slot_mapping", what);
  const QuantCache d = cache_of(p, view, const_cast<uint8_t*>(key_cache),
                                const_cast<uint8_t*>(value_cache));
  const Rows16 s{keys, values, p->new_kv_stride_token, p->new_kv_stride_head};
  return with_slots(p, slot_mapping, slot_index_type, [&](const auto& r) {
    return dequantise(p, d, s, r, num_tokens, stream);
  });
}
