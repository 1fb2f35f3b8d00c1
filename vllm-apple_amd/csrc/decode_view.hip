// Paged decode attention over a cache as vaa_kv_view describes it: 16-bit or e4m3
// rows, the whole context or a sliding window behind a few first tokens.
//
//   out[s, h] = sum_j softmax_j(scale q[s, h] . K_j) V_j   over the keys
//   j < L,  j < first or j >= L - window,   L = seq_lens[s]
//
// Bound by the stream of K and V from HBM.  The structure is the paged decode's
// (S^T = K Q^T and O^T += V^T P^T on the matrix cores, one running maximum and sum
// per head, K straight into operand registers, V through a transposing LDS read,
// waves combined in LDS, long contexts split over workgroups and merged), with
// three things of its own:
//  - The tiles of a sequence are numbered through: those of the first tokens, then
//    those of the window.  Splits count these tiles, so a share is what is read.
//  - e4m3 rows are half as wide, so a tile is 32 tokens instead of 16: the bytes in
//    flight per wave stay the same.  Both operands are made 16-bit on the way in
//    (v_cvt_scalef32_pk, which applies the row's exponent): K in registers, V as it
//    goes to LDS.  The PV product then takes 32 tokens in one MFMA step.
//  - P enters the PV product as a pair hi + lo of 16-bit values for both types (two
//    MFMAs; the stream hides them), for fp16 2^8 above its softmax value so that the
//    lo half stays a normal number down to 2^-10.  One rounding of P would cost as
//    much as the rounding of the output itself.
//
// Measured (heads 32 on 8 of 128, blocks of 16): 32 contexts of 8192, e4m3 93 us, 5.8
// TB/s (a kernel that only reads the rows 80.5; the 16-bit decode of them 162); windows of
// 4096 and 4 first tokens, 27 sequences of 16-bit rows 87 us (75 only read), 64 of e4m3
// rows 117 us with the merge (95).  A wave's tile is a chain (wait, convert, QK, softmax,
// PV) at two waves a SIMD: taking the exponents away, or three tiles ahead, changed
// nothing.
#include "fp8.h"
#include "kv_view.h"

#include <algorithm>
#include <atomic>

namespace vaa {
namespace {

typedef short i16x4 __attribute__((ext_vector_type(4)));

// P is computed 2^kPShift times its value (bf16 needs none).
template <typename T>
constexpr float kPShift = 8.f;
template <>
constexpr float kPShift<bf16> = 0.f;
constexpr int kQuantum = 128;     // fixed partitions: a multiple of this many tokens
constexpr int kWideWaves = 8;     // waves of a workgroup with a long partition
constexpr int kWaves4 = 4;        // ... with a short one, and of the balanced split
// Partitions up to this long take four waves.  Eight against four, us (heads 32 on 8 of
// 128): 32 x 8192 e4m3 in partitions of 512 199 / 138, of 2048 118 / 102; 8 x 32768 in
// 2048 16-bit 180 / 170, in 4096 e4m3 112 / 105, 16-bit 170 / 165.  Longer ones are few:
// 4 x 32768 e4m3, heads 16 on 4, in 4096 50 / 50, in 8192 78 / 85.
constexpr int kShortTokens = 4096;
// Balanced: workgroups per CU's worth.  1, 2, 3: 27 ragged contexts of 100 to 9000, e4m3
// 65, 59, 73 us; 64 windows of 4096 128, 117, 122 us.
constexpr int kBalPerCu = 2;
// Balanced: least share of a workgroup.  8 x 2048 e4m3 32 us at 32 tiles, 20 at 8.
constexpr int kBalMinTiles = 8;
// Balanced: a sequence's start-up, in tiles.  2, 8: 27 ragged contexts 62, 59 us.
constexpr int kSeqTiles = 8;
constexpr int kBalMaxSeqs = 8192;

struct Args {
  const uint16_t* q;
  const uint8_t* kc;
  const uint8_t* vc;
  const uint8_t* ke;
  const uint8_t* ve;
  const int32_t* bt;
  const int32_t* seq_lens;
  uint16_t* out;
  // Partials of split sequences, a row per (piece, query head): unnormalised acc
  // [D], and (max in the log2 domain, sum).  Fixed partitions: row (seq * H + head)
  // * max_parts + part.  Balanced: (y * (max_parts + num_seqs) + c + seq) * Gc + h, y
  // = kv head x head chunk, and hdr holds (share, starts[0 .. num_seqs]).
  float* ws_acc;
  float* ws_ml;
  int* ws_hdr;
  float scale_log2;
  int hd, num_seqs, max_blocks, block_size, kvh, H, G;
  int Gc, chunks;  // query heads per workgroup (<= 16), and workgroups per kv head
  int part_tiles, max_parts;
  int lds_main;
  int window, first;
  int bs_shift;         // log2(block_size) where it is a power of two, else -1
  uint32_t num_blocks;  // at most 2^31: block ids are 32-bit
  // Bytes.  Block strides are below 2^32 and offsets inside a block 32-bit.
  uint32_t k_sb, k_st, v_sb, v_st;
  int64_t k_sh, v_sh;
  int64_t ke_sb, ke_sh, ke_st, ve_sb, ve_sh, ve_st;  // bytes
  int64_t q_st, q_sh, o_st, o_sh;                    // elements
};

__device__ __forceinline__ int block_of(const Args& a, int key) {
  return a.bs_shift >= 0 ? key >> a.bs_shift : key / a.block_size;
}

template <int D, bool Q8>
struct Cfg {
  static constexpr int R = Q8 ? 32 : 16;  // tokens per tile
  static constexpr int NG = R / 16;       // 16-row groups: MFMA row blocks
  static constexpr int NS = D / 32;       // QK steps
  static constexpr int NDT = D / 16;      // PV dim tiles
  // A lane's K piece: 16 bytes (8 values, or 16 codes for two steps), or 8 codes
  // where D has an odd number of steps.
  static constexpr bool WIDE = !Q8 || D % 64 == 0;
  static constexpr int KL = Q8 && WIDE ? D / 64 : D / 32;  // pieces per group
  static constexpr int VCH = Q8 ? D / 16 : D / 8;          // 16-byte chunks of a V row
  static constexpr int VLD = R * VCH / kWave;              // V loads per lane
  static constexpr int VPER = Q8 ? 16 : 8;                 // values per V chunk
  static constexpr bool SWZ = D == 64 || D == 128;
  // Rows of V load i all lie in one 16-row group.
  static constexpr bool VUNI = NG == 1 || (kWave % VCH == 0 && 16 % (kWave / VCH) == 0);
};

// Chunk swizzle of the V tile in LDS: physical 16-byte chunk = logical ^ swz(row).
// Four rows side by side, which a transposing read takes together, differ in their
// chunk pair; two rows side by side, which a write of two chunks a lane takes
// together, in the chunk of the pair.
template <int D>
__device__ __forceinline__ int swz(int row) {
  return (D == 64 || D == 128) ? ((row & 3) << 1) | (row & 1) : 0;
}

template <bool kWidePiece>
struct Piece { typedef u32x4 t; };
template <>
struct Piece<false> { typedef u32x2 t; };

template <int D, bool Q8>
struct Tile {
  using C = Cfg<D, Q8>;
  using KP = typename Piece<C::WIDE>::t;
  KP k[C::NG * C::KL];
  u32x4 v[C::VLD];
  uint32_t ke, ve;  // Q8: exponent bytes of row lane % 32
};

// How a sequence's tiles lie: nf tiles of first tokens, then those from real tile
// w0 on; n in all.  A query sees keys below `first`, and from `lo` up to L.
struct Span {
  int L, lo, first, nf, skip, n;
  __device__ __forceinline__ int real(int t) const { return t < nf ? t : t + skip; }
};

template <int R>
__device__ __forceinline__ Span span_of(const Args& a, int L) {
  Span s;
  s.L = L;
  const int tiles = (L + R - 1) / R;
  s.lo = a.window > 0 ? max(0, L - a.window) : 0;
  s.first = min(a.first, s.lo);
  s.nf = (s.first + R - 1) / R;
  s.skip = max(0, s.lo / R - s.nf);
  s.n = tiles - s.skip;
  return s;
}

__device__ __forceinline__ uint32_t low_bits(int n) {
  return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u;
}

// Rows of the tile from token tok0 that the query sees.
__device__ __forceinline__ uint32_t seen_rows(const Span& s, int tok0) {
  return low_bits(s.L - tok0) & (~low_bits(s.lo - tok0) | low_bits(s.first - tok0));
}

template <int D, bool Q8>
struct LaneMap {
  using C = Cfg<D, Q8>;
  int vrow[C::VLD];
  uint32_t koff, voff[C::VLD];  // byte offsets inside a 16-row group / from its rows
  uint32_t wlds[C::VLD];        // element offset in the LDS tile
  uint32_t keoff, veoff;        // Q8: byte offset of row lane % 16's exponents
  uint32_t trbase;
  int trsw;
  uint32_t kval, vval;  // kAny: bit i set where piece i lies below hd
};

__device__ __forceinline__ int load_window(const Args& a, int seq, int blk0, int lane) {
  const int e = blk0 + lane;
  return e < a.max_blocks ? a.bt[static_cast<int64_t>(seq) * a.max_blocks + e] : -1;
}

// Loads the tile of tokens tok0 .. tok0 + R - 1 (table entries from block blk0 on in
// the lanes of vals) and returns its rows in valid blocks.  Rows in others are
// read from the start of block 0 and masked.
template <int D, bool Q8, bool kAny>
__device__ __forceinline__ uint32_t issue(const Args& a, const LaneMap<D, Q8>& m, int vals,
                                          int blk0, int tok0, int kvh, int lane,
                                          Tile<D, Q8>& t) {
  using C = Cfg<D, Q8>;
  using KP = typename Tile<D, Q8>::KP;
  const uint8_t* kb = a.kc + kvh * a.k_sh;
  const uint8_t* vb = a.vc + kvh * a.v_sh;
  const int c16 = lane & 15;
  uint32_t ok = 0;
  if (!kAny || a.block_size % 16 == 0) {
    uint64_t kr[C::NG], vr[C::NG];
    uint64_t ker[C::NG], ver[C::NG];
#pragma unroll
    for (int grp = 0; grp < C::NG; ++grp) {
      const int tok = tok0 + 16 * grp;
      const int bi = block_of(a, tok);
      uint32_t rin = tok - bi * a.block_size;
      // The second group of a window's last tile may lie past the 64 entries.
      uint32_t p = bi - blk0 < kWave
                       ? static_cast<uint32_t>(__builtin_amdgcn_readlane(vals, bi - blk0))
                       : ~0u;
      if (p < a.num_blocks) {
        ok |= 0xFFFFu << (16 * grp);
      } else {
        p = 0;
        rin = 0;
      }
      kr[grp] = static_cast<uint64_t>(p) * a.k_sb + rin * a.k_st;
      vr[grp] = static_cast<uint64_t>(p) * a.v_sb + rin * a.v_st;
      if constexpr (Q8) {
        ker[grp] = p * a.ke_sb + kvh * a.ke_sh + rin * a.ke_st;
        ver[grp] = p * a.ve_sb + kvh * a.ve_sh + rin * a.ve_st;
      }
    }
#pragma unroll
    for (int grp = 0; grp < C::NG; ++grp)
#pragma unroll
      for (int i = 0; i < C::KL; ++i) {
        const KP* src = reinterpret_cast<const KP*>(
            kb + kr[grp] + i * (Q8 ? (C::WIDE ? 64 : 32) : 64) + m.koff);
        if (kAny && !((m.kval >> i) & 1u))
          t.k[grp * C::KL + i] = KP{};
        else
          t.k[grp * C::KL + i] = __builtin_nontemporal_load(src);
      }
#pragma unroll
    for (int i = 0; i < C::VLD; ++i) {
      uint64_t r;
      if constexpr (C::NG == 1)
        r = vr[0];
      else if constexpr (C::VUNI)
        r = vr[i * (kWave / C::VCH) / 16];
      else
        r = m.vrow[i] < 16 ? vr[0] : vr[C::NG - 1];
      if (kAny && !((m.vval >> i) & 1u))
        t.v[i] = u32x4{0u, 0u, 0u, 0u};
      else
        t.v[i] = ld16_stream(vb + r + m.voff[i]);
    }
    if constexpr (Q8) {
      const bool up = lane & 16;
      t.ke = a.ke[(up ? ker[C::NG - 1] : ker[0]) + m.keoff];
      t.ve = a.ve[(up ? ver[C::NG - 1] : ver[0]) + m.veoff];
    }
    return ok;
  }
  // Rows that find their own blocks.
  auto row_at = [&](int row, int64_t& phys, int& rin) {
    const int tok = tok0 + row;
    const int bi = tok / a.block_size, w = bi - blk0;
    phys = __shfl(vals, min(w, kWave - 1), kWave);
    rin = tok - bi * a.block_size;
    const bool good = w < kWave && phys >= 0 && static_cast<uint32_t>(phys) < a.num_blocks;
    if (!good) {
      phys = 0;
      rin = 0;
    }
    return good;
  };
#pragma unroll
  for (int grp = 0; grp < C::NG; ++grp) {
    int64_t p;
    int r;
    const bool good = row_at(16 * grp + c16, p, r);
    ok |= (static_cast<uint32_t>(__builtin_amdgcn_ballot_w64(good)) & 0xFFFFu) << (16 * grp);
    const uint8_t* row =
        kb + p * a.k_sb + static_cast<int64_t>(r) * a.k_st + (m.koff - c16 * a.k_st);
#pragma unroll
    for (int i = 0; i < C::KL; ++i) {
      const KP* src = reinterpret_cast<const KP*>(row + i * (Q8 ? (C::WIDE ? 64 : 32) : 64));
      t.k[grp * C::KL + i] = ((m.kval >> i) & 1u) ? *src : KP{};
    }
  }
#pragma unroll
  for (int i = 0; i < C::VLD; ++i) {
    int64_t p;
    int r;
    row_at(m.vrow[i], p, r);
    const int ch = (i * kWave + lane) % C::VCH;
    t.v[i] = ((m.vval >> i) & 1u) ? ld16(vb + p * a.v_sb + static_cast<int64_t>(r) * a.v_st + ch * 16)
                                  : u32x4{0u, 0u, 0u, 0u};
  }
  if constexpr (Q8) {
    int64_t p;
    int r;
    row_at(lane & 31, p, r);
    t.ke = a.ke[p * a.ke_sb + kvh * a.ke_sh + r * a.ke_st];
    t.ve = a.ve[p * a.ve_sb + kvh * a.ve_sh + r * a.ve_st];
  }
  return ok;
}

// The maximum over the lanes l, l ^ 16, l ^ 32, l ^ 48, in all of them: the swaps
// exchange odd rows of 16 lanes (halves of the wave) of one operand with even rows
// (the lower half) of the other, so with x in both the two results hold x and its
// partner's x.  In the VALU: no LDS round trip between the two products.
__device__ __forceinline__ float groups_max(float x) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// One tile of math; bit r of seen: row r counts (kMask false: all do).
template <int D, typename T, bool Q8, bool kMask>
__device__ __forceinline__ void tile_product(const LaneMap<D, Q8>& m, const Tile<D, Q8>& t,
                                          const u32x4* qb, T* vt, uint32_t seen, int lane,
                                          float scale_log2, float& m_run, float& l_part,
                                          f32x4* acc) {
  using C = Cfg<D, Q8>;
  using X4 = typename Elem<T>::x4;
  using X8 = typename Elem<T>::x8;
  const int c16 = lane & 15, g = lane >> 4;
  const u32x4 zero = {0u, 0u, 0u, 0u};
  // V to LDS; rows that do not count become zeros, whatever they hold.
#pragma unroll
  for (int i = 0; i < C::VLD; ++i) {
    const bool in = !kMask || ((seen >> m.vrow[i]) & 1u);
    if constexpr (Q8) {
      const float s = scale_of(__shfl(t.ve, m.vrow[i], kWave));
      const u32x4 lo = deq8<T>(t.v[i][0], t.v[i][1], s), hi = deq8<T>(t.v[i][2], t.v[i][3], s);
      *reinterpret_cast<u32x4*>(vt + m.wlds[i]) = in ? lo : zero;
      *reinterpret_cast<u32x4*>(vt + (m.wlds[i] ^ (C::SWZ ? 8 : 0)) + (C::SWZ ? 0 : 8)) =
          in ? hi : zero;
    } else {
      *reinterpret_cast<u32x4*>(vt + m.wlds[i]) = in ? t.v[i] : zero;
    }
  }
  // S^T = K Q^T, 16 tokens x 16 heads a group.
  f32x4 s4[C::NG];
#pragma unroll
  for (int grp = 0; grp < C::NG; ++grp) {
    s4[grp] = f32x4{0.f, 0.f, 0.f, 0.f};
    float ks = 0.f;
    if constexpr (Q8) ks = scale_of(__shfl(t.ke, 16 * grp + c16, kWave));
#pragma unroll
    for (int s = 0; s < C::NS; ++s) {
      u32x4 k;
      if constexpr (!Q8)
        k = t.k[grp * C::KL + s];
      else if constexpr (C::WIDE)
        k = deq8<T>(t.k[grp * C::KL + s / 2][2 * (s % 2)],
                    t.k[grp * C::KL + s / 2][2 * (s % 2) + 1], ks);
      else
        k = deq8<T>(t.k[grp * C::KL + s][0], t.k[grp * C::KL + s][1], ks);
      s4[grp] = Elem<T>::mfma16x16x32(__builtin_bit_cast(X8, k), __builtin_bit_cast(X8, qb[s]),
                                      s4[grp]);
    }
  }
  // Online softmax, log2 domain: lane = head, tokens 16 grp + 4g + r.
  float mx = -INFINITY;
#pragma unroll
  for (int grp = 0; grp < C::NG; ++grp)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if (kMask && !((seen >> (16 * grp + 4 * g + r)) & 1u)) s4[grp][r] = -INFINITY;
      mx = fmaxf(mx, s4[grp][r]);
    }
  mx = groups_max(mx) * scale_log2;
  const float m_new = fmaxf(m_run, mx);
  if (m_new != m_run) {
    const float alpha = fast_exp2(m_run - m_new);  // 0 when m_run = -inf
    l_part *= alpha;
#pragma unroll
    for (int dt = 0; dt < C::NDT; ++dt) acc[dt] *= alpha;
    m_run = m_new;
  }
  const float m_sub = m_run == -INFINITY ? 0.f : m_run - kPShift<T>;
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef decltype(Elem<T>::from_f(0.f)) E2 __attribute__((ext_vector_type(2)));
  X4 ph[C::NG], pl[C::NG];
#pragma unroll
  for (int grp = 0; grp < C::NG; ++grp)
#pragma unroll
    for (int r = 0; r < 4; r += 2) {
      const f32x2 p = {fast_exp2(fmaf(s4[grp][r], scale_log2, -m_sub)),
                       fast_exp2(fmaf(s4[grp][r + 1], scale_log2, -m_sub))};
      const E2 h = __builtin_convertvector(p, E2);
      const E2 l = __builtin_convertvector(
          f32x2{p[0] - Elem<T>::to_f(h[0]), p[1] - Elem<T>::to_f(h[1])}, E2);
      ph[grp][r] = h[0];
      ph[grp][r + 1] = h[1];
      pl[grp][r] = l[0];
      pl[grp][r + 1] = l[1];
      l_part += p[0] + p[1];
    }
  // O^T += V^T P^T; one transposing read gives a lane V[16 grp + 4g + r][16 dt + c16].
#pragma unroll
  for (int dt = 0; dt < C::NDT; ++dt) {
    X4 va[C::NG];
#pragma unroll
    for (int grp = 0; grp < C::NG; ++grp)
      va[grp] = __builtin_bit_cast(
          X4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                  (__attribute__((address_space(3))) i16x4*)(
                      vt + grp * 16 * D + m.trbase + (((2 * dt) ^ m.trsw) << 3))));
    if constexpr (C::NG == 2) {
      const X8 a8 = __builtin_shufflevector(va[0], va[1], 0, 1, 2, 3, 4, 5, 6, 7);
      const X8 h8 = __builtin_shufflevector(ph[0], ph[1], 0, 1, 2, 3, 4, 5, 6, 7);
      const X8 l8 = __builtin_shufflevector(pl[0], pl[1], 0, 1, 2, 3, 4, 5, 6, 7);
      acc[dt] = Elem<T>::mfma16x16x32(a8, h8, acc[dt]);
      acc[dt] = Elem<T>::mfma16x16x32(a8, l8, acc[dt]);
    } else {
      acc[dt] = Elem<T>::mfma16x16x16(va[0], ph[0], acc[dt]);
      acc[dt] = Elem<T>::mfma16x16x16(va[0], pl[0], acc[dt]);
    }
  }
}

template <int D, typename T, bool Q8>
__device__ __forceinline__ void tile_math(const LaneMap<D, Q8>& m, const Tile<D, Q8>& t,
                                          const u32x4* qb, T* vt, uint32_t seen, int lane,
                                          float scale_log2, float& m_run, float& l_part,
                                          f32x4* acc) {
  if (seen == low_bits(Cfg<D, Q8>::R))
    tile_product<D, T, Q8, false>(m, t, qb, vt, seen, lane, scale_log2, m_run, l_part, acc);
  else
    tile_product<D, T, Q8, true>(m, t, qb, vt, seen, lane, scale_log2, m_run, l_part, acc);
}

// Where the result of one (sequence, kv head, range of tiles) goes.
struct RangeOut {
  bool whole;         // all of the sequence: normalised rows of out
  int64_t row, step;  // else: workspace row of the first query head, and the stride
};

// The NW waves of the workgroup attend query heads qh0 .. qh0 + nh - 1 over the
// tiles [t0, t1) of the sequence: each wave a contiguous run, combined in LDS.
template <int D, typename T, bool Q8, int NW, bool kAny>
__device__ __forceinline__ void decode_range(const Args& a, unsigned char* smem, int seq, int kvh,
                                             int qh0, int nh, const Span& sp, int t0, int t1,
                                             const RangeOut& ro, bool trailing_barrier) {
  using C = Cfg<D, Q8>;
  // Uniform, so that tiles, blocks and masks are the scalar unit's.
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lane = threadIdx.x % kWave;
  const int c16 = lane & 15, g = lane >> 4;
  const int per = (t1 - t0 + NW - 1) / NW;
  const int jb = min(t0 + wave * per, t1), je = min(jb + per, t1);

  LaneMap<D, Q8> m;
  m.koff = c16 * a.k_st + g * (C::WIDE ? 16 : 8);
  m.keoff = c16 * static_cast<uint32_t>(a.ke_st);
  m.veoff = c16 * static_cast<uint32_t>(a.ve_st);
  m.kval = 0;
  m.vval = 0;
#pragma unroll
  for (int i = 0; i < C::VLD; ++i) {
    const int f = i * kWave + lane, row = f / C::VCH, ch = f % C::VCH;
    m.vrow[i] = row;
    m.voff[i] = (row & 15) * a.v_st + ch * 16;
    const int ch8 = Q8 ? 2 * ch : ch;
    m.wlds[i] = row * D + ((ch8 ^ swz<D>(row)) * 8);
    m.vval |= (ch * C::VPER < a.hd ? 1u : 0u) << i;
  }
  // First dim of K piece i: 16 codes at 64i + 16g, 8 codes at 32i + 8g, or 8 values
  // at 32i + 8g.
#pragma unroll
  for (int i = 0; i < C::KL; ++i)
    m.kval |= ((Q8 && C::WIDE ? 64 * i + 16 * g : 32 * i + 8 * g) < a.hd ? 1u : 0u) << i;
  {
    const int row = 4 * g + (c16 >> 2), j = c16 & 3;
    m.trsw = swz<D>(row) & ~1;
    m.trbase = row * D + ((j >> 1) ^ (swz<D>(row) & 1)) * 8 + (j & 1) * 4;
  }

  // Q^T as the B operand, its dims in the order of K's pieces.
  u32x4 qb[C::NS];
  {
    const bool hv = c16 < nh;
    const uint16_t* qp = a.q + seq * a.q_st + (qh0 + (hv ? c16 : 0)) * a.q_sh;
#pragma unroll
    for (int s = 0; s < C::NS; ++s) {
      const int d = Q8 && C::WIDE ? 64 * (s / 2) + 16 * g + 8 * (s % 2) : 32 * s + 8 * g;
      qb[s] = hv && (!kAny || d < a.hd) ? ld16(qp + d) : u32x4{0u, 0u, 0u, 0u};
    }
  }

  T* vt = reinterpret_cast<T*>(smem) + wave * (C::R * D);
  float m_run = -INFINITY, l_part = 0.f;
  f32x4 acc[C::NDT];
#pragma unroll
  for (int dt = 0; dt < C::NDT; ++dt) acc[dt] = f32x4{0.f, 0.f, 0.f, 0.f};

  // A run covers tiles that follow each other in the context and whose blocks lie
  // within 64 table entries (one per lane); loads go one tile ahead of the math.
  for (int cb = jb; cb < je;) {
    const int r0 = sp.real(cb);
    const int blk0 = block_of(a, r0 * C::R);
    const int64_t fits = (static_cast<int64_t>(blk0) + kWave) * a.block_size / C::R - r0;
    int ce = cb < sp.nf ? min(je, sp.nf) : je;
    // A tile that crosses the 64th entry is the next run's, unless it is the first
    // (blocks of fewer tokens than a tile never are).
    ce = static_cast<int>(min(static_cast<int64_t>(ce), cb + max(fits, int64_t{1})));
    const int vals = load_window(a, seq, blk0, lane);
    const int skip = r0 - cb, jl = ce - 1;
    auto get = [&](int j, Tile<D, Q8>& t) -> uint32_t {
      const int tok0 = (j + skip) * C::R;
      return issue<D, Q8, kAny>(a, m, vals, blk0, tok0, kvh, lane, t) & seen_rows(sp, tok0);
    };
    Tile<D, Q8> ta, tb;
    uint32_t va = get(cb, ta), vb;
    int j = cb;
    for (; j + 2 <= ce; j += 2) {
      vb = get(j + 1, tb);
      tile_math<D, T, Q8>(m, ta, qb, vt, va, lane, a.scale_log2, m_run, l_part, acc);
      va = get(min(j + 2, jl), ta);
      tile_math<D, T, Q8>(m, tb, qb, vt, vb, lane, a.scale_log2, m_run, l_part, acc);
    }
    if (j < ce) tile_math<D, T, Q8>(m, ta, qb, vt, va, lane, a.scale_log2, m_run, l_part, acc);
    cb = ce;
  }

  l_part += __shfl_xor(l_part, 16, kWave);
  l_part += __shfl_xor(l_part, 32, kWave);

  // Combine the waves: wm / wl [wave][16], wa [wave][nh][D].
  __syncthreads();
  float* wm = reinterpret_cast<float*>(smem);
  float* wl = wm + NW * 16;
  float* wa = wl + NW * 16;
  if (c16 < nh) {
    if (g == 0) {
      wm[wave * 16 + c16] = m_run;
      wl[wave * 16 + c16] = l_part;
    }
#pragma unroll
    for (int dt = 0; dt < C::NDT; ++dt)
      *reinterpret_cast<f32x4*>(wa + (wave * nh + c16) * D + 16 * dt + 4 * g) = acc[dt];
  }
  __syncthreads();
  for (int idx = threadIdx.x; idx < nh * D; idx += NW * kWave) {
    const int h = idx / D, d = idx % D;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, wm[w * 16 + h]);
    float num = 0.f, den = 0.f;
    if (M != -INFINITY) {
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float mw = wm[w * 16 + h];
        if (mw == -INFINITY) continue;
        const float sc = fast_exp2(mw - M);
        num += sc * wa[(w * nh + h) * D + d];
        den += sc * wl[w * 16 + h];
      }
    }
    if (ro.whole) {
      if (!kAny || d < a.hd)
        reinterpret_cast<T*>(a.out)[seq * a.o_st + (qh0 + h) * a.o_sh + d] =
            Elem<T>::from_f(M != -INFINITY ? num / den : 0.f);
    } else {
      const int64_t row = ro.row + h * ro.step;
      a.ws_acc[row * D + d] = num;
      if (d == 0) {
        a.ws_ml[row * 2] = M;
        a.ws_ml[row * 2 + 1] = den;
      }
    }
  }
  if (trailing_barrier) __syncthreads();
}

__device__ __forceinline__ int clamped_len(const Args& a, int seq) {
  const int64_t cap = static_cast<int64_t>(a.max_blocks) * a.block_size;
  const int L = a.seq_lens[seq];
  return L > cap ? static_cast<int>(cap) : L;
}

// Fixed partitions: grid (kv head x head chunk, partition, sequence).
template <int D, typename T, bool Q8, int NW, bool kAny>
__global__ void __launch_bounds__(NW* kWave) __attribute__((amdgpu_waves_per_eu(2)))
decode_view_kernel(Args a) {
  extern __shared__ __align__(16) unsigned char smem[];
  const int part = blockIdx.y, seq = blockIdx.z;
  const int kvh = blockIdx.x / a.chunks, hc = blockIdx.x % a.chunks;
  const int qh0 = kvh * a.G + hc * a.Gc, nh = min(a.Gc, a.G - hc * a.Gc);
  const int L = clamped_len(a, seq);
  if (L <= 0) {
    if (part == 0)
      for (int i = threadIdx.x; i < nh * a.hd; i += NW * kWave)
        a.out[seq * a.o_st + (qh0 + i / a.hd) * a.o_sh + i % a.hd] = 0;
    return;
  }
  const Span sp = span_of<Cfg<D, Q8>::R>(a, L);
  const int parts = min((sp.n + a.part_tiles - 1) / a.part_tiles, a.max_parts);
  if (part >= parts) return;
  const int t0 = part * a.part_tiles;
  const int t1 = part == a.max_parts - 1 ? sp.n : min(t0 + a.part_tiles, sp.n);
  const RangeOut ro{parts == 1,
                    (static_cast<int64_t>(seq) * a.H + qh0) * a.max_parts + part,
                    a.max_parts};
  decode_range<D, T, Q8, NW, kAny>(a, smem, seq, kvh, qh0, nh, sp, t0, t1, ro, false);
}

// Balanced split: the tiles of all sequences, with kSeqTiles in front of each for
// its start-up, laid end to end and dealt in equal shares; every workgroup derives
// the same prefix sums from seq_lens.
template <int R>
__device__ __forceinline__ int cost_of(const Args& a, int seq) {
  const int L = clamped_len(a, seq);
  return L > 0 ? span_of<R>(a, L).n + kSeqTiles : 0;
}

template <int R>
__device__ __forceinline__ void cost_prefix(const Args& a, int* starts, int* wsum) {
  const int B = a.num_seqs, nt = blockDim.x;
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const int per = (B + nt - 1) / nt;
  const int s0 = min(B, static_cast<int>(threadIdx.x) * per), s1 = min(B, s0 + per);
  int sum = 0;
  for (int s = s0; s < s1; ++s) sum += cost_of<R>(a, s);
  int x = sum;
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const int y = __shfl_up(x, o, kWave);
    if (lane >= o) x += y;
  }
  if (lane == kWave - 1) wsum[wave] = x;
  __syncthreads();
  int run = x - sum;
  for (int w = 0; w < wave; ++w) run += wsum[w];
  for (int s = s0; s < s1; ++s) {
    starts[s] = run;
    run += cost_of<R>(a, s);
  }
  if (threadIdx.x == nt - 1) starts[B] = run;
  __syncthreads();
}

template <int D, typename T, bool Q8, int NW, bool kAny>
__global__ void __launch_bounds__(NW* kWave) __attribute__((amdgpu_waves_per_eu(2)))
decode_view_balanced_kernel(Args a) {
  extern __shared__ __align__(16) unsigned char smem[];
  constexpr int R = Cfg<D, Q8>::R;
  const int c = blockIdx.x, y = blockIdx.y, nc = gridDim.x;
  const int kvh = y / a.chunks, hc = y % a.chunks;
  const int qh0 = kvh * a.G + hc * a.Gc, nh = min(a.Gc, a.G - hc * a.Gc);
  const int B = a.num_seqs;
  int* starts = reinterpret_cast<int*>(smem + a.lds_main);
  cost_prefix<R>(a, starts, starts + B + 1);
  const int total = starts[B];
  const int per = max((total + nc - 1) / nc, kBalMinTiles);
  if (c == 0 && y == 0) {
    if (threadIdx.x == 0) a.ws_hdr[0] = per;
    for (int s = threadIdx.x; s <= B; s += NW * kWave) a.ws_hdr[1 + s] = starts[s];
  }
  const int r0 = c * per, r1 = min(total, r0 + per);
  if (r0 >= r1) return;
  int lo = 0, hi = B - 1;  // first sequence with tiles at or after r0
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (starts[mid + 1] <= r0) lo = mid + 1;
    else hi = mid;
  }
  for (int seq = lo, pos = r0; pos < r1; ++seq) {
    const int s0 = starts[seq], s1 = starts[seq + 1];
    if (s1 <= pos) continue;
    const int u1 = min(r1, s1) - s0;
    const int t0 = max(0, pos - s0 - kSeqTiles), t1 = u1 - kSeqTiles;
    pos = s0 + u1;
    if (t1 <= t0) continue;  // start-up only: the tiles are the next workgroup's
    const Span sp = span_of<R>(a, clamped_len(a, seq));
    const RangeOut ro{t0 == 0 && t1 == sp.n,
                      (static_cast<int64_t>(y) * (nc + B) + c + seq) * a.Gc, 1};
    decode_range<D, T, Q8, NW, kAny>(a, smem, seq, kvh, qh0, nh, sp, t0, t1, ro, true);
  }
}

// Log-sum-exp merge of the pieces of the split sequences, a wave per (sequence,
// query head): D / 4 lanes take four dims each, and the 64 / (D / 4) such groups
// every so-manieth piece.  Each piece's loads are independent of the others'.
// Also zeroes the rows of empty sequences of a balanced split.
template <int D, typename T, bool Q8, bool kBalanced>
__global__ void __launch_bounds__(kWaves4* kWave) decode_view_merge_kernel(Args a) {
  constexpr int D4 = D / 4, NP = kWave / D4;
  constexpr int R = Cfg<D, Q8>::R;
  const int lane = threadIdx.x % kWave;
  const int qh = blockIdx.x * kWaves4 + threadIdx.x / kWave, seq = blockIdx.y;
  if (qh >= a.H) return;
  const int grp = lane / D4, d = 4 * (lane % D4);
  T* o = reinterpret_cast<T*>(a.out) + seq * a.o_st + qh * a.o_sh + d;
  const int L = clamped_len(a, seq);
  int64_t row0, step;
  int pieces;
  if constexpr (kBalanced) {
    const int per = a.ws_hdr[0], h0 = a.ws_hdr[1 + seq], h1 = a.ws_hdr[2 + seq];
    if (L <= 0) {
      if (grp == 0 && d < a.hd)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = Elem<T>::from_f(0.f);
      return;
    }
    const int c0 = (h0 + kSeqTiles) / per, c1 = (h1 - 1) / per;
    const int hg = qh % a.G, y = (qh / a.G) * a.chunks + hg / a.Gc;
    row0 = (static_cast<int64_t>(y) * (a.max_parts + a.num_seqs) + seq + c0) * a.Gc + hg % a.Gc;
    step = a.Gc;
    pieces = c1 - c0 + 1;
  } else {
    if (L <= 0) return;
    pieces = min((span_of<R>(a, L).n + a.part_tiles - 1) / a.part_tiles, a.max_parts);
    row0 = (static_cast<int64_t>(seq) * a.H + qh) * a.max_parts;
    step = 1;
  }
  if (pieces <= 1) return;  // written by the decode kernel
  float M = -INFINITY, den = 0.f;
  f32x4 num = {0.f, 0.f, 0.f, 0.f};
  auto add = [&](float mp, float lp, const f32x4& ap) {
    if (mp == -INFINITY) return;  // a piece that saw nothing
    const float Mn = fmaxf(M, mp);
    const float so = fast_exp2(M - Mn), sn = fast_exp2(mp - Mn);
    num = num * so + ap * sn;
    den = den * so + lp * sn;
    M = Mn;
  };
  if (grp < NP)
#pragma unroll 4
    for (int p = grp; p < pieces; p += NP) {
      const int64_t row = row0 + p * step;
      add(a.ws_ml[row * 2], a.ws_ml[row * 2 + 1],
          *reinterpret_cast<const f32x4*>(a.ws_acc + row * D + d));
    }
  // The groups' states into group 0's lanes.
#pragma unroll
  for (int p = 1; p < NP; ++p) {
    const int src = lane % D4 + p * D4;
    const float mp = __shfl(M, src, kWave), lp = __shfl(den, src, kWave);
    f32x4 ap;
#pragma unroll
    for (int i = 0; i < 4; ++i) ap[i] = __shfl(num[i], src, kWave);
    if (grp == 0) add(mp, lp, ap);
  }
  if (grp != 0 || d >= a.hd) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = Elem<T>::from_f(M != -INFINITY ? num[i] / den : 0.f);
}

constexpr int kMaxDevices = 64;
std::atomic<int> g_cus[kMaxDevices];

int num_cus() {
  int dev = 0, n = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= kMaxDevices) return 256;
  n = g_cus[dev].load(std::memory_order_relaxed);
  if (n > 0) return n;
  if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess ||
      n <= 0)
    n = 256;
  g_cus[dev].store(n, std::memory_order_relaxed);
  return n;
}

int head_chunks(int G) { return (G + 15) / 16; }
int heads_per_chunk(int G) { return (G + head_chunks(G) - 1) / head_chunks(G); }

struct Split {
  bool balanced;
  int part, max_parts;
  size_t ws_bytes, hdr_bytes;
};

// As vaa_paged_attention_decode's, over the tokens that are seen.
int plan_split(const char* what, const vaa_attn_params* p, const vaa_kv_view* view, Split* sp) {
  const int R = view->cache_type == VAA_CACHE_E4M3 ? 32 : 16;
  const int64_t cap = static_cast<int64_t>(p->max_blocks_per_seq) * p->block_size;
  int64_t len = std::max<int64_t>(1, std::min<int64_t>(p->max_seq_len, cap));
  if (view->window > 0) {
    // Whole tiles of the first tokens, and a window that begins and ends inside one.
    const int64_t seen = (static_cast<int64_t>(view->first_tokens) + R - 1) / R * R +
                         (static_cast<int64_t>(view->window) + 2 * R - 2) / R * R;
    len = std::min(len, seen);
  }
  const size_t row_bytes = (static_cast<size_t>(padded_head(p->head_size)) + 2) * sizeof(float);
  const int ys = p->num_kv_heads * head_chunks(p->queries_per_kv);
  const int64_t pairs = static_cast<int64_t>(p->num_seqs) * ys;
  int64_t part = p->partition_size;
  sp->balanced = part == VAA_PARTITION_BALANCED;
  if (sp->balanced) {
    if (p->num_seqs > kBalMaxSeqs)
      return fail(VAA_ERR_UNSUPPORTED, "%s: balanced split: num_seqs=%d > %d", what, p->num_seqs,
                  kBalMaxSeqs);
    sp->part = VAA_PARTITION_BALANCED;
    sp->hdr_bytes = ((static_cast<size_t>(p->num_seqs) + 2) * sizeof(int) + 255) / 256 * 256;
    sp->max_parts = std::max(1, (kBalPerCu * num_cus() + ys - 1) / ys);
    sp->ws_bytes = sp->hdr_bytes + static_cast<size_t>(ys) * (sp->max_parts + p->num_seqs) *
                                       heads_per_chunk(p->queries_per_kv) * row_bytes;
    return VAA_OK;
  }
  if (part < 0)
    return fail(VAA_ERR_UNSUPPORTED, "%s: partition_size=%lld (> 0, 0 or VAA_PARTITION_BALANCED)",
                what, (long long)part);
  if (part % kQuantum)
    return fail(VAA_ERR_INVALID_ARG, "%s: partition_size=%lld must be a multiple of %d", what,
                (long long)part, kQuantum);
  if (part == 0) {
    const int64_t splits = std::max<int64_t>(1, pairs > 0 ? (num_cus() + pairs - 1) / pairs : 1);
    part = (len + splits - 1) / splits;
    part = (part + kQuantum - 1) / kQuantum * kQuantum;
  }
  part = std::min<int64_t>(part, int64_t{1} << 30);
  const int64_t parts = (len + part - 1) / part;
  if (parts > 65535)
    return fail(VAA_ERR_UNSUPPORTED, "%s: partition_size=%lld makes more than 65535 partitions",
                what, (long long)part);
  sp->part = static_cast<int>(part);
  sp->max_parts = static_cast<int>(parts);
  sp->hdr_bytes = 0;
  sp->ws_bytes = parts <= 1 ? 0 : static_cast<size_t>(p->num_seqs) * p->num_query_heads * parts *
                                      row_bytes;
  return VAA_OK;
}

int check_decode(const char* what, const vaa_attn_params* p, const vaa_kv_view* view) {
  int st = check_view(what, p, view);
  if (st) return st;
  if (p->num_seqs < 0 || p->max_blocks_per_seq <= 0)
    return fail(VAA_ERR_INVALID_ARG, "%s: num_seqs=%d max_blocks_per_seq=%d", what, p->num_seqs,
                p->max_blocks_per_seq);
  if (p->num_seqs > 65535)
    return fail(VAA_ERR_UNSUPPORTED, "%s: num_seqs=%d > 65535", what, p->num_seqs);
  return VAA_OK;
}

template <int D, typename T, bool Q8, bool kAny>
int launch(const Args& a0, const Split& sp, hipStream_t stream) {
  Args a = a0;
  using C = Cfg<D, Q8>;
  auto lds = [&](int nw) {
    return std::max(static_cast<size_t>(nw) * C::R * D * 2,
                    (2 * nw * 16 + static_cast<size_t>(nw) * a.Gc * D) * sizeof(float));
  };
  const dim3 merge((a.H + kWaves4 - 1) / kWaves4, a.num_seqs);
  if (sp.balanced) {
    a.lds_main = static_cast<int>((lds(kWaves4) + 15) / 16 * 16);
    hipLaunchKernelGGL((decode_view_balanced_kernel<D, T, Q8, kWaves4, kAny>),
                       dim3(a.max_parts, a.kvh * a.chunks), dim3(kWaves4 * kWave),
                       a.lds_main + (a.num_seqs + 1 + kWaves4) * sizeof(int), stream, a);
    int st = check_launch("decode_view_balanced_kernel");
    if (st) return st;
    hipLaunchKernelGGL((decode_view_merge_kernel<D, T, Q8, true>), merge, dim3(kWaves4 * kWave),
                       0, stream, a);
    return check_launch("decode_view_merge_kernel");
  }
  const dim3 grid(a.kvh * a.chunks, a.max_parts, a.num_seqs);
  if (a.max_parts > 1 && sp.part <= kShortTokens)
    hipLaunchKernelGGL((decode_view_kernel<D, T, Q8, kWaves4, kAny>), grid,
                       dim3(kWaves4 * kWave), lds(kWaves4), stream, a);
  else
    hipLaunchKernelGGL((decode_view_kernel<D, T, Q8, kWideWaves, kAny>), grid,
                       dim3(kWideWaves * kWave), lds(kWideWaves), stream, a);
  int st = check_launch("decode_view_kernel");
  if (st || a.max_parts <= 1) return st;
  hipLaunchKernelGGL((decode_view_merge_kernel<D, T, Q8, false>), merge, dim3(kWaves4 * kWave), 0,
                     stream, a);
  return check_launch("decode_view_merge_kernel");
}

template <int D>
int launch_d(const Args& a, const Split& sp, bool bf, bool q8, hipStream_t s) {
  const bool any = a.hd != D || a.block_size % 16 != 0;
  if (q8) {
    if (any)
      return bf ? launch<D, bf16, true, true>(a, sp, s) : launch<D, f16, true, true>(a, sp, s);
    return bf ? launch<D, bf16, true, false>(a, sp, s) : launch<D, f16, true, false>(a, sp, s);
  }
  if (any)
    return bf ? launch<D, bf16, false, true>(a, sp, s) : launch<D, f16, false, true>(a, sp, s);
  return bf ? launch<D, bf16, false, false>(a, sp, s) : launch<D, f16, false, false>(a, sp, s);
}

}  // namespace
}  // namespace vaa

using namespace vaa;

extern "C" size_t vaa_paged_attention_decode_view_workspace_size(const vaa_attn_params* p,
                                                                 const vaa_kv_view* view,
                                                                 int32_t* partition_size_out) {
  const char* what = "vaa_paged_attention_decode_view_workspace_size";
  Split sp;
  if (check_decode(what, p, view) || p->num_seqs == 0 || plan_split(what, p, view, &sp)) return 0;
  if (partition_size_out) *partition_size_out = sp.part;
  return sp.ws_bytes;
}

extern "C" int vaa_paged_attention_decode_view(const vaa_attn_params* p, const vaa_kv_view* view,
                                               const uint16_t* query, const void* key_cache,
                                               const void* value_cache,
                                               const int32_t* block_table,
                                               const int32_t* seq_lens, uint16_t* output,
                                               void* workspace, size_t workspace_bytes,
                                               void* stream) {
  const char* what = "vaa_paged_attention_decode_view";
  int st = check_decode(what, p, view);
  if (st) return st;
  if (p->num_seqs == 0) return VAA_OK;
  if (!query || !key_cache || !value_cache || !block_table || !seq_lens || !output)
    return fail(VAA_ERR_INVALID_ARG, "%s: null pointer", what);
  if (!aligned16(query) || !aligned16(key_cache) || !aligned16(value_cache))
    return fail(VAA_ERR_INVALID_ARG, "%s: query and caches must be 16-byte aligned", what);
  Split sp;
  st = plan_split(what, p, view, &sp);
  if (st) return st;
  const bool q8 = view->cache_type == VAA_CACHE_E4M3;
  Args a{};
  if (sp.ws_bytes > 0) {
    if (!workspace || workspace_bytes < sp.ws_bytes)
      return fail(VAA_ERR_WORKSPACE, "%s: workspace %zu bytes < %zu needed", what,
                  workspace ? workspace_bytes : size_t{0}, sp.ws_bytes);
    if (!aligned16(workspace))
      return fail(VAA_ERR_INVALID_ARG, "%s: workspace must be 16-byte aligned", what);
    const int dp = padded_head(p->head_size);
    unsigned char* base = static_cast<unsigned char*>(workspace);
    a.ws_hdr = reinterpret_cast<int*>(base);
    a.ws_acc = reinterpret_cast<float*>(base + sp.hdr_bytes);
    a.ws_ml = a.ws_acc + (sp.ws_bytes - sp.hdr_bytes) / ((dp + 2) * sizeof(float)) * dp;
  }
  a.q = query;
  a.kc = static_cast<const uint8_t*>(key_cache);
  a.vc = static_cast<const uint8_t*>(value_cache);
  a.ke = view->key_exps;
  a.ve = view->value_exps;
  a.bt = block_table;
  a.seq_lens = seq_lens;
  a.out = output;
  a.scale_log2 = p->scale * kLog2e;
  a.hd = p->head_size;
  a.num_seqs = p->num_seqs;
  a.max_blocks = p->max_blocks_per_seq;
  a.block_size = p->block_size;
  a.kvh = p->num_kv_heads;
  a.H = p->num_query_heads;
  a.G = p->queries_per_kv;
  a.chunks = head_chunks(a.G);
  a.Gc = heads_per_chunk(a.G);
  a.part_tiles = sp.balanced ? 0 : sp.part / (q8 ? 32 : 16);
  a.max_parts = sp.max_parts;
  a.window = view->window;
  a.first = view->first_tokens;
  a.bs_shift = (a.block_size & (a.block_size - 1)) == 0 ? __builtin_ctz(a.block_size) : -1;
  a.num_blocks = static_cast<uint32_t>(std::min<int64_t>(p->num_blocks, int64_t{1} << 31));
  const int w = q8 ? 1 : 2;  // bytes of a cached value
  a.k_sb = static_cast<uint32_t>(p->k_stride_block * w);
  a.v_sb = static_cast<uint32_t>(p->v_stride_block * w);
  a.k_st = static_cast<uint32_t>(p->k_stride_token * w);
  a.v_st = static_cast<uint32_t>(p->v_stride_token * w);
  a.k_sh = p->k_stride_head * w;
  a.v_sh = p->v_stride_head * w;
  a.ke_sb = view->ke_stride_block; a.ke_sh = view->ke_stride_head;
  a.ke_st = view->ke_stride_token;
  a.ve_sb = view->ve_stride_block; a.ve_sh = view->ve_stride_head;
  a.ve_st = view->ve_stride_token;
  a.q_st = p->q_stride_token; a.q_sh = p->q_stride_head;
  a.o_st = p->o_stride_token; a.o_sh = p->o_stride_head;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool bf = p->dtype == VAA_DTYPE_BF16;
  switch (padded_head(p->head_size)) {
    case 32: return launch_d<32>(a, sp, bf, q8, s);
    case 64: return launch_d<64>(a, sp, bf, q8, s);
    case 96: return launch_d<96>(a, sp, bf, q8, s);
    default: return launch_d<128>(a, sp, bf, q8, s);
  }
}
