// Chunked-prefill attention over a cache as vaa_kv_view describes it: 16-bit or
// e4m3 rows, the whole context or a sliding window behind a few first tokens.
//
//   out[t, h] = sum_j softmax_j(scale q[t, h] . K_j) V_j   over the keys
//   j <= p,  j < first or j > p - window,   p = positions[t]
//
// Bound by the matrix cores where the chunk is long, by latency where it is short.
//
// Work: a workgroup takes 128 query rows of one kv head, a row being a (token, head
// of the group) pair with the heads fastest, so that every GQA group size fills
// the rows; each of its 4 waves takes 32 rows.  For each sequence among its tokens
// (normally one) it walks the 64-key tiles that any of its rows sees: those of the
// first tokens, then those from the oldest key in a window to the youngest row.
// Few rows: the tiles are dealt to several workgroups (grid y) and merged.
//   S^T[64 keys x 32 rows] = K Q^T,  P = exp2(S scale log2e - m),
//   O^T[D x 32 rows] += V^T P^T      on 32x32x16 MFMAs; a lane owns one row.
//
// e4m3 rows pass through registers: the next tile's codes are loaded before this
// tile's math and written to LDS as 16-bit values behind it.  K becomes c 2^(b-127)
// in the query's type, exactly.  V becomes fp16 for both types, relative to the
// largest exponent E seen so far: c 2^(b - E), exact but for values 2^14 below the
// largest row.  P can then be one fp16 value (11 bits) where a bf16 product needs the
// pair hi + lo, and a third of the MFMAs is saved.  E is the workgroup's: the
// accumulators are rescaled when it grows, as they are when the maximum does, and
// in a tile that makes it grow each 16-key group brings its own E_g, whose 2^(E_g - E)
// goes into the group's P.
//
// 16-bit rows go to LDS by direct loads, as in the paged prefill.
//
// Measured (heads 32 on 8 of 128, blocks of 16): 4 x 512 tokens over 2048, e4m3, bf16
// 117 us, 660 TFLOP/s (62 us at a large product's rate); 2 x 2048 tokens of which each
// sees a window of 4096 and 4 first tokens, bf16 390 us, 705 TFLOP/s; the same over e4m3
// rows about as long.  64 accumulators, Q, a tile's scores and P fill the 256 registers
// that two waves a SIMD leave, so that a wave has 32 rows and each K and V tile is read
// from LDS once for every 32: LDS reads, the exponentials and the MFMAs take about the
// same time each, and the two waves hide part of one beneath the other.
#include "fp8.h"
#include "kv_view.h"
#include "prefill_tile.h"

#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

namespace vaa {
namespace {

constexpr int kRows = 128;    // query rows of a workgroup
constexpr int kWavesV = 4;
constexpr int kThreadsV = kWavesV * kWave;
constexpr int kKT = 64;       // keys per tile: a 16-key group per wave
constexpr int kXcds = 8;
constexpr int kMaxSplits = 64;
// A tile's time in the partials that are written and read back in it: 1.5 us, 2 MB/us.
constexpr int64_t kTileBytes = 3 << 20;
constexpr float kRescale = 8.f;     // lazy rescale: P stays below 2^8

struct Args {
  const uint16_t* q;
  const char* kc;
  const char* vc;
  const uint8_t* ke;
  const uint8_t* ve;
  const int32_t* bt;
  const int32_t* tok_seq;
  const int32_t* pos;
  uint16_t* out;
  float* ws_acc;  // [row (token * H + head)][split][D], normalised
  float* ws_lse;  // [row][split], log2 domain; -inf: saw nothing
  float scale_log2;
  int hd, num_tokens, num_seqs, max_blocks, block_size, kvh, H, G;
  int window, first, n_splits;
  int bs_shift;  // log2(block_size) where it is a power of two, else -1
  int tiles_x, padded;  // query tiles; workgroups in use (a multiple of 8)
  uint32_t num_blocks;  // at most 2^31: block ids are 32-bit
  // Bytes.  Block and token strides are below 2^32 and 2^25, so that a row's offset
  // takes 32-bit factors.
  uint32_t k_sb, k_st, v_sb, v_st;
  int64_t k_sh, v_sh;
  int64_t ke_sb, ke_sh, ke_st, ve_sb, ve_sh, ve_st;
  int64_t q_st, q_sh, o_st, o_sh;                    // elements
};

template <int D, bool Q8>
struct Cfg {
  static constexpr int CH = D / 8;     // 16-byte chunks of a 16-bit LDS row
  static constexpr int NK = D / 16;    // QK steps
  static constexpr int NDT = D / 32;   // PV dim tiles
  static constexpr int TILE = kKT * D;
  static constexpr int ROWB = D * 2;
  static constexpr int GCH = Q8 ? D / 16 : D / 8;  // 16-byte chunks of a cached row
  static constexpr int NI = (16 * GCH + kWave - 1) / kWave;  // loads per lane per group
};

// The bits of x, out of the compiler's sight: the file is built as if there were no
// NaN, and a comparison that it sees would be made one that a NaN fails.
__device__ __forceinline__ uint32_t laundered(float x) {
  uint32_t u = __float_as_uint(x);
  asm volatile("" : "+v"(u));
  return u;
}

// What the workgroup keeps in LDS beside the tiles.
struct Shared {
  int red[3][kWavesV];
  int bad[kWavesV];  // waves whose O^T is not finite
  uint64_t ok[2];   // per buffer: the tile's keys that are in LDS (the others are zeros)
  uint32_t ev[2];   // Q8: byte w, the exponent byte that 16-key group w's V is relative to
};

__device__ __forceinline__ uint64_t low64(int n) {
  return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1ull;
}
__device__ __forceinline__ uint32_t low16(int n) {
  return n <= 0 ? 0u : n >= 16 ? 0xFFFFu : (1u << n) - 1u;
}

// A wave's next 16-key group, on its way to LDS (Q8: through these registers).
template <int D, bool Q8>
struct Group {
  static constexpr int N = Q8 ? Cfg<D, Q8>::NI : 1;
  u32x4 k[N], v[N];
  uint32_t ke[N], ve[N];
  uint32_t ok;  // bit r: row r is read
};

// The keys that any row of the workgroup sees: below kv_len, and below first or
// from lo on.
struct Range {
  int kv_len, first, lo;
};

__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>(
      (const __attribute__((address_space(3))) char*)p));
}

struct Window {
  int base, vals;  // lane i: table entry base + i, or -1
};

// The lane, computed anew (two instructions) instead of kept in a register: the
// accumulators leave few, and one that is spilled in the loop waits for the loads.
__device__ __forceinline__ int lane_now() {
  int x;
  asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(x));
  return x;
}

// This lane's piece of a 16-key group for load i: row, and byte offset in the cached
// row of its K and V chunk.  16-bit pieces are the ones that the direct load's slot
// holds.
struct Piece {
  uint32_t row, k, v;
  bool in;  // Q8: the piece lies in the group (D = 96 and 32 leave some over)
};
template <int D, bool Q8>
__device__ __forceinline__ Piece piece(uint32_t i, uint32_t lane) {
  using C = Cfg<D, Q8>;
  uint32_t r, c;
  if constexpr (kWave % C::GCH == 0) {
    r = lane / C::GCH + i * (kWave / C::GCH);
    c = lane % C::GCH;
  } else {
    r = (64 * i + lane) / C::GCH;
    c = (64 * i + lane) % C::GCH;
  }
  if constexpr (Q8)
    return {r & 15, 16 * c, 16 * c, r < 16};
  else
    return {r, 16 * (c ^ swzk<D>(r)), 16 * (c ^ swz<D>(r)), true};
}

// Starts the loads of keys k0 .. k0 + 15, this wave's group of a tile.  Rows that no
// row of the workgroup sees, or in a missing block, become zeros.
template <int D, bool Q8, bool kAny>
__device__ __forceinline__ void fetch(const Args& a, const int32_t* bts, int kvh, int k0,
                                      const Range& rg, int wave, Window& w, f16* kd, f16* vd,
                                      Group<D, Q8>& gr) {
  using C = Cfg<D, Q8>;
  const int lane = lane_now();
  const u32x4 z = {0u, 0u, 0u, 0u};
  const char* kb = a.kc + kvh * a.k_sh;
  const char* vb = a.vc + kvh * a.v_sh;
  char* kl = reinterpret_cast<char*>(kd) + 1024 * (wave * C::NI);
  char* vl = reinterpret_cast<char*>(vd) + 1024 * (wave * C::NI);
  const uint32_t ka = __builtin_amdgcn_readfirstlane(lds_address(kl));
  const uint32_t va = __builtin_amdgcn_readfirstlane(lds_address(vl));
  // The rows that are read; all of them but at the ends of what is seen.
  uint32_t ok = 0xFFFFu;
  if (k0 + 16 > rg.kv_len || (k0 < rg.lo && k0 + 16 > rg.first))
    ok = low16(rg.kv_len - k0) & (~low16(rg.lo - k0) | low16(rg.first - k0));
  const bool any_block = kAny && a.block_size % 16 != 0;
  const int bi = a.bs_shift >= 0 ? k0 >> a.bs_shift : k0 / a.block_size;
  if (ok) {
    const int last = any_block ? min(k0 + 15, rg.kv_len - 1) / a.block_size : bi;
    if (bi < w.base || last >= w.base + kWave) {
      w.base = bi;
      const int e = bi + lane;
      w.vals = e < a.max_blocks ? bts[e] : -1;
    }
  }
  const uint32_t row_bytes = a.hd * (Q8 ? 1 : 2);  // kAny: pieces past them are zeros
  if (any_block) {
    // Rows that find their own blocks.
    auto row_at = [&](int r, int64_t& p, int& rin) {
      const int tok = k0 + r, b = tok / a.block_size;
      const int e = __shfl(w.vals, max(0, min(kWave - 1, b - w.base)), kWave);
      p = e;
      rin = tok - b * a.block_size;
      return ((ok >> r) & 1u) && static_cast<uint32_t>(e) < a.num_blocks;
    };
    int64_t p;
    int rin;
    ok = static_cast<uint32_t>(__builtin_amdgcn_ballot_w64(row_at(lane & 15, p, rin))) & 0xFFFFu;
#pragma unroll
    for (int i = 0; i < C::NI; ++i) {
      const Piece pc = piece<D, Q8>(i, lane);
      const bool good = row_at(pc.row, p, rin) && pc.in;
      const char* ks = kb + p * a.k_sb + static_cast<int64_t>(rin) * a.k_st + pc.k;
      const char* vs = vb + p * a.v_sb + static_cast<int64_t>(rin) * a.v_st + pc.v;
      const bool kin = good && pc.k < row_bytes, vin = good && pc.v < row_bytes;
      if constexpr (Q8) {
        gr.k[i] = kin ? ld16(ks) : z;
        gr.v[i] = vin ? ld16(vs) : z;
        gr.ke[i] = good ? a.ke[p * a.ke_sb + kvh * a.ke_sh + rin * a.ke_st] : 0;
        gr.ve[i] = good ? a.ve[p * a.ve_sb + kvh * a.ve_sh + rin * a.ve_st] : 0;
      } else {
        if (kin) dma16(ks, ka + 1024 * i);
        else *reinterpret_cast<u32x4*>(kl + 1024 * i + 16 * lane) = z;
        if (vin) dma16(vs, va + 1024 * i);
        else *reinterpret_cast<u32x4*>(vl + 1024 * i + 16 * lane) = z;
      }
    }
    gr.ok = ok;
    return;
  }
  // The group lies in one block.
  uint32_t phys = 0;
  if (ok) {
    phys = static_cast<uint32_t>(__builtin_amdgcn_readlane(w.vals, bi - w.base));
    if (phys >= a.num_blocks) {
      ok = 0;
      phys = 0;
    }
  }
  const uint32_t rin = k0 - bi * a.block_size;
  kb += static_cast<uint64_t>(phys) * a.k_sb + rin * a.k_st;
  vb += static_cast<uint64_t>(phys) * a.v_sb + rin * a.v_st;
  gr.ok = ok;
  if constexpr (Q8) {
    const uint8_t* ke = a.ke + phys * a.ke_sb + kvh * a.ke_sh + rin * a.ke_st;
    const uint8_t* ve = a.ve + phys * a.ve_sb + kvh * a.ve_sh + rin * a.ve_st;
    constexpr bool kFull = !kAny && 16 * C::GCH % kWave == 0;  // every lane's pieces lie in the rows
#pragma unroll
    for (int i = 0; i < C::NI; ++i) {
      const Piece pc = piece<D, Q8>(i, lane);
      const bool good = ((ok >> pc.row) & 1u) && pc.in;
      gr.k[i] = z;
      gr.v[i] = z;
      gr.ke[i] = 0;
      gr.ve[i] = 0;
      if (good && (kFull || pc.k < row_bytes)) {
        gr.k[i] = ld16(kb + pc.row * a.k_st + pc.k);
        gr.v[i] = ld16(vb + pc.row * a.v_st + pc.v);
      }
      if (good) {
        gr.ke[i] = ke[pc.row * a.ke_st];
        gr.ve[i] = ve[pc.row * a.ve_st];
      }
    }
  } else {
    if (!kAny && ok == 0xFFFFu) {
#pragma unroll
      for (int i = 0; i < C::NI; ++i) {
        const Piece pc = piece<D, Q8>(i, lane);
        if constexpr (kWave % C::GCH == 0) {  // rows of load i: the first load's, further on
          const uint32_t up = i * (kWave / C::GCH), r0 = pc.row - up;
          dma16s(kb + up * a.k_st, r0 * a.k_st + pc.k, ka + 1024 * i);
          dma16s(vb + up * a.v_st, r0 * a.v_st + pc.v, va + 1024 * i);
        } else {
          dma16s(kb, pc.row * a.k_st + pc.k, ka + 1024 * i);
          dma16s(vb, pc.row * a.v_st + pc.v, va + 1024 * i);
        }
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < C::NI; ++i) {
      const Piece pc = piece<D, Q8>(i, lane);
      const bool good = (ok >> pc.row) & 1u;
      if (good && (!kAny || pc.k < row_bytes))
        dma16(kb + pc.row * a.k_st + pc.k, ka + 1024 * i);
      else
        *reinterpret_cast<u32x4*>(kl + 1024 * i + 16 * lane) = z;
      if (good && (!kAny || pc.v < row_bytes))
        dma16(vb + pc.row * a.v_st + pc.v, va + 1024 * i);
      else
        *reinterpret_cast<u32x4*>(vl + 1024 * i + 16 * lane) = z;
    }
  }
}

// Q8: the group's codes as 16-bit values in LDS.  Either way its rows in sh.
template <int D, typename T, bool Q8>
__device__ __forceinline__ void deliver(const Group<D, Q8>& gr, int wave, f16* kd, f16* vd,
                                        Shared& sh, int buf, int e_run) {
  using C = Cfg<D, Q8>;
  const int lane = lane_now();
  if constexpr (Q8) {
    uint32_t top = gr.ve[0];
#pragma unroll
    for (int i = 1; i < C::NI; ++i) top = max(top, gr.ve[i]);
    int eg = e_run;
    if (__builtin_amdgcn_ballot_w64(static_cast<int>(top) > e_run) != 0)
      eg = __builtin_amdgcn_readfirstlane(max(e_run, wave_max_i(static_cast<int>(top))));
#pragma unroll
    for (int i = 0; i < C::NI; ++i) {
      const Piece pc = piece<D, Q8>(i, lane);
      if (!pc.in) continue;
      const int ch = pc.k / 16, R = 16 * wave + pc.row;
      const float ks = scale_of(gr.ke[i]);
      const float vs = __uint_as_float(
          static_cast<uint32_t>(max(1, 127 + static_cast<int>(gr.ve[i]) - eg)) << 23);
      char* kr = reinterpret_cast<char*>(kd) + R * C::ROWB;
      char* vr = reinterpret_cast<char*>(vd) + R * C::ROWB;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        *reinterpret_cast<u32x4*>(kr + ((2 * ch + j) ^ swzk<D>(R)) * 16) =
            deq8<T>(gr.k[i][2 * j], gr.k[i][2 * j + 1], ks);
        *reinterpret_cast<u32x4*>(vr + ((2 * ch + j) ^ swz<D>(R)) * 16) =
            deq8<f16>(gr.v[i][2 * j], gr.v[i][2 * j + 1], vs);
      }
    }
    if (lane == 0) reinterpret_cast<uint8_t*>(&sh.ev[buf])[wave] = static_cast<uint8_t>(eg);
  }
  if (lane == 0) reinterpret_cast<uint16_t*>(&sh.ok[buf])[wave] = static_cast<uint16_t>(gr.ok);
}

// Per-lane LDS addresses of the MFMA operands: K's for step s, V's for dim tile dt.
// The rows are a power of two wide but for D = 96, and the chunk swizzle is an XOR,
// so the address of a later step is the first one's XOR a constant: one register
// instead of one per step (the accumulators leave few).
template <int D>
struct Lanes {
  static constexpr bool XOR = D != 96;
  int k[XOR ? 1 : D / 16], v[XOR ? 1 : D / 32];
  __device__ __forceinline__ int kaddr(int s) const { return XOR ? k[0] ^ (16 * s) : k[s]; }
  __device__ __forceinline__ int vaddr(int dt) const { return XOR ? v[0] ^ (64 * dt) : v[dt]; }
};

// A row's state: its running maximum (log2 domain), its part of the sum, O^T.
template <int D>
struct State {
  float m = -INFINITY, l = 0.f;
  f32x16 acc[D / 32];
  int e = 0;  // Q8: exponent byte that acc is relative to
};

// What a row sees of the sequence: keys up to lim, from lo on or below first.  A row
// that is never written sees everything, so that it asks for no mask.
struct Sees {
  int lim, lo;
};

constexpr int kAheadK = 4, kAheadV = 4;  // LDS operand reads ahead of their MFMAs

// One tile for this wave's 32 rows.  kCareful: V may hold infinities or NaN in keys
// that some rows do not see, and 0 * NaN in the product would reach those rows too.
// The product takes them as zeros, and a second one of two counts says which rows
// see them: +inf counts 1, -inf counts 32 and NaN both, 16 keys at a time.
template <int D, typename T, bool Q8, bool kCareful>
__device__ __forceinline__ void tile_math(const Args& a, const f16* kt, const f16* vt, int key0,
                                          const Sees& see, const Shared& sh, int buf, int hb,
                                          Lanes<D> L, const u32x4 (&qb)[D / 16],
                                          State<D>& st) {
  using C = Cfg<D, Q8>;
  // The XORs stay in the loop.
  if constexpr (Lanes<D>::XOR) asm volatile("" : "+v"(L.k[0]), "+v"(L.v[0]));
  using PT = typename std::conditional<Q8, f16, T>::type;  // type of V and P
  using X4 = typename Elem<PT>::x4;
  using P8 = typename Elem<PT>::x8;
  using X8 = typename Elem<T>::x8;
  constexpr bool kPair = !Q8 && Elem<T>::kSplitP;
  // Does every row of the wave see the whole tile, by position?  (A wave that sees
  // nothing of it goes through all the same: a way around the products would keep a
  // second set of accumulators, and a copy of them per tile.)
  uint64_t seen = ~0ull;
  const bool inside = see.lim - key0 >= kKT - 1 && (see.lo <= key0 || a.first - key0 >= kKT);
  const bool whole = __builtin_amdgcn_ballot_w64(inside) == ~0ull;
  if (!whole)
    seen = low64(see.lim + 1 - key0) & (~low64(see.lo - key0) | low64(a.first - key0));
  // What the tile holds, and its exponents: used behind the first product.
  const uint64_t held = sh.ok[buf];
  const uint32_t held_e = Q8 ? sh.ev[buf] : 0;

  const char* kbytes = reinterpret_cast<const char*>(kt);
  const char* vbytes = reinterpret_cast<const char*>(vt);
  constexpr int NKR = 2 * C::NK, NPV = C::NDT * 4;
  u32x4 kA[NKR];
  auto kread = [&](int i) {
    kA[i] = *reinterpret_cast<const u32x4*>(kbytes + L.kaddr(i >> 1) + 32 * (i & 1) * C::ROWB);
  };
#pragma unroll
  for (int i = 0; i < kAheadK && i < NKR; ++i) kread(i);
  __builtin_amdgcn_sched_barrier(0);
  f32x16 s[2];
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int r = 0; r < 16; ++r) s[j][r] = 0.f;
  // Products go before the other workgroup's exponentials: 4 x 512 over 2048, 16-bit
  // fp16 115 -> 109 us with this and P beneath the products.
  __builtin_amdgcn_s_setprio(1);
#pragma unroll
  for (int i = 0; i < NKR; ++i) {
    if (i + kAheadK < NKR) kread(i + kAheadK);
    s[i & 1] = Elem<T>::mfma32x32x16(__builtin_bit_cast(X8, kA[i]),
                                     __builtin_bit_cast(X8, qb[i >> 1]), s[i & 1]);
    __builtin_amdgcn_sched_barrier(0);
  }
  __builtin_amdgcn_s_setprio(0);
  X4 vlo[NPV], vhi[NPV];
  auto vread = [&](int i) {
    const int g = i / C::NDT, dt = i % C::NDT;
    const f16* vp = reinterpret_cast<const f16*>(vbytes + L.vaddr(dt) + 16 * g * C::ROWB);
    vlo[i] = lds_tr4<PT>(vp);
    vhi[i] = lds_tr4<PT>(vp + 8 * D);
  };
#pragma unroll
  for (int i = 0; i < kAheadV && i < NPV; ++i) vread(i);
  __builtin_amdgcn_sched_barrier(0);
  // Lane holds keys 32j + 8(r/4) + 4hb + r%4 of its row.
  seen &= held;
  if (!whole || __builtin_amdgcn_ballot_w64(held == ~0ull) != ~0ull) {
    const uint64_t mine = seen >> (4 * hb);
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (!((static_cast<uint32_t>(mine >> (32 * j)) >> (8 * (r >> 2) + (r & 3))) & 1u))
          s[j][r] = -INFINITY;
  }
  float mx0 = fmaxf(s[0][0], s[0][1]), mx1 = fmaxf(s[1][0], s[1][1]);
#pragma unroll
  for (int r = 2; r < 16; r += 2) {
    mx0 = fmaxf(fmaxf(mx0, s[0][r]), s[0][r + 1]);
    mx1 = fmaxf(fmaxf(mx1, s[1][r]), s[1][r + 1]);
  }
  const float mx = half_max(fmaxf(mx0, mx1)) * a.scale_log2;
  if (__builtin_amdgcn_ballot_w64(mx > st.m + kRescale) != 0 && mx > st.m) {
    const float alpha = fast_exp2(st.m - mx);  // 0 when m = -inf
    st.l *= alpha;
#pragma unroll
    for (int dt = 0; dt < C::NDT; ++dt) st.acc[dt] *= alpha;
    st.m = mx;
  }
  const float sub = st.m == -INFINITY ? 0.f : st.m;
  bool even = true;  // the groups' V share the exponent that acc is relative to
  uint32_t ev = 0;
  if constexpr (Q8) {
    ev = __builtin_amdgcn_readfirstlane(static_cast<int>(held_e));
    const int top = max(max(ev >> 24, (ev >> 16) & 255), max((ev >> 8) & 255, ev & 255));
    if (top > st.e) {
      const float alpha = __uint_as_float(static_cast<uint32_t>(max(1, 127 + st.e - top)) << 23);
#pragma unroll
      for (int dt = 0; dt < C::NDT; ++dt) st.acc[dt] *= alpha;
      st.e = top;
    }
    even = ev == static_cast<uint32_t>(st.e) * 0x01010101u;
  }
  if (!even) {
    // A tile that raises E: the product takes P 2^(E_g - E), the sum P itself.
    float l = 0.f;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) l += fast_exp2(fmaf(s[j][r], a.scale_log2, -sub));
    st.l += l;
  }
  P8 pb[4], pl[4];
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef decltype(Elem<PT>::from_f(0.f)) E2 __attribute__((ext_vector_type(2)));
  float l0 = 0.f, l1 = 0.f;
  // P of the lane's pair i of group g.
  auto put = [&](int g, int i) {
    float sg = sub;
    if constexpr (Q8) sg += static_cast<float>(st.e - static_cast<int>((ev >> (8 * g)) & 255));
    const int j = g >> 1, r = 8 * (g & 1) + 2 * i;
    const f32x2 p = {fast_exp2(fmaf(s[j][r], a.scale_log2, -sg)),
                     fast_exp2(fmaf(s[j][r + 1], a.scale_log2, -sg))};
    const E2 h = __builtin_convertvector(p, E2);
    pb[g][2 * i] = h[0];
    pb[g][2 * i + 1] = h[1];
    float& l = i & 1 ? l1 : l0;
    if constexpr (kPair) {
      const f32x2 back = {Elem<PT>::to_f(h[0]), Elem<PT>::to_f(h[1])};
      const E2 lo = __builtin_convertvector(f32x2{p[0] - back[0], p[1] - back[1]}, E2);
      pl[g][2 * i] = lo[0];
      pl[g][2 * i + 1] = lo[1];
      l += p[0] + p[1];
    } else {
      // The sum takes P as the product sees it, two values per v_dot2_f32_f16.
      typedef _Float16 h2 __attribute__((ext_vector_type(2)));
      const h2 one = {static_cast<_Float16>(1.f), static_cast<_Float16>(1.f)};
      l = __builtin_amdgcn_fdot2(h2{h[0], h[1]}, one, l, false);
    }
  };
#pragma unroll
  for (int i = 0; i < 4; ++i) put(0, i);
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_setprio(1);
#pragma unroll
  for (int i = 0; i < NPV; ++i) {
    if (i + kAheadV < NPV) vread(i + kAheadV);
    const int g = i / C::NDT, dt = i % C::NDT;
    P8 va = __builtin_shufflevector(vlo[i], vhi[i], 0, 1, 2, 3, 4, 5, 6, 7);
    if constexpr (kCareful) {
      // In integers, out of the compiler's sight like laundered().
      constexpr uint32_t kExp = std::is_same<PT, bf16>::value ? 0x7F80u : 0x7C00u;
      constexpr uint32_t kFrac = 0x7FFFu - kExp;
      u32x4 w = __builtin_bit_cast(u32x4, va);
      P8 odd, sees;
      const uint64_t mine = seen >> (16 * g + 4 * hb);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        uint32_t bits = (w[e >> 1] >> (16 * (e & 1))) & 0xFFFFu;
        asm volatile("" : "+v"(bits));
        const bool bad = (bits & kExp) == kExp;
        const float count = !bad ? 0.f : (bits & kFrac) ? 33.f : (bits & 0x8000u) ? 32.f : 1.f;
        odd[e] = Elem<PT>::from_f(count);
        sees[e] = Elem<PT>::from_f((mine >> (8 * (e >> 2) + (e & 3))) & 1u ? 1.f : 0.f);
        if (bad) w[e >> 1] &= 0xFFFFu << (16 * (~e & 1));
      }
      va = __builtin_bit_cast(P8, w);
      f32x16 n;
#pragma unroll
      for (int r = 0; r < 16; ++r) n[r] = 0.f;
      n = Elem<PT>::mfma32x32x16(odd, sees, n);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int c = static_cast<int>(n[r]);
        float x = st.acc[dt][r];
        if (c & 31) asm volatile("v_add_f32 %0, %1, %0" : "+v"(x) : "v"(0x7F800000));
        if (c >> 5) asm volatile("v_add_f32 %0, %1, %0" : "+v"(x) : "v"(0xFF800000));
        st.acc[dt][r] = x;
      }
    }
    st.acc[dt] = Elem<PT>::mfma32x32x16(va, pb[g], st.acc[dt]);
    if constexpr (kPair) st.acc[dt] = Elem<PT>::mfma32x32x16(va, pl[g], st.acc[dt]);
    // The next group's P beneath this one's products.
    if (g < 3)
#pragma unroll
      for (int e = 4 * dt / C::NDT; e < 4 * (dt + 1) / C::NDT; ++e) put(g + 1, e);
    __builtin_amdgcn_sched_barrier(0);
  }
  if (even) st.l += l0 + l1;
  __builtin_amdgcn_s_setprio(0);
}

// A query row's sequence and position; false where the row is left unwritten.
__device__ __forceinline__ bool row_place(const Args& a, int64_t tok, int& seq, int& pos) {
  seq = a.tok_seq[tok];
  pos = a.pos[tok];
  return seq >= 0 && seq < a.num_seqs && pos >= 0 &&
         (static_cast<int64_t>(pos) + a.block_size) / a.block_size <= a.max_blocks;
}

// This lane's query row (lanes l and l + 32 share one): its token, head, sequence
// and position; ok: it is written.
struct Row {
  int64_t tok;
  int head, seq, pos;
  bool ok;
};
__device__ __forceinline__ Row row_of(const Args& a, int tile, int kvh, int wave, int lane) {
  const uint32_t n_rows = static_cast<uint32_t>(a.num_tokens) * a.G;  // below 2^30 + kRows
  uint32_t rho = static_cast<uint32_t>(tile) * kRows + 32 * wave + (lane & 31);
  const bool in = rho < n_rows;
  rho = in ? rho : 0;
  Row r;
  r.tok = rho / static_cast<uint32_t>(a.G);
  r.head = kvh * a.G + static_cast<int>(rho % static_cast<uint32_t>(a.G));
  r.ok = row_place(a, r.tok, r.seq, r.pos) && in;
  return r;
}

// All keys of this workgroup's split for its rows, sequence by sequence.  Rows and Q
// are read here, so that neither lives on behind the loop.
template <int D, typename T, bool Q8, bool kAny, bool kCareful>
__device__ __forceinline__ void walk(const Args& a, f16* ks, f16* vs, Shared& sh, int tile,
                                     int kvh, int split, int wave, State<D>& st) {
  using C = Cfg<D, Q8>;
  const int lane = lane_now(), hb = lane >> 5;
  Lanes<D> L;
  u32x4 qb[C::NK];
  int tseq, tpos;
  bool row_ok;
  {
    const Row r = row_of(a, tile, kvh, wave, lane);
    tseq = r.seq;
    tpos = r.pos;
    row_ok = r.ok;
    const uint16_t* qp = a.q + r.tok * a.q_st + r.head * a.q_sh + hb * (D / 2);
#pragma unroll
    for (int s = 0; s < C::NK; ++s)
      qb[s] = !kAny || hb * (D / 2) + 8 * s < a.hd ? ld16(qp + 8 * s) : u32x4{0u, 0u, 0u, 0u};
    const int qj = lane & 31;
#pragma unroll
    for (int s = 0; s < (Lanes<D>::XOR ? 1 : C::NK); ++s)
      L.k[s] = qj * C::ROWB + ((hb * (C::CH / 2) + s) ^ swzk<D>(qj)) * 16;
    const int g16 = lane >> 4, i16 = lane & 15;
    const int rv = 4 * hb + (i16 >> 2), j4 = i16 & 3;
#pragma unroll
    for (int dt = 0; dt < (Lanes<D>::XOR ? 1 : C::NDT); ++dt)
      L.v[dt] = rv * C::ROWB + ((4 * dt + 2 * (g16 & 1) + (j4 >> 1)) ^ swz<D>(rv)) * 16 +
                (j4 & 1) * 8;
  }
  st.m = -INFINITY;
  st.l = 0.f;
  st.e = 0;
#pragma unroll
  for (int dt = 0; dt < C::NDT; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) st.acc[dt][r] = 0.f;

  int e_run = 0;  // Q8: largest V exponent byte so far, the same in every wave
  bool done = !row_ok;
  while (true) {
    // The next sequence among the unfinished rows, and the positions it has here.
    int s = wave_min_i(done ? INT32_MAX : tseq);
    if (lane == 0) sh.red[0][wave] = s;
    lds_bar();
    s = sh.red[0][0];
#pragma unroll
    for (int w = 1; w < kWavesV; ++w) s = min(s, sh.red[0][w]);
    s = __builtin_amdgcn_readfirstlane(s);
    if (s == INT32_MAX) break;
    const bool active = !done && tseq == s;
    int pmax = wave_max_i(active ? tpos : -1), pmin = wave_min_i(active ? tpos : INT32_MAX);
    if (lane == 0) {
      sh.red[1][wave] = pmax;
      sh.red[2][wave] = pmin;
    }
    lds_bar();
    pmax = sh.red[1][0];
    pmin = sh.red[2][0];
#pragma unroll
    for (int w = 1; w < kWavesV; ++w) {
      pmax = max(pmax, sh.red[1][w]);
      pmin = min(pmin, sh.red[2][w]);
    }
    pmax = __builtin_amdgcn_readfirstlane(pmax);
    pmin = __builtin_amdgcn_readfirstlane(pmin);
    const int32_t* bts = a.bt + static_cast<int64_t>(s) * a.max_blocks;
    Sees see{row_ok ? -1 : INT32_MAX - 1, 0};
    if (active) {
      see.lim = tpos;
      see.lo = a.window > 0 ? max(0, tpos + 1 - a.window) : 0;
    }
    Range rg;
    rg.kv_len = pmax + 1;
    rg.lo = a.window > 0 ? max(0, pmin + 1 - a.window) : 0;
    rg.first = a.first;
    const int nf = (min(a.first, rg.lo) + kKT - 1) / kKT;
    const int skip = max(0, rg.lo / kKT - nf);
    const int n = (rg.kv_len + kKT - 1) / kKT - skip;
    const int share = (n + a.n_splits - 1) / a.n_splits;
    const int t_lo = split * share, t_hi = min(n, t_lo + share);
    if (t_lo < t_hi) {
      auto key_of = [&](int t) { return (t < nf ? t : t + skip) * kKT; };
      Window w{-(1 << 30), -1};
      Group<D, Q8> gr;
      auto get = [&](int t, int buf) {
        if (t < t_hi)
          fetch<D, Q8, kAny>(a, bts, kvh, key_of(t) + 16 * wave, rg, wave, w, ks + buf * C::TILE, vs + buf * C::TILE, gr);
      };
      // The tile is in LDS: codes converted, direct loads landed, for every wave.
      auto put = [&](int t, int buf) {
        if (t < t_hi)
          deliver<D, T, Q8>(gr, wave, ks + buf * C::TILE, vs + buf * C::TILE, sh, buf, e_run);
        wait_all();
        __builtin_amdgcn_s_barrier();
        if (Q8 && t < t_hi) {
          const uint32_t ev = __builtin_amdgcn_readfirstlane(static_cast<int>(sh.ev[buf]));
          e_run = max(e_run, static_cast<int>(max(max(ev >> 24, (ev >> 16) & 255),
                                                  max((ev >> 8) & 255, ev & 255))));
        }
      };
      get(t_lo, 0);
      put(t_lo, 0);
      for (int t = t_lo, buf = 0; t < t_hi; ++t, buf ^= 1) {
        get(t + 1, buf ^ 1);
        tile_math<D, T, Q8, kCareful>(a, ks + buf * C::TILE, vs + buf * C::TILE, key_of(t), see, sh,
                                      buf, hb, L, qb, st);
        put(t + 1, buf ^ 1);
      }
    }
    done = done || active;
  }
}

template <int D, typename T, bool Q8, bool kAny>
__global__ void __launch_bounds__(kThreadsV) __attribute__((amdgpu_waves_per_eu(2, 2)))
prefill_view_kernel(Args a) {
  using C = Cfg<D, Q8>;
  __shared__ __align__(16) f16 ks[2 * C::TILE];
  __shared__ __align__(16) f16 vs[2 * C::TILE];
  __shared__ Shared sh;

  // Consecutive workgroup ids go to the 8 XCDs in turn; each XCD gets a contiguous
  // range of (kv head, query tile), whose tiles read the same keys, the second
  // half backwards, so that a CU pairs an early tile of a chunk with a late one.
  const int id = blockIdx.x;
  const int per_xcd = a.padded / kXcds;
  int kx = id / kXcds;
  if (kx >= per_xcd / 2) kx = per_xcd - 1 - (kx - per_xcd / 2);
  const int logical = (id % kXcds) * per_xcd + kx;
  if (logical >= a.tiles_x * a.kvh) return;
  const int kvh = logical / a.tiles_x, split = blockIdx.y;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int tile = logical % a.tiles_x;
  State<D> st;
  walk<D, T, Q8, kAny, false>(a, ks, vs, sh, tile, kvh, split, wave, st);
  {
    // An infinity or a NaN in O^T: all over again with care, since it may come from a
    // key that its row does not see.
    uint32_t top = 0;
#pragma unroll
    for (int dt = 0; dt < C::NDT; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = max(top, laundered(st.acc[dt][r]) & 0x7FFFFFFFu);
    // (Rows that are not written count too: they hold what their garbage gives.)
    const bool bad = __builtin_amdgcn_ballot_w64(top >= 0x7F800000u) != 0;
    if (lane_now() == 0) sh.bad[wave] = bad;
    lds_bar();
    int any = 0;
#pragma unroll
    for (int w = 0; w < kWavesV; ++w) any |= sh.bad[w];
    if (__builtin_amdgcn_readfirstlane(any)) {
      walk<D, T, Q8, kAny, true>(a, ks, vs, sh, tile, kvh, split, wave, st);
    }
  }

  const float l = half_sum(st.l);
  const int lane = lane_now(), hb = lane >> 5;
  const Row r = row_of(a, tile, kvh, wave, lane);
  if (!r.ok) return;
  float inv = l > 0.f ? 1.f / l : 0.f;
  const float back = Q8 ? scale_of(static_cast<uint32_t>(max(1, st.e))) : 1.f;
  const int64_t row = r.tok * a.H + r.head;
  if (a.n_splits > 1) {
    float* dst = a.ws_acc + (row * a.n_splits + split) * D;
#pragma unroll
    for (int dt = 0; dt < C::NDT; ++dt)
#pragma unroll
      for (int rg = 0; rg < 4; ++rg) {
        f32x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = st.acc[dt][4 * rg + i] * inv * back;
        *reinterpret_cast<f32x4*>(dst + 32 * dt + 8 * rg + 4 * hb) = v;
      }
    if (hb == 0)
      // A NaN (of a NaN key) is not 0, and reaches the row.
      a.ws_lse[row * a.n_splits + split] =
          laundered(l) != 0u ? st.m + __builtin_log2f(l) : -INFINITY;
    return;
  }
  uint16_t* op = a.out + r.tok * a.o_st + r.head * a.o_sh;
#pragma unroll
  for (int dt = 0; dt < C::NDT; ++dt)
#pragma unroll
    for (int rg = 0; rg < 4; ++rg) {
      typename Elem<T>::x4 o;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = Elem<T>::from_f(st.acc[dt][4 * rg + i] * inv * back);
      const int d = 32 * dt + 8 * rg + 4 * hb;
      if (!kAny || d < a.hd) *reinterpret_cast<typename Elem<T>::x4*>(op + d) = o;
    }
}

// Joins the splits of every row: out = sum_z 2^(lse_z - M) o_z / sum_z 2^(lse_z - M).
// A thread takes four dims of one row.
template <int D, typename T>
__global__ void __launch_bounds__(256) prefill_view_merge_kernel(Args a) {
  constexpr int D4 = D / 4;
  const uint32_t it = blockIdx.x * 256 + threadIdx.x;  // below 2^31: few rows are split
  const int d = 4 * static_cast<int>(it % D4);
  const uint32_t r = it / D4, tok = r / static_cast<uint32_t>(a.H);
  const int64_t row = r;
  if (tok >= static_cast<uint32_t>(a.num_tokens) || d >= a.hd) return;
  int seq, pos;
  if (!row_place(a, tok, seq, pos)) return;
  const float* lse = a.ws_lse + row * a.n_splits;
  const float* src = a.ws_acc + row * a.n_splits * D + d;
  constexpr int kAtOnce = 8;  // loads in flight: the kernel is bound by their latency
  float M = -INFINITY, den = 0.f;
  f32x4 num = {0.f, 0.f, 0.f, 0.f};
  for (int z0 = 0; z0 < a.n_splits; z0 += kAtOnce) {
    float x[kAtOnce];
    f32x4 o[kAtOnce];  // zeros of a split that saw nothing
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int z = min(z0 + i, a.n_splits - 1);
      x[i] = lse[z];
      o[i] = *reinterpret_cast<const f32x4*>(src + z * D);
    }
    float top = M;
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      if (z0 + i >= a.n_splits) {  // the last one again: 0 * inf is not nothing
        x[i] = -INFINITY;
        o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
      top = fmaxf(top, x[i]);
    }
    const float base = top == -INFINITY ? 0.f : top, so = fast_exp2(M - base);
    num *= so;
    den *= so;
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      // -inf: nothing; a NaN goes on.
      const float w = laundered(x[i]) == 0xFF800000u ? 0.f : fast_exp2(x[i] - base);
      num += o[i] * w;
      den += w;
    }
    M = top;
  }
  T* o = reinterpret_cast<T*>(a.out) + tok * a.o_st + (r - tok * a.H) * a.o_sh + d;
  const float inv = den > 0.f ? 1.f / den : 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = Elem<T>::from_f(num[i] * inv);
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

int64_t query_tiles(const vaa_attn_params* p, int num_tokens) {
  return (static_cast<int64_t>(num_tokens) * p->queries_per_kv + kRows - 1) / kRows;
}

// Workgroups over the keys: as many as fill the two slots of every CU, but no more
// than pay.  n splits of T tiles cost T / n tiles and n times the rows' partials, B
// bytes; the sum is least at n^2 = T kTileBytes / B.  Measured (whole call, heads 32 on 8
// of 128 unless said): 64 tokens over 4000 15 splits 30.1 us, 31 37.5 us; over 1000 4
// splits 24.4, 8 23.2, 17 28.7 us; 5 tokens over 4000 15 splits 22.0, 31 20.2, 63 22.3
// us; 8 x 5 tokens over 1000, heads 14 on 2 of 64: 4 splits 49.0, 16 23.9 us.
int plan_splits(const vaa_attn_params* p, const vaa_kv_view* view, int num_tokens) {
  const int64_t wgs = query_tiles(p, num_tokens) * p->num_kv_heads;
  const int64_t cap = static_cast<int64_t>(p->max_blocks_per_seq) * p->block_size;
  int64_t len = p->max_seq_len > 0 ? std::min<int64_t>(p->max_seq_len, cap) : cap;
  if (view->window > 0)
    len = std::min<int64_t>(len, static_cast<int64_t>(view->window) + view->first_tokens +
                                     std::min<int64_t>(num_tokens, kRows));
  const int64_t tiles = (len + kKT - 1) / kKT;
  const int64_t slots = 2 * num_cus();
  int64_t n = wgs > 0 ? slots / wgs : 1;
  const int64_t bytes = static_cast<int64_t>(num_tokens) * p->num_query_heads *
                        padded_head(p->head_size) * sizeof(float);
  n = std::min<int64_t>({n, tiles, kMaxSplits});
  if (n > 1)
    n = std::min(n, static_cast<int64_t>(std::sqrt(static_cast<double>(tiles * kTileBytes) /
                                                   static_cast<double>(bytes))));
  return static_cast<int>(std::max<int64_t>(1, n));
}

int check_prefill(const char* what, const vaa_attn_params* p, const vaa_kv_view* view,
                  int num_tokens) {
  int st = check_view(what, p, view);
  if (st) return st;
  if (num_tokens < 0 || p->num_seqs < 0 || p->max_blocks_per_seq <= 0)
    return fail(VAA_ERR_INVALID_ARG, "%s: num_tokens=%d num_seqs=%d max_blocks_per_seq=%d", what,
                num_tokens, p->num_seqs, p->max_blocks_per_seq);
  if (query_tiles(p, num_tokens) * p->num_kv_heads > (int64_t{1} << 23))
    return fail(VAA_ERR_UNSUPPORTED, "%s: num_tokens=%d: too many query rows", what, num_tokens);
  return VAA_OK;
}

size_t ws_rows(const vaa_attn_params* p, int num_tokens, int splits) {
  return static_cast<size_t>(num_tokens) * p->num_query_heads * splits;
}

template <int D, typename T, bool Q8, bool kAny>
int launch(const Args& a, hipStream_t stream) {
  hipLaunchKernelGGL((prefill_view_kernel<D, T, Q8, kAny>), dim3(a.padded, a.n_splits),
                     dim3(kThreadsV), 0, stream, a);
  int st = check_launch("prefill_view_kernel");
  if (st || a.n_splits <= 1) return st;
  const int64_t items = static_cast<int64_t>(a.num_tokens) * a.H * (D / 4);
  hipLaunchKernelGGL((prefill_view_merge_kernel<D, T>),
                     dim3(static_cast<unsigned>((items + 255) / 256)), dim3(256), 0, stream, a);
  return check_launch("prefill_view_merge_kernel");
}

template <int D>
int launch_d(const Args& a, bool bf, bool q8, hipStream_t s) {
  const bool any = a.hd != D || a.block_size % 16 != 0;
  if (q8) {
    if (any) return bf ? launch<D, bf16, true, true>(a, s) : launch<D, f16, true, true>(a, s);
    return bf ? launch<D, bf16, true, false>(a, s) : launch<D, f16, true, false>(a, s);
  }
  if (any) return bf ? launch<D, bf16, false, true>(a, s) : launch<D, f16, false, true>(a, s);
  return bf ? launch<D, bf16, false, false>(a, s) : launch<D, f16, false, false>(a, s);
}

}  // namespace
}  // namespace vaa

using namespace vaa;

extern "C" size_t vaa_paged_attention_prefill_view_workspace_size(const vaa_attn_params* p,
                                                                  const vaa_kv_view* view,
                                                                  int num_tokens) {
  const char* what = "vaa_paged_attention_prefill_view_workspace_size";
  if (check_prefill(what, p, view, num_tokens) || num_tokens == 0) return 0;
  const int n = plan_splits(p, view, num_tokens);
  return n <= 1 ? 0
                : ws_rows(p, num_tokens, n) * (padded_head(p->head_size) + 1) * sizeof(float);
}

extern "C" int vaa_paged_attention_prefill_view(const vaa_attn_params* p, const vaa_kv_view* view,
                                                const uint16_t* query, const void* key_cache,
                                                const void* value_cache,
                                                const int32_t* block_table,
                                                const int32_t* token_to_seq,
                                                const int32_t* positions, uint16_t* output,
                                                int num_tokens, void* workspace,
                                                size_t workspace_bytes, void* stream) {
  const char* what = "vaa_paged_attention_prefill_view";
  int st = check_prefill(what, p, view, num_tokens);
  if (st) return st;
  if (num_tokens == 0) return VAA_OK;
  if (!query || !key_cache || !value_cache || !block_table || !token_to_seq || !positions ||
      !output)
    return fail(VAA_ERR_INVALID_ARG, "%s: null pointer", what);
  if (!aligned16(query) || !aligned16(key_cache) || !aligned16(value_cache) ||
      reinterpret_cast<uintptr_t>(output) % 8)
    return fail(VAA_ERR_INVALID_ARG,
                "%s: query and caches must be 16-byte aligned, the output 8-byte aligned", what);
  const bool q8 = view->cache_type == VAA_CACHE_E4M3;
  Args a{};
  a.n_splits = plan_splits(p, view, num_tokens);
  if (a.n_splits > 1) {
    const size_t rows = ws_rows(p, num_tokens, a.n_splits);
    const int dp = padded_head(p->head_size);
    const size_t need = rows * (dp + 1) * sizeof(float);
    if (!workspace || workspace_bytes < need)
      return fail(VAA_ERR_WORKSPACE, "%s: workspace %zu bytes < %zu needed", what,
                  workspace ? workspace_bytes : size_t{0}, need);
    if (!aligned16(workspace))
      return fail(VAA_ERR_INVALID_ARG, "%s: workspace must be 16-byte aligned", what);
    a.ws_acc = static_cast<float*>(workspace);
    a.ws_lse = a.ws_acc + rows * dp;
  }
  a.q = query;
  a.kc = static_cast<const char*>(key_cache);
  a.vc = static_cast<const char*>(value_cache);
  a.ke = view->key_exps;
  a.ve = view->value_exps;
  a.bt = block_table;
  a.tok_seq = token_to_seq;
  a.pos = positions;
  a.out = output;
  a.scale_log2 = p->scale * kLog2e;
  a.hd = p->head_size;
  a.num_tokens = num_tokens;
  a.num_seqs = p->num_seqs;
  a.max_blocks = p->max_blocks_per_seq;
  a.block_size = p->block_size;
  a.kvh = p->num_kv_heads;
  a.H = p->num_query_heads;
  a.G = p->queries_per_kv;
  a.window = view->window;
  a.first = view->first_tokens;
  a.bs_shift = (a.block_size & (a.block_size - 1)) == 0 ? __builtin_ctz(a.block_size) : -1;
  a.tiles_x = static_cast<int>(query_tiles(p, num_tokens));
  a.padded = (a.tiles_x * a.kvh + kXcds - 1) / kXcds * kXcds;
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
    case 32: return launch_d<32>(a, bf, q8, s);
    case 64: return launch_d<64>(a, bf, q8, s);
    case 96: return launch_d<96>(a, bf, q8, s);
    default: return launch_d<128>(a, bf, q8, s);
  }
}
