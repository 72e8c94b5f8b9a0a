// Attention of drafted tokens over the paged cache (bf16, or e4m3 with a scale a token and head).
//
// A sequence's qlen new tokens are its last keys: base = ctx - qlen committed keys stand before them.  Row (token i, head h) sees key j where
// j < base, or where bit (j - base) of the token's mask is set (no masks: j - base <= i, a chain or a single token).
//
// S^T = K Q^T and O^T += V^T P^T on mfma_f32_16x16x32_bf16, one lane column (lane & 15) a row, so that a row's maximum and sum stay in a lane
// and P leaves the scores as the second product's operand.  Lane group g (lane >> 4) holds the scores of CK / 4 NEIGHBOURING keys of a chunk
// of CK: the K rows are dealt to the tiles for that (key CK / 4 * (m / 4) + 4 t + m % 4 is row m of tile t), which costs nothing, and makes a
// lane's part of V^T one vector load (the V cache is stored transposed, 16 keys a block).
//
// Few rows (up to 32; e4m3: any number, 48 at a time): a workgroup is four waves over the same 16 RF rows (heads of one kv head, tokens x group), each
// with its own chunks.  K and V go to registers once for all rows and are never staged; the waves meet in LDS at the end.  Bound by memory: 64
// single tokens of 500 to 6000 keys, 8 kv heads of 128, 112 us (5.2 TB/s), over e4m3 65 (4.6).  More rows: tree_wide_kernel below.
//
// Weights enter the second product as bf16, half a step (2^-8) each: the product's operands have one type, and f32 ones run at a sixteenth of the rate.
// Steps of many keys fall either way, so the output is off by 0.0022 to 0.0024 of its norm where rounding the exact result to bf16 alone makes 0.0017.
// Scores, maxima, the sum of weights and the output's sums stay in 32 bits, pieces between launches too.
//
// e4m3 caches: codes become bf16 exactly (three bits behind the leading one), the key's scale multiplies its score and the value's its weight,
// ahead of the weight's rounding to bf16; the sum of weights is of the unrounded ones.
//
// Split: all (sequence, kv head, row block, range of `ulen` keys; whole contexts where they are short) form one list, cut into equal parts for the workgroups that fit the chip at
// once; a row block counts for some units more than its keys, for the way in and out of it (queries, masks, sums).  Every workgroup finds its
// part from the lengths on the device, so ragged batches whose contexts are cut are even, nothing is planned on the host and a captured graph takes new lengths.  A
// part's first and last piece may be of a row block that others hold too: their sums go to the workspace in 32 bits and a second launch joins
// them, in order (no atomics: the same bits every time).
#include "common.h"

namespace {
constexpr int BS = 16, NW = 4;
constexpr float LOG2E = 1.4426950408889634f, SLACK = 8.f;

struct TreeArgs {
  const u16* q;             // [T, nq, d], token and head strides
  long q_ts, q_hs;
  const void *kc, *vc;      // [blocks, nkv, 16, d], [blocks, nkv, d, 16]
  const float *ks, *vs;     // [blocks, nkv, 16]; e4m3 only
  const int* bt;            // [S, max_blocks]
  const int *qstart, *qlen, *ctx;
  const int* mask;          // [T, W] or null
  u16* out;                 // [T, nq, d]
  float *part_o, *part_ml;  // [2 nwg, R, d], [2 nwg, R, 2]
  int* joins;               // [nwg, 8]: what the join has to do for a part that begins a block others end; [nwg]: the number of parts
  int W, S, T, nq, nkv, G, max_blocks, num_blocks, nwg, ulen, way, least;
  float scale_log2;
};

// ---- the list of units (32-bit: the launcher makes units long enough; lengths that contradict each other end at MOST and reach no memory but their own)
constexpr int MOST = 1 << 30;
// Two counts of up to MOST (their sum does not fit 31 bits).
static constexpr int add_units(int x, int y) { return (uint32_t)x + (uint32_t)y < (uint32_t)MOST ? x + y : MOST; }
static_assert(add_units(MOST, MOST) == MOST && add_units(MOST - 1, 1) == MOST && add_units(5, 7) == 12, "counts end at MOST");
struct Shape {
  int qlen, ctx, nb, nt;    // row blocks, and units of each: a.way for its way in and out, and its key ranges
};

static __device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Where a unit of the list lies: a wave's scan over the sequences, each lane `count` neighbouring ones.  What the whole wave goes by is in
// scalar registers.
struct List {
  int incl, first, count, total;
  int qlen, ctx, qstart;    // of the lane's one sequence, where it has no more (up to 64 sequences: nothing is read twice)
};
static __device__ __forceinline__ Shape shape_of(const TreeArgs& a, int qlen, int ctx, int R) {
  Shape h;
  h.qlen = min(max(qlen, 0), a.T);
  h.ctx = min(max(ctx, 0), a.max_blocks * BS);
  h.nb = (h.qlen * a.G + R - 1) / R;                          // (T nq fits 32 bits)
  h.nt = a.ulen ? a.way + max(1, (h.ctx + a.ulen - 1) / a.ulen) : 1;
  return h;
}
static __device__ __forceinline__ int units_of(const TreeArgs& a, const Shape& h) { return (int)min((long)a.nkv * h.nb * h.nt, (long)MOST); }
static __device__ __forceinline__ Shape shape_of(const TreeArgs& a, const List& q, int s, int R) {
  if (q.count == 1) return shape_of(a, __builtin_amdgcn_readlane(q.qlen, s), __builtin_amdgcn_readlane(q.ctx, s), R);
  return shape_of(a, a.qlen[s], a.ctx[s], R);
}
static __device__ __forceinline__ int qstart_of(const TreeArgs& a, const List& q, int s) {
  return q.count == 1 ? __builtin_amdgcn_readlane(q.qstart, s) : a.qstart[s];
}
static __device__ __forceinline__ List scan_units(const TreeArgs& a, int R) {
  const int lane = threadIdx.x & 63;
  List q;
  q.count = (a.S + 63) / 64;
  q.first = lane * q.count;
  q.incl = 0;
  for (int i = 0; i < q.count; ++i) {
    const int s = min(q.first + i, a.S - 1);
    q.qlen = a.qlen[s];
    q.ctx = a.ctx[s];
    q.qstart = a.qstart[s];
    const Shape h = shape_of(a, q.qlen, q.ctx, R);
    if (q.first + i < a.S) q.incl = add_units(q.incl, units_of(a, h));
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    if (o < a.S) {                                            // (lanes from S on are not looked at)
      const int y = __shfl_up(q.incl, o, 64);
      if (lane >= o) q.incl = add_units(q.incl, y);
    }
  }
  q.total = __builtin_amdgcn_readlane(q.incl, min(a.S, 64) - 1);
  return q;
}
// The sequence of `unit` (below the total), and its units' start.
static __device__ __forceinline__ int place_of(const TreeArgs& a, int R, const List& q, int unit, int& start) {
  const int who = __builtin_ctzll(__ballot(q.incl > unit));
  int s = uniform(who * q.count);
  start = who ? __builtin_amdgcn_readlane(q.incl, who - 1) : 0;
  if (q.count == 1) return s;
  for (; s < a.S - 1; ++s) {
    const Shape h = shape_of(a, a.qlen[s], a.ctx[s], R);
    const int n = uniform(units_of(a, h));
    if (start + n > unit) break;
    start += n;
  }
  return s;
}
static __device__ __forceinline__ int part_len(const TreeArgs& a, int total) { return max(uniform((total + a.nwg - 1) / a.nwg), a.least); }

// ---- operands
static __device__ __forceinline__ uint4 flip(uint4 v, uint32_t sign) { return make_uint4(v.x ^ sign, v.y ^ sign, v.z ^ sign, v.w ^ sign); }
static __device__ __forceinline__ bf16x8 cvt8(uint2 r) {
  typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
  union { bf2 p[4]; bf16x8 v; } u;
  u.p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(r.x, 1.f, false);
  u.p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(r.x, 1.f, true);
  u.p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(r.y, 1.f, false);
  u.p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(r.y, 1.f, true);
  return u.v;
}

template <int D, int RF, bool EIGHT> struct Form {
  static constexpr int CK = EIGHT && RF == 1 ? 64 : 32;       // keys of a wave's chunk
  static constexpr int KS = D / 32, NT = D / 16, TL = CK / 16, KPG = CK / 4, R = 16 * RF;
  static constexpr bool QL = RF == 3 || (RF == 2 && D == 128 && !EIGHT);      // Q fragments in LDS: their registers would spill
  static constexpr int PITCH = D + 4;
};

template <int D, int RF, bool EIGHT> struct TreeSmem {
  using F = Form<D, RF, EIGHT>;
  union {                                                     // the queries' place is the outputs' in the end
    alignas(16) float o[NW][16][F::PITCH];
    alignas(16) u16 q[F::QL ? RF * F::KS * 64 * 8 : 8];
  };
  float m[NW][16], l[NW][16];
  alignas(16) float sc[EIGHT ? NW : 1][2][64];                // scales of a wave's chunk
  int odd;                                                    // infinities or NaN among V were left out
};

// Keys kb .. kb + 31 that a token sees, as bits.
static __device__ __forceinline__ uint32_t window(const TreeArgs& a, int kb, int base, int ctx, int tok, long row) {
  const int rem = ctx - kb, n0 = kb - base;
  const uint32_t lim = rem <= 0 ? 0u : rem >= 32 ? ~0u : (1u << rem) - 1u;
  if (a.mask == nullptr) {
    const int c = tok + 1 - n0;
    return lim & (c <= 0 ? 0u : c >= 32 ? ~0u : (1u << c) - 1u);
  }
  if (n0 <= -32) return lim;
  const int* w = a.mask + row * a.W;
  const int i = n0 < 0 ? 0 : n0 >> 5, sh = n0 & 31;
  const uint32_t lo = i < a.W ? (uint32_t)w[i] : 0u;
  if (n0 < 0) return lim & (((1u << -n0) - 1u) | (lo << -n0));
  const uint32_t hi = sh && i + 1 < a.W ? (uint32_t)w[i + 1] << (32 - sh) : 0u;
  return lim & ((lo >> sh) | hi);
}

// The top bit of every value of a word that is an infinity or NaN; and the word with those as zeros.
template <bool EIGHT> static __device__ __forceinline__ uint32_t odd_bits(uint32_t w) {
  return EIGHT ? ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u : ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
}
template <bool EIGHT> static __device__ __forceinline__ uint32_t tame(uint32_t w) {
  return w & ~(EIGHT ? (odd_bits<true>(w) >> 7) * 0xffu : (odd_bits<false>(w) >> 15) * 0xffffu);
}

// Which of a lane group's keys (CK / 4 of a chunk at kb) row `r` of a kv head's sees, as bits.
template <int CK>
static __device__ __forceinline__ uint32_t row_window(const TreeArgs& a, int kb, int base, int ctx, int r, int qlen, int qstart, int g) {
  int G = a.G;
  asm volatile("" : "+s"(G));                                 // (kept here: as loop invariants these were ten registers a row block)
  const int t = r / G;
  const long at = (long)qstart + t;
  if (t >= qlen || at < 0 || at >= a.T) return 0u;
  return window(a, kb + (CK == 64 ? 32 * (g >> 1) : 0), base, ctx, t, at) >> (CK == 64 ? 16 * (g & 1) : 8 * g);
}

// Scores times their keys' scales (e4m3), and what a row does not see at -inf.
template <int RF, int TL, bool EIGHT> static __device__ __forceinline__ void scale_scores(f32x4 (&p)[RF][TL], const float* ks) {
  if constexpr (EIGHT) {
#pragma unroll
    for (int t = 0; t < TL; ++t) {
      const f32x4 k4 = *reinterpret_cast<const f32x4*>(ks + 4 * t);
#pragma unroll
      for (int f = 0; f < RF; ++f) p[f][t] *= k4;
    }
  }
}
template <int TL> static __device__ __forceinline__ void hide(f32x4 (&p)[TL], uint32_t mine) {
#pragma unroll
  for (int t = 0; t < TL; ++t)
#pragma unroll
    for (int q = 0; q < 4; ++q) p[t][q] = (mine >> (4 * t + q)) & 1u ? p[t][q] : -INFINITY;
}

// Scores of a lane's rows to weights, with the running maximum m (of the exponent, c times the score) and sum l of each.  vs: the values' scales
// (e4m3).
template <int RF, int NT, int TL, bool EIGHT>
static __device__ __forceinline__ void weights(f32x4 (&p)[RF][TL], const float* vs, float c, float (&m)[RF], float (&l)[RF], f32x4 (&acc)[RF][NT],
                                               bf16x8 (&pf)[RF][TL / 2]) {
  float top[RF];
  bool up = false;
#pragma unroll
  for (int f = 0; f < RF; ++f) {
    top[f] = -INFINITY;
#pragma unroll
    for (int t = 0; t < TL; ++t)
#pragma unroll
      for (int q = 0; q < 4; ++q) top[f] = fmaxf(top[f], p[f][t][q]);
    up |= top[f] * c > m[f] + SLACK;
  }
  // The sums' unit follows the maximum only where a score is 2^SLACK above it: weights of up to 2^SLACK lose nothing, and the exchange between
  // lane groups and the pass over the sums are left out nearly always.
  if (__any(up)) {
#pragma unroll
    for (int f = 0; f < RF; ++f) {
      const float m_new = fmaxf(m[f], lane_max(lane_max(top[f], 16), 32) * c), al = __builtin_amdgcn_exp2f(m[f] - (m_new == -INFINITY ? 0.f : m_new));
      m[f] = m_new;
      l[f] *= al;
#pragma unroll
      for (int n = 0; n < NT; ++n) acc[f][n] *= al;
    }
  }
#pragma unroll
  for (int f = 0; f < RF; ++f) {
    const float ms = m[f] == -INFINITY ? 0.f : m[f];
#pragma unroll
    for (int t = 0; t < TL; ++t)
#pragma unroll
      for (int q = 0; q < 4; ++q) { p[f][t][q] = __builtin_amdgcn_exp2f(fmaf(p[f][t][q], c, -ms)); l[f] += p[f][t][q]; }
  }
  if constexpr (EIGHT) {
#pragma unroll
    for (int t = 0; t < TL; ++t) {
      const f32x4 v4 = *reinterpret_cast<const f32x4*>(vs + 4 * t);
#pragma unroll
      for (int f = 0; f < RF; ++f) p[f][t] *= v4;
    }
  }
#pragma unroll
  for (int f = 0; f < RF; ++f)
#pragma unroll
    for (int e = 0; e < TL / 2; ++e)
      pf[f][e] = __builtin_bit_cast(bf16x8, make_uint4(f2bf2(p[f][2 * e][0], p[f][2 * e][1]), f2bf2(p[f][2 * e][2], p[f][2 * e][3]),
                                                       f2bf2(p[f][2 * e + 1][0], p[f][2 * e + 1][1]), f2bf2(p[f][2 * e + 1][2], p[f][2 * e + 1][3])));
}

// (rare) infinities and NaN of V among keys k0 .. k1 (k0 a multiple of 16) at N neighbouring dims from `col`, to a row that sees them.  Only those of
// chunks with drafted keys were left out, so a caller begins there; 16 bytes of a dim are looked at at once (key by key from a context's first one on, a
// NaN of one sequence of 30000 keys made a call's 53 us 1650).
template <int N, bool EIGHT, class O>
static __device__ __forceinline__ void add_odd(const TreeArgs& a, const int* bt, int kvh, int D, int k0, int k1, int base, int ctx, int t, long row, int col, O&& o) {
  constexpr int RUN = EIGHT ? 16 : 8;
  for (int j = k0; j < k1; j += RUN) {
    const int page = bt[j >> 4];
    uint32_t see = window(a, j, base, ctx, t, row) & ((1u << RUN) - 1u);
    if ((unsigned)page >= (unsigned)a.num_blocks || !see) continue;
    const long at = ((long)page * a.nkv + kvh) * BS, x = at * D + col * BS + (j & 15);
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint4 v = ld16((const uint8_t*)a.vc + (x + i * BS) * (EIGHT ? 1 : 2));
      any |= odd_bits<EIGHT>(v.x) | odd_bits<EIGHT>(v.y) | odd_bits<EIGHT>(v.z) | odd_bits<EIGHT>(v.w);
    }
    if constexpr (EIGHT) {
#pragma unroll
      for (int i = 0; i < RUN; ++i) any |= !(fabsf(a.vs[at + i]) < INFINITY);
    }
    if (!any) continue;
    for (; see; see &= see - 1) {
      const int k = __builtin_ctz(see);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float v;
        if constexpr (EIGHT) v = __builtin_amdgcn_cvt_f32_fp8(((const uint8_t*)a.vc)[x + i * BS + k], 0) * a.vs[at + k];
        else v = bf2f(((const u16*)a.vc)[x + i * BS + k]);
        if (!(fabsf(v) < INFINITY)) o[i] += v;
      }
    }
  }
}

// Where a piece goes: the output, or slot `slot` of the workspace (< 0: the output).
template <int D, int RF, bool EIGHT>
static __device__ __forceinline__ void piece(const TreeArgs& a, TreeSmem<D, RF, EIGHT>& sm, const int seq, const int qstart, const Shape h, const int kvh, const int blk,
                                             const int k0, const int k1, const int turn, const int slot) {
  using F = Form<D, RF, EIGHT>;
  constexpr int CK = F::CK, KS = F::KS, NT = F::NT, TL = F::TL, KPG = F::KPG;
  constexpr int KW = EIGHT ? 2 : 4, VW = EIGHT && CK == 32 ? 2 : 4;     // words of a lane's K step and V row
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, rl = lane & 15;
  const int base = h.ctx - h.qlen;
  const int* bt = a.bt + (long)seq * a.max_blocks;

  const int row0 = blk * F::R;
  auto token = [&](int f) { return (row0 + 16 * f + rl) / a.G; };
  auto real = [&](int t) { const long at = (long)qstart + t; return t < h.qlen && at >= 0 && at < a.T; };
  // Q fragments: dims 32 s + 8 g (bf16), or as the code loads deal them (pairs of steps share a 16-byte load)
  auto dim0 = [&](int s) { return EIGHT && (s | 1) < KS ? 64 * (s >> 1) + 16 * g + 8 * (s & 1) : 32 * s + 8 * g; };
  const uint32_t sign = a.scale_log2 < 0.f ? 0x80008000u : 0u;      // c below is positive
  auto q_at = [&](int f, int s) {
    const int t = token(f), head = kvh * a.G + (row0 + 16 * f + rl) % a.G;
    return real(t) ? flip(ld16(a.q + (qstart + (long)t) * a.q_ts + head * a.q_hs + dim0(s)), sign) : make_uint4(0u, 0u, 0u, 0u);
  };
  f32x4 acc[RF][NT];
  float m[RF], l[RF];
#pragma unroll
  for (int f = 0; f < RF; ++f) {
    m[f] = -INFINITY;
    l[f] = 0.f;
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[f][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // what a score is multiplied by on its way to the exponent (a scale of 0: a number that leaves -inf what it is)
  const float c = fmaxf(fabsf(a.scale_log2), 0x1p-120f);

  // A lane's pages: of its K rows and of its lane group's keys.  One outside the pool hides its keys.
  const int last_block = (h.ctx - 1) >> 4, bk = CK == 64 ? rl >> 2 : rl >> 3, bv = CK == 64 ? g : g >> 1;
  uint32_t kr[TL][KS][KW], vr[NT][VW];
  float ks_l = 0.f, vs_l = 0.f;                               // e4m3: scales of key KPG g + rl of the chunk (rl < KPG)
  int pk, pv, pk_n, pv_n;
  auto pages = [&](int kb, int& to_k, int& to_v) {
    to_k = bt[min((kb >> 4) + bk, last_block)];
    to_v = bt[min((kb >> 4) + bv, last_block)];
  };
  auto in_pool = [&](int p) { return (unsigned)p < (unsigned)a.num_blocks; };
  auto load_k = [&](int p) {
    const long hk = ((long)(in_pool(p) ? p : 0) * a.nkv + kvh) * BS;
#pragma unroll
    for (int t = 0; t < TL; ++t) {
      const long row = hk + (CK == 64 ? 0 : 8 * ((rl >> 2) & 1)) + 4 * t + (rl & 3);
      if constexpr (EIGHT) {
        const uint8_t* x = (const uint8_t*)a.kc + row * D;
#pragma unroll
        for (int s = 0; s < KS; s += 2) {
          if (s + 1 < KS) {
            const uint4 v = ld16(x + 32 * s + 16 * g);
            kr[t][s][0] = v.x; kr[t][s][1] = v.y; kr[t][s + 1][0] = v.z; kr[t][s + 1][1] = v.w;
          } else {
            const uint2 v = *reinterpret_cast<const uint2*>(x + 32 * s + 8 * g);
            kr[t][s][0] = v.x; kr[t][s][1] = v.y;
          }
        }
      } else {
        const u16* x = (const u16*)a.kc + row * D + 8 * g;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          const uint4 v = ld16(x + 32 * s);
          kr[t][s][0] = v.x; kr[t][s][1] = v.y; kr[t][s][KW - 2] = v.z; kr[t][s][KW - 1] = v.w;
        }
      }
    }
  };
  auto load_v = [&](int kb, int p) {
    const bool there = in_pool(p);
    const long hv = ((long)(there ? p : 0) * a.nkv + kvh) * BS;
    if constexpr (EIGHT) {
      ks_l = vs_l = 0.f;
      if (there && rl < KPG && kb + KPG * g + rl < h.ctx) {
        const long at = hv + (CK == 64 ? rl : 8 * (g & 1) + rl);
        ks_l = a.ks[at];
        vs_l = a.vs[at];
      }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const uint8_t* x = (const uint8_t*)a.vc + (hv * D + (16 * n + rl) * BS) * (EIGHT ? 1 : 2) + (EIGHT ? (CK == 64 ? 0 : 8) : 16) * (g & 1);
      if constexpr (VW == 4) {
        const uint4 v = ld16(x);
        vr[n][0] = v.x; vr[n][1] = v.y; vr[n][VW - 2] = v.z; vr[n][VW - 1] = v.w;
      } else {
        const uint2 v = *reinterpret_cast<const uint2*>(x);
        vr[n][0] = v.x; vr[n][1] = v.y;
      }
    }
  };
  auto k_frag = [&](int t, int s) {
    if constexpr (EIGHT) return cvt8(make_uint2(kr[t][s][0], kr[t][s][1]));
    else return __builtin_bit_cast(bf16x8, make_uint4(kr[t][s][0], kr[t][s][1], kr[t][s][KW - 2], kr[t][s][KW - 1]));
  };
  bf16x8 qr[F::QL ? 1 : RF][KS];
  auto q_frag = [&](int f, int s) {
    if constexpr (F::QL) return __builtin_bit_cast(bf16x8, ld16(&sm.q[((f * KS + s) * 64 + lane) * 8]));
    else return qr[f][s];
  };

  // K of the next chunk is asked for as soon as the scores have used this one's registers, V as soon as the second product has, pages a chunk
  // ahead of both: two chunks' latencies overlap without registers for two chunks.
  constexpr int ROUND = CK * NW;
  const int k_wave = k0 + CK * wave;
  int left = (k1 - k_wave + ROUND - 1) / ROUND, kb = k_wave + turn < k1 ? k_wave + turn : k_wave;
  auto after = [&](int x) { return x + ROUND < k1 ? x + ROUND : k_wave; };
  if (left > 0) pages(kb, pk, pv);
  if constexpr (F::QL) {
#pragma unroll
    for (int f = 0; f < RF; ++f)
      if (f % NW == wave) {
#pragma unroll
        for (int s = 0; s < KS; ++s) qr[0][s] = __builtin_bit_cast(bf16x8, q_at(f, s));
      }
  } else {
#pragma unroll
    for (int f = 0; f < RF; ++f)
#pragma unroll
      for (int s = 0; s < KS; ++s) qr[f][s] = __builtin_bit_cast(bf16x8, q_at(f, s));
  }
  if (left > 0) {
    load_k(pk);
    load_v(kb, pv);
    pages(after(kb), pk_n, pv_n);
  }
  __syncthreads();                                            // the piece before is done with LDS
  if (threadIdx.x == 0) sm.odd = 0;
  if constexpr (F::QL) {
#pragma unroll
    for (int f = 0; f < RF; ++f)
      if (f % NW == wave) {
#pragma unroll
        for (int s = 0; s < KS; ++s) st16(&sm.q[((f * KS + s) * 64 + lane) * 8], __builtin_bit_cast(uint4, qr[0][s]));
      }
  }
  __syncthreads();
  for (int next; left > 0; kb = next) {
    next = after(kb);
    --left;
    const bool paged = in_pool(pv);
    const bool drafted = kb + CK > base;                      // some of its keys are, or there are none
    const bool plain = !drafted && !__any(!paged);            // every row sees the whole chunk
    bool odd = false;
    if constexpr (EIGHT) {
      odd = drafted && !(fabsf(vs_l) < INFINITY);
      if (odd) vs_l = 0.f;                                    // (what is seen is added at the end)
      if (rl < KPG) {
        sm.sc[wave][0][KPG * g + rl] = ks_l;
        sm.sc[wave][1][KPG * g + rl] = vs_l;
      }
      __builtin_amdgcn_wave_barrier();
    }
    const float *ks = &sm.sc[EIGHT ? wave : 0][0][KPG * g], *vs = &sm.sc[EIGHT ? wave : 0][1][KPG * g];
    f32x4 sc[RF][TL];
#pragma unroll
    for (int f = 0; f < RF; ++f)
#pragma unroll
      for (int t = 0; t < TL; ++t) sc[f][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      bf16x8 kf[TL];
#pragma unroll
      for (int t = 0; t < TL; ++t) kf[t] = k_frag(t, s);
#pragma unroll
      for (int f = 0; f < RF; ++f) {
        const bf16x8 qf = q_frag(f, s);
#pragma unroll
        for (int t = 0; t < TL; ++t) sc[f][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[t], qf, sc[f][t], 0, 0, 0);
      }
    }
    if (left > 0) load_k(pk_n);
    bf16x8 pf[RF][TL / 2];
    scale_scores<RF, TL, EIGHT>(sc, ks);
    if (!plain) {
#pragma unroll
      for (int f = 0; f < RF; ++f) hide(sc[f], paged ? row_window<CK>(a, kb, base, h.ctx, row0 + 16 * f + rl, h.qlen, qstart, g) : 0u);
      // what no row may see (keys past ctx, pages outside the pool: stale memory) is zero in V; an infinity or NaN of a drafted token that a
      // row does not see would reach it as 0 * inf, so those are zero too and added at the end, to the rows that see them (committed keys: all rows)
      const int n = paged ? h.ctx - kb - KPG * g : 0;         // keys of this lane that exist
      uint32_t real_w[VW], any = 0;
#pragma unroll
      for (int w = 0; w < VW; ++w) {
        const int per = EIGHT ? 4 : 2, left = min(max(n - per * w, 0), per);
        real_w[w] = left == per ? ~0u : (1u << ((EIGHT ? 8 : 16) * left)) - 1u;
      }
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int w = 0; w < VW; ++w) any |= odd_bits<EIGHT>(vr[i][w] &= real_w[w]);
      if (drafted && __any(any != 0 || odd)) {
        sm.odd = 1;
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int w = 0; w < VW; ++w) vr[i][w] = tame<EIGHT>(vr[i][w]);
      }
    }
    weights<RF, NT, TL, EIGHT>(sc, vs, c, m, l, acc, pf);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < CK / 32; ++e) {
        bf16x8 vf;
        if constexpr (EIGHT) vf = cvt8(make_uint2(vr[n][(2 * e) % VW], vr[n][(2 * e + 1) % VW]));
        else vf = __builtin_bit_cast(bf16x8, make_uint4(vr[n][0], vr[n][1], vr[n][VW - 2], vr[n][VW - 1]));
#pragma unroll
        for (int f = 0; f < RF; ++f) acc[f][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[f][e], acc[f][n], 0, 0, 0);
      }
    if constexpr (EIGHT) __builtin_amdgcn_wave_barrier();     // scales are read before the next chunk's are written
    if (left > 0) {
      load_v(next, pv_n);
      pv = pv_n;
      pages(after(next), pk_n, pv_n);
    }
  }

  // ---- the waves meet, sixteen rows at a time.  acc[f][n][r] = O^T[dim 16 n + 4 g + r][row 16 f + rl]
#pragma unroll
  for (int f = 0; f < RF; ++f) {
    const float lw = lane_add(lane_add(l[f], 16), 32);
    __syncthreads();
    if (g == 0) { sm.m[wave][rl] = m[f]; sm.l[wave][rl] = lw; }
#pragma unroll
    for (int n = 0; n < NT; ++n) *reinterpret_cast<f32x4*>(&sm.o[wave][rl][16 * n + 4 * g]) = acc[f][n];
    __syncthreads();
    for (int e = 8 * threadIdx.x; e < 16 * D; e += 8 * 64 * NW) {
      const int row = e / D, col = e % D;
      float M = -INFINITY, L = 0.f, o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < NW; ++i) M = fmaxf(M, sm.m[i][row]);
      const float Ms = M == -INFINITY ? 0.f : M;
#pragma unroll
      for (int i = 0; i < NW; ++i) {
        const float c = __builtin_amdgcn_exp2f(sm.m[i][row] - Ms);
        L += sm.l[i][row] * c;
        const f32x4 x = *reinterpret_cast<const f32x4*>(&sm.o[i][row][col]), y = *reinterpret_cast<const f32x4*>(&sm.o[i][row][col + 4]);
#pragma unroll
        for (int j = 0; j < 4; ++j) { o[j] += x[j] * c; o[4 + j] += y[j] * c; }
      }
      const int of_block = f * 16 + row, r = row0 + of_block, t = r / a.G;
      if (!real(t)) continue;
      if (sm.odd) add_odd<8, EIGHT>(a, bt, kvh, D, max(k0, base & -CK), k1, base, h.ctx, t, (long)qstart + t, col, o);
      if (slot >= 0) {
        const long at = (long)slot * F::R + of_block;
        *reinterpret_cast<f32x4*>(a.part_o + at * D + col) = f32x4{o[0], o[1], o[2], o[3]};
        *reinterpret_cast<f32x4*>(a.part_o + at * D + col + 4) = f32x4{o[4], o[5], o[6], o[7]};
        if (col == 0) { a.part_ml[2 * at] = M; a.part_ml[2 * at + 1] = L; }
        continue;
      }
      const float inv = L == 0.f ? 0.f : 1.f / L;             // a row that sees nothing is zero
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] *= inv;
      st16(a.out + ((qstart + (long)t) * a.nq + kvh * a.G + r % a.G) * D + col, pack8(o));
    }
  }
}

// A workgroup's part of the list: run(sequence, its first row, its shape, kv head, row block, first key, last key, turn, slot) for every piece of it.
// A piece begins `turn` keys behind its first one and comes to those in the end: parts of the row blocks of a kv head, which read the same keys and are cut at
// different ones, are so at the same keys (modulo a part) at the same time, and find them in L2 (512 rows of 8000 to 32000 keys: 8.3 M misses, 4.4 M so;
// 5 us of 195).
template <class F> static __device__ __forceinline__ void walk(const TreeArgs& a, int R, F&& run) {
  const List q = scan_units(a, R);
  const bool lead = threadIdx.x == 0 && a.joins;
  if (q.total == 0) {
    if (lead && blockIdx.x == 0) a.joins[8 * a.nwg] = 0;
    return;
  }
  const int part = part_len(a, q.total);
  // parts in the order of the list to workgroups of one XCD, whose L2 the row blocks of a kv head then share
  const int parts = uniform((q.total + part - 1) / part), q8 = parts / 8, r8 = parts % 8, x = blockIdx.x % 8, i = blockIdx.x / 8;
  if (i >= q8 + (x < r8)) return;
  const int me = x * q8 + min(x, r8) + i, end = min(q.total, (me + 1) * part);
  if (lead && me == 0) a.joins[8 * a.nwg] = parts;
  if (lead) a.joins[8 * me] = -1;
  int u = me * part, start, slot = 2 * me;
  int seq = place_of(a, R, q, u, start), qstart = qstart_of(a, q, seq);
  Shape h = shape_of(a, q, seq, R);                           // (later ones from memory: the lanes' lengths are not kept for them)
  while (u < end) {
    const int n = uniform(units_of(a, h));
    if (u - start >= n) {
      if (++seq >= a.S) return;
      start += n;
      h = shape_of(a, a.qlen[seq], a.ctx[seq], R);
      qstart = a.qstart[seq];
      continue;
    }
    const int nt = uniform(h.nt), nb = uniform(h.nb), row = uniform((u - start) / nt), at = u - start - row * nt, take = min(nt - at, end - u);
    const int kvh = uniform(row / nb), blk = row - kvh * nb, r0 = max(at - a.way, 0), r1 = at + take - a.way, ranges = nt - a.way;
    if (r1 > r0) {
      const bool whole = r0 == 0 && r1 == ranges;
      if (lead && r0 == 0 && !whole) {
        int* to = a.joins + 8 * me;
        to[0] = slot;
        to[1] = min((u - at + nt - 1) / part, a.nwg - 1);
        to[2] = blk * R;
        to[3] = kvh;
        to[4] = qstart;
        to[5] = h.qlen;
      }
      const int past = r0 % part, turn = past && part - past < r1 - r0 ? part - past : 0;
      run(seq, qstart, h, kvh, blk, r0 * a.ulen, r1 == ranges ? h.ctx : r1 * a.ulen, turn * a.ulen, whole ? -1 : slot);
      slot = 2 * me + 1;
    }
    u += take;
  }
}

template <int D, int RF, bool EIGHT>
__global__ void __launch_bounds__(64 * NW, (RF > 1 || D > 64 ? 2 : 3)) tree_attn_kernel(TreeArgs a) {
  __shared__ TreeSmem<D, RF, EIGHT> sm;
  walk(a, Form<D, RF, EIGHT>::R, [&](int seq, int qstart, const Shape& h, int kvh, int blk, int k0, int k1, int turn, int slot) __attribute__((always_inline)) {
    piece<D, RF, EIGHT>(a, sm, seq, qstart, h, kvh, blk, k0, k1, turn, slot);
  });
}

// ---- many rows: the waves have rows of their own and share the keys.
// Four waves of 16 RF rows read every chunk from LDS, in two stages: a wave asks for its share of the next chunk, computes on this one and then writes
// what has arrived.  One operand fragment is a kilobyte in lane order, read back as it lies, without conflicts.  K and V leave L2 once for 64 RF
// rows: with rows of one wave only, every 48 read them again, and ragged trees of 80 to 160 rows (8 kv heads of 128, 32 sequences of 200 to 3000 keys)
// ran at what L2 misses of four such readings allow (115 us, 65 so).  512 rows of 8000 to 32000 keys: 178 us, 630 TFLOP/s; vector instructions take 42 %
// of the time and products 38, and two waves a SIMD hardly overlap them.  (Loads straight to LDS made the compiler wait for all of them ahead of
// any LDS read; 48 rows a wave spill; 64 keys a stage, loads two chunks ahead and a higher priority within products gain nothing.)
template <int D, int RF> struct Wide {
  static constexpr int CK = D > 64 ? 32 : 64, KS = D / 32, NT = D / 16, TL = CK / 16, KPG = CK / 4, R = 16 * RF * NW;
  // one-kilobyte slots of a stage: K a tile and 32 dims (slot t * KS + s), V eight keys a lane group and sixteen dims (KSL + e * NT + n)
  static constexpr int KSL = TL * KS, SL = KSL + NT * (CK / 32), GI = SL / NW, PAGES = 1024;
  // waves 0 and 1 stage K, 2 and 3 V, whole rows of tiles each
  static_assert(SL == NW * GI && KSL == 2 * GI && GI % KS == 0 && NT % GI == 0, "a wave's slots");
};
template <int D, int RF> struct WideSmem {
  using F = Wide<D, RF>;
  alignas(16) unsigned char ring[2][F::SL * 1024];
  int page[F::PAGES];                                         // from block `first` of the sequence on; -1: outside the pool
  int odd;                                                    // infinities or NaN among V were left out
  int holes;                                                  // a page outside the pool was met
};

template <int D, int RF>
static __device__ __forceinline__ void wide_piece(const TreeArgs& a, WideSmem<D, RF>& sm, const int seq, const int qstart, const Shape h, const int kvh, const int blk,
                                                  const int k0, const int k1, const int turn, const int slot) {
  using F = Wide<D, RF>;
  constexpr int CK = F::CK, KS = F::KS, NT = F::NT, KPG = F::KPG;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, rl = lane & 15;
  const int base = h.ctx - h.qlen, row0 = (blk * NW + wave) * 16 * RF;
  const int* bt = a.bt + (long)seq * a.max_blocks;
  const bool idle = row0 >= h.qlen * a.G;                     // no row: this wave stages only
  const int steps = (k1 - k0 + CK - 1) / CK, last_block = (h.ctx - 1) >> 4;
  auto real = [&](int t) { const long at = (long)qstart + t; return t < h.qlen && at >= 0 && at < a.T; };

  const uint32_t sign = a.scale_log2 < 0.f ? 0x80008000u : 0u;      // c below is positive
  bf16x8 qf[RF][KS];
#pragma unroll
  for (int f = 0; f < RF; ++f) {
    const int r = row0 + 16 * f + rl, t = r / a.G, head = kvh * a.G + r % a.G;
#pragma unroll
    for (int s = 0; s < KS; ++s)
      qf[f][s] = __builtin_bit_cast(bf16x8, real(t) ? flip(ld16(a.q + (qstart + (long)t) * a.q_ts + head * a.q_hs + 32 * s + 8 * g), sign) : make_uint4(0u, 0u, 0u, 0u));
  }
  int first = k0 >> 4, holes;
  auto fill = [&](int from) {
    first = from;
    for (int i = threadIdx.x; i < F::PAGES; i += 64 * NW) {
      const int b = from + i, p = b <= last_block ? bt[b] : -1;
      const bool in = (unsigned)p < (unsigned)a.num_blocks;
      sm.page[i] = in ? p : -1;
      if (b <= last_block && !in) sm.holes = 1;
    }
    __syncthreads();
    holes = uniform(sm.holes);
  };
  __syncthreads();                                            // the piece before is done with LDS
  if (threadIdx.x == 0) sm.odd = 0;
  fill(first);

  f32x4 acc[RF][NT];
  float m[RF], l[RF];
#pragma unroll
  for (int f = 0; f < RF; ++f) {
    m[f] = -INFINITY;
    l[f] = 0.f;
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[f][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  uint4 next[F::GI];                                          // this wave's share of a chunk
  const int rot = steps * CK <= BS * F::PAGES ? turn / CK : 0;
  auto key_of = [&](int i) { return k0 + CK * (i + rot < steps ? i + rot : i + rot - steps); };
  const bool of_k = wave < NW / 2;
  const int own = (wave % (NW / 2)) * F::GI;                  // the first of its slots, of K's or of V's
  const int from = of_k ? ((CK == 64 ? 0 : 8 * ((rl >> 2) & 1)) + 4 * (own / KS) + (rl & 3)) * D + 8 * g
                        : (16 * (own % NT) + rl) * BS + (CK == 64 ? 8 * (own / NT) : 8 * (g & 1));
  const u16* lane_src = (const u16*)(of_k ? a.kc : a.vc) + (long)kvh * BS * D + from;
  const int lane_page = CK == 64 ? (of_k ? rl >> 2 : g) : (of_k ? rl >> 3 : g >> 1);
  const uint32_t page_len = (uint32_t)a.nkv * BS * D;         // (fewer than 2^20 kv heads: fits)
  int page = 0;
  auto load = [&](int i) {
    page = sm.page[(key_of(i) >> 4) - first + lane_page];
    const u16* x = lane_src + (uint64_t)(uint32_t)max(page, 0) * page_len;
#pragma unroll
    for (int j = 0; j < F::GI; ++j) next[j] = ld16(x + (of_k ? 4 * (j / KS) * D + 32 * (j % KS) : 16 * j * BS));
  };
  auto store = [&](int i) {
    unsigned char* ring = sm.ring[i & 1];
    const int kb = key_of(i);
    if (!of_k && (kb + CK > base || holes)) {
      const int n = page >= 0 ? h.ctx - kb - KPG * g : 0;     // keys of this lane's that exist
      // what no row may see (keys past ctx, pages outside the pool: stale memory) is zero in V; an infinity or NaN of a drafted token that a
      // row does not see would reach it as 0 * inf, so those are zero too and added at the end, to the rows that see them (committed keys: all rows)
      const uint32_t drafted = kb + CK > base ? ~0u : 0u;
      uint32_t odd = 0;
#pragma unroll
      for (int j = 0; j < F::GI; ++j) {
        uint32_t w[4] = {next[j].x, next[j].y, next[j].z, next[j].w};
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int left = min(max(n - 8 * (own / NT) - 2 * x, 0), 2);
          w[x] &= left == 2 ? ~0u : (1u << (16 * left)) - 1u;
          const uint32_t bits = odd_bits<false>(w[x]) & drafted;
          odd |= bits;
          w[x] &= ~((bits >> 15) * 0xffffu);
        }
        next[j] = make_uint4(w[0], w[1], w[2], w[3]);
      }
      if (__any(odd != 0)) sm.odd = 1;
    }
#pragma unroll
    for (int j = 0; j < F::GI; ++j) st16(ring + (wave * F::GI + j) * 1024 + lane * 16, next[j]);
  };
  const float c = fmaxf(fabsf(a.scale_log2), 0x1p-120f);
  if (steps > 0) { load(0); store(0); }
  for (int i = 0; i < steps; ++i) {
    const int kb = key_of(i);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();                             // stage i is whole, and the other one free
    asm volatile("" ::: "memory");
    if (i + 1 < steps) {
      if (((key_of(i + 1) + CK) >> 4) - first > F::PAGES) {   // the window of pages moves on (uniform, every 16 PAGES keys, in their order)
        fill(kb >> 4);
      }
      load(i + 1);
    }
    if (!idle) {
    const unsigned char* ring = sm.ring[i & 1];
    const bool plain = kb + CK <= base && !holes;
#pragma unroll 1
    for (int e = 0; e < CK / 32; ++e) {                       // tiles 2 e, 2 e + 1: eight neighbouring keys of a lane group's
      f32x4 sc[RF][2];
#pragma unroll
      for (int f = 0; f < RF; ++f) sc[f][0] = sc[f][1] = f32x4{0.f, 0.f, 0.f, 0.f};
      // operands of a product are all on their way before its first instruction, V's while the weights are computed: read one by one, two waves a
      // SIMD spent half their time waiting for LDS
      bf16x8 kf[2][KS], vf[NT];
#pragma unroll
      for (int t2 = 0; t2 < 2; ++t2)
#pragma unroll
        for (int s = 0; s < KS; ++s) kf[t2][s] = __builtin_bit_cast(bf16x8, ld16(ring + ((2 * e + t2) * KS + s) * 1024 + lane * 16));
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int f = 0; f < RF; ++f)
#pragma unroll
          for (int t2 = 0; t2 < 2; ++t2) sc[f][t2] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[t2][s], qf[f][s], sc[f][t2], 0, 0, 0);
#pragma unroll
      for (int n = 0; n < NT; ++n) vf[n] = __builtin_bit_cast(bf16x8, ld16(ring + (F::KSL + e * NT + n) * 1024 + lane * 16));
      __builtin_amdgcn_sched_barrier(0);
      bf16x8 pf[RF][1];
      if (!plain) {
        const bool paged = sm.page[(kb >> 4) - first + (CK == 64 ? g : g >> 1)] >= 0;
#pragma unroll
        for (int f = 0; f < RF; ++f) hide(sc[f], paged ? row_window<CK>(a, kb, base, h.ctx, row0 + 16 * f + rl, h.qlen, qstart, g) >> (8 * e) : 0u);
      }
      weights<RF, NT, 2, false>(sc, nullptr, c, m, l, acc, pf);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int f = 0; f < RF; ++f) acc[f][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[n], pf[f][0], acc[f][n], 0, 0, 0);
    }
    }
    if (i + 1 < steps) store(i + 1);
  }

  // acc[f][n][r] = O^T[dim 16 n + 4 g + r][row 16 f + rl]: four neighbouring dims of the lane's own row
  __syncthreads();
  const bool any_odd = sm.odd != 0;
#pragma unroll
  for (int f = 0; f < RF; ++f) {
    const float L = lane_add(lane_add(l[f], 16), 32);
    const int r = row0 + 16 * f + rl, t = r / a.G;
    if (!real(t)) continue;
    const float inv = L == 0.f ? 0.f : 1.f / L;               // a row that sees nothing is zero
    const long at = (long)slot * F::R + (wave * RF + f) * 16 + rl;
    u16* to = a.out + ((qstart + (long)t) * a.nq + kvh * a.G + r % a.G) * D;
    if (slot >= 0 && g == 0) { a.part_ml[2 * at] = m[f]; a.part_ml[2 * at + 1] = L; }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int col = 16 * n + 4 * g;
      f32x4 o = acc[f][n];
      if (any_odd) add_odd<4, false>(a, bt, kvh, D, max(k0, base & -CK), k1, base, h.ctx, t, (long)qstart + t, col, o);
      if (slot >= 0) *reinterpret_cast<f32x4*>(a.part_o + at * D + col) = o;
      else *reinterpret_cast<uint2*>(to + col) = make_uint2(f2bf2(o[0] * inv, o[1] * inv), f2bf2(o[2] * inv, o[3] * inv));
    }
  }
}

template <int D, int RF> __global__ void __launch_bounds__(64 * NW, 2) tree_wide_kernel(TreeArgs a) {
  __shared__ WideSmem<D, RF> sm;
  if (threadIdx.x == 0) sm.holes = 0;
  walk(a, Wide<D, RF>::R, [&](int seq, int qstart, const Shape& h, int kvh, int blk, int k0, int k1, int turn, int slot) __attribute__((always_inline)) {
    wide_piece<D, RF>(a, sm, seq, qstart, h, kvh, blk, k0, k1, turn, slot);
  });
}

// Joins the pieces of one row block that several parts hold: part blockIdx.x has its first keys (and left word of it), parts up to i1 the others as their
// first pieces.
template <int D>
__global__ void __launch_bounds__(64 * NW) tree_join_kernel(TreeArgs a, int R) {
  const int i0 = blockIdx.x;
  const int* to_do = a.joins + 8 * i0;
  const int parts = a.joins[8 * a.nwg], first = to_do[0], i1 = to_do[1], row0 = to_do[2], kvh = to_do[3], qstart = to_do[4], qlen = to_do[5];
  if (i0 >= parts || first < 0) return;                       // (asked for together: a trip to memory less)
  constexpr int LR = D / 4 <= 16 ? 16 : 32, RW = 64 * NW / LR;      // lanes of a row (four values each), rows at a time
  const int lr = threadIdx.x % LR, col = min(4 * lr, D - 4);
  for (int rr = RW * blockIdx.y + threadIdx.x / LR; rr < R; rr += RW * gridDim.y) {
    const int r = row0 + rr, t = r / a.G;
    const long to = (long)qstart + t;
    if (t >= qlen || to < 0 || to >= a.T) continue;
    auto slot_row = [&](int i) { return (long)(i == i0 ? first : 2 * i) * R + rr; };
    float M = -INFINITY, L = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int i = i0; i <= i1; i += 4) {                       // four pieces' sums and maxima in one trip
      float2 ml[4];
      f32x4 x[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const long at = slot_row(min(i + c, i1));
        ml[c] = *reinterpret_cast<const float2*>(a.part_ml + 2 * at);
        x[c] = *reinterpret_cast<const f32x4*>(a.part_o + at * D + col);
      }
      float top = M;
#pragma unroll
      for (int c = 0; c < 4; ++c) top = fmaxf(top, ml[c].x);
      const float ts = top == -INFINITY ? 0.f : top, w0 = __builtin_amdgcn_exp2f(M - ts);
      M = top;
      L *= w0;
      o *= w0;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if (i + c > i1) continue;
        const float w = __builtin_amdgcn_exp2f(ml[c].x - ts);
        L += ml[c].y * w;
        o += x[c] * w;
      }
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    if (4 * lr < D)
      *reinterpret_cast<uint2*>(a.out + (to * a.nq + kvh * a.G + r % a.G) * D + col) = make_uint2(f2bf2(o[0] * inv, o[1] * inv), f2bf2(o[2] * inv, o[3] * inv));
  }
}

template <int D> int launch_d(const TreeArgs& a, int rf, bool wide, int rows, hipStream_t st) {
  const bool e = a.ks != nullptr;
  const dim3 grid(a.nwg), block(64 * NW);
  if (wide && !e && rf == 1) hipLaunchKernelGGL((tree_wide_kernel<D, 1>), grid, block, 0, st, a);
  else if (wide && !e && rf == 2) hipLaunchKernelGGL((tree_wide_kernel<D, 2>), grid, block, 0, st, a);
  else if (wide) return -5;
  else if (rf == 1 && e) hipLaunchKernelGGL((tree_attn_kernel<D, 1, true>), grid, block, 0, st, a);
  else if (rf == 1) hipLaunchKernelGGL((tree_attn_kernel<D, 1, false>), grid, block, 0, st, a);
  else if (rf == 2 && e) hipLaunchKernelGGL((tree_attn_kernel<D, 2, true>), grid, block, 0, st, a);
  else if (rf == 2) hipLaunchKernelGGL((tree_attn_kernel<D, 2, false>), grid, block, 0, st, a);
  else if (e) hipLaunchKernelGGL((tree_attn_kernel<D, 3, true>), grid, block, 0, st, a);
  else return -5;
  if (a.ulen && a.nwg > 1) hipLaunchKernelGGL((tree_join_kernel<D>), dim3(a.nwg - 1, (rows + 15) / 16), dim3(64 * NW), 0, st, a, 16 * rf * (wide ? NW : 1));
  return (int)hipGetLastError();
}
}  // namespace

// rf: a wave has 16 rf rows (bf16 1 or 2, e4m3 up to 3).  wide (bf16): a row block is four waves' rows, else one's.  ulen: keys of a unit, whole rounds of a workgroup's
// chunks (64 keys wide, 256 of e4m3 in 16 rows, else 128), since a piece begins units behind its first key and goes on in rounds; 0: a row block is
// one unit (no workspace, one launch).  max_blocks of 0: no sequence has a key, nothing is read but the lengths and queries, and all rows are zero.  way: units that a row block counts for beside its keys; least: units of a part.  rows: those of a block that the join's grid has waves for.
extern "C" int dllm_tree_attention(const void* q, long q_ts, long q_hs, const void* kc, const void* vc, const float* ks, const float* vs,
                                   const int* bt, const int* qstart, const int* qlen, const int* ctx, const int* mask, void* out, float* part_o,
                                   float* part_ml, int* joins, int W, int S, int T, int nq, int nkv, int d, int max_blocks, int num_blocks, int nwg, int ulen, int way, int least,
                                   int rf, int wide, int rows, float scale, hipStream_t st) {
  if (nkv < 1 || nq < nkv || nq % nkv || rf < 1 || rf > 3 || rows < 1) return -1;
  if ((ks == nullptr) != (vs == nullptr) || S < 1 || T < 1 || max_blocks < 0 || num_blocks < 0 || (max_blocks && !num_blocks) || nwg < 1) return -2;
  const int round = wide ? 64 : ks && rf == 1 ? 256 : 128;
  if (ulen < 0 || ulen % round || way < 0 || least < 1 || (ulen && (!part_o || !part_ml || !joins))) return -3;
  TreeArgs a{(const u16*)q, q_ts, q_hs, kc, vc, ks, vs, bt, qstart, qlen, ctx, mask, (u16*)out, part_o, part_ml,
             ulen ? joins : nullptr, W, S, T, nq, nkv, nq / nkv, max_blocks, num_blocks, nwg, ulen, ulen ? way : 0, ulen ? least : 1, scale * LOG2E};
  switch (d) {
    case 64: return launch_d<64>(a, rf, wide, rows, st);
    case 96: return launch_d<96>(a, rf, wide, rows, st);
    case 128: return launch_d<128>(a, rf, wide, rows, st);
  }
  return -4;
}
