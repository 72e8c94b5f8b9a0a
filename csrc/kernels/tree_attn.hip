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
// A workgroup is four waves over the same RF * 16 rows (heads of one kv head, tokens x group), each with its own chunks: K and V go to
// registers once for all rows and are never staged.  The waves meet in LDS at the end.
//
// e4m3 caches: codes become bf16 exactly (three bits behind the leading one), the key's scale multiplies its score and the value's its weight,
// ahead of the weight's rounding to bf16; the sum of weights is of the unrounded ones.
//
// Split: all (sequence, kv head, row block, range of `ulen` keys) form one list, cut into equal parts for the workgroups that fit the chip at
// once; every workgroup finds its part from the lengths on the device, so ragged batches are even, nothing is planned on the host and a
// captured graph takes new lengths.  A part's first and last piece may be of a row block that others hold too: their sums go to the workspace
// in 32 bits and a second launch joins them, in order (no atomics: the same bits every time).
#include "common.h"

namespace {
constexpr int BS = 16, NW = 4;
constexpr float LOG2E = 1.4426950408889634f;

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
  int W, S, T, nq, nkv, G, max_blocks, num_blocks, nwg, ulen;
  float scale_log2;
};

// ---- the list of units
struct Place {
  int seq;                  // sequence, and unit within it, of one place in the list
  long local;
};
struct Shape {
  int qlen, ctx, nb, nt;    // row blocks and key ranges
};

static __device__ __forceinline__ Shape shape_of(const TreeArgs& a, int s, int R) {
  Shape h;
  h.qlen = max(a.qlen[s], 0);
  h.ctx = min(max(a.ctx[s], 0), a.max_blocks * BS);
  h.nb = (int)(((long)h.qlen * a.G + R - 1) / R);
  h.nt = max(1, (int)(((long)h.ctx + a.ulen - 1) / a.ulen));
  return h;
}
static __device__ __forceinline__ long units_of(const TreeArgs& a, const Shape& h) { return (long)a.nkv * h.nb * h.nt; }

// Units in all; each lane keeps the inclusive sum up to its own sequences.
static __device__ __forceinline__ long scan_units(const TreeArgs& a, int R, long& incl, int& first, int& count) {
  const int lane = threadIdx.x & 63;
  count = (a.S + 63) / 64;
  first = lane * count;
  long own = 0;
  for (int i = 0; i < count; ++i)
    if (first + i < a.S) own += units_of(a, shape_of(a, first + i, R));
  incl = own;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const long y = __shfl_up(incl, o, 64);
    if (lane >= o) incl += y;
  }
  return __shfl(incl, 63, 64);
}
static __device__ __forceinline__ Place place_of(const TreeArgs& a, int R, long incl, int first, int count, long unit) {
  const unsigned long long at = __ballot(incl > unit);        // unit < total: some lane's
  const int who = __builtin_ctzll(at);
  int s = first;
  long before = incl;
  if ((int)(threadIdx.x & 63) == who) {
    long own = 0;
    for (int i = 0; i < count; ++i)
      if (first + i < a.S) own += units_of(a, shape_of(a, first + i, R));
    before -= own;
    for (; s < a.S; ++s) {
      const long n = units_of(a, shape_of(a, s, R));
      if (before + n > unit) break;
      before += n;
    }
  }
  Place p;
  p.seq = __builtin_amdgcn_readlane(s, who);
  p.local = unit - __shfl(before, who, 64);
  return p;
}
static __device__ __forceinline__ long part_len(const TreeArgs& a, long total) { return (total + a.nwg - 1) / a.nwg; }

// ---- operands
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
  static constexpr int CK = EIGHT && RF <= 2 ? 64 : 32;       // keys of a wave's chunk
  static constexpr int KS = D / 32, NT = D / 16, TL = CK / 16, KPG = CK / 4, R = 16 * RF;
  static constexpr bool QL = RF == 4;                         // Q fragments in LDS: their registers would cost a wave a SIMD
  static constexpr int PITCH = D + 4;
};

template <int D, int RF, bool EIGHT> struct TreeSmem {
  using F = Form<D, RF, EIGHT>;
  alignas(16) float o[NW][16][F::PITCH];
  float m[NW][16], l[NW][16];
  alignas(16) float sc[EIGHT ? NW : 1][2][64];                // scales of a wave's chunk
  alignas(16) u16 q[F::QL ? RF * F::KS * 64 * 8 : 8];
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

template <bool EIGHT> static __device__ __forceinline__ bool odd_bits(uint32_t w) {     // an infinity or NaN among the values of a word
  if (EIGHT) {
    const uint32_t t = ~w & 0x7f7f7f7fu;                      // a byte that is 0 here is a NaN code
    return ((t - 0x01010101u) & ~t & 0x80808080u) != 0;
  }
  return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
}
template <bool EIGHT> static __device__ __forceinline__ uint32_t tame(uint32_t w) {     // those as zeros
  if (EIGHT) {
#pragma unroll
    for (int b = 0; b < 32; b += 8)
      if (((w >> b) & 0x7fu) == 0x7fu) w &= ~(0xffu << b);
    return w;
  }
  if ((w & 0x7f80u) == 0x7f80u) w &= 0xffff0000u;
  if ((w & 0x7f800000u) == 0x7f800000u) w &= 0xffffu;
  return w;
}

// Where a piece goes: the output, or slot `slot` of the workspace (< 0: the output).
template <int D, int RF, bool EIGHT>
static __device__ __forceinline__ void piece(const TreeArgs& a, TreeSmem<D, RF, EIGHT>& sm, const int seq, const Shape h, const int kvh, const int blk,
                                             const int k0, const int k1, const int slot) {
  using F = Form<D, RF, EIGHT>;
  constexpr int CK = F::CK, KS = F::KS, NT = F::NT, TL = F::TL, KPG = F::KPG, R = F::R;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, rl = lane & 15;
  const int qstart = a.qstart[seq], base = h.ctx - h.qlen;
  const int* bt = a.bt + (long)seq * a.max_blocks;

  int tok[RF];
  bool ok[RF];
#pragma unroll
  for (int f = 0; f < RF; ++f) {
    const int r = blk * R + 16 * f + rl;
    tok[f] = r / a.G;
    const long at = (long)qstart + tok[f];
    ok[f] = tok[f] < h.qlen && at >= 0 && at < a.T;
  }
  // Q fragments: dims 32 s + 8 g (bf16), or as the code loads deal them (pairs of steps share a 16-byte load)
  auto dim0 = [&](int s) { return EIGHT && (s | 1) < KS ? 64 * (s >> 1) + 16 * g + 8 * (s & 1) : 32 * s + 8 * g; };
  auto q_at = [&](int f, int s) {
    const int head = kvh * a.G + (blk * R + 16 * f + rl) % a.G;
    return ok[f] ? ld16(a.q + (qstart + (long)tok[f]) * a.q_ts + head * a.q_hs + dim0(s)) : make_uint4(0u, 0u, 0u, 0u);
  };
  bf16x8 qr[F::QL ? 1 : RF][KS];
  if constexpr (F::QL) {
    __syncthreads();                                          // the piece before is done with LDS
#pragma unroll
    for (int f = 0; f < RF; ++f)
      if (f % NW == wave) {
#pragma unroll
        for (int s = 0; s < KS; ++s) st16(&sm.q[((f * KS + s) * 64 + lane) * 8], q_at(f, s));
      }
    __syncthreads();
  } else {
#pragma unroll
    for (int f = 0; f < RF; ++f)
#pragma unroll
      for (int s = 0; s < KS; ++s) qr[f][s] = __builtin_bit_cast(bf16x8, q_at(f, s));
  }

  f32x4 acc[RF][NT];
  float m[RF], l[RF];
#pragma unroll
  for (int f = 0; f < RF; ++f) {
    m[f] = -INFINITY;
    l[f] = 0.f;
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[f][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  const int last_block = (h.ctx - 1) >> 4;
  for (int kb = k0 + CK * wave; kb < k1; kb += CK * NW) {
    // blocks of this lane's key rows and of its lane group's keys; a page outside the pool hides its keys
    const int ik = min((kb >> 4) + (CK == 64 ? rl >> 2 : rl >> 3), last_block), iv = min((kb >> 4) + (CK == 64 ? g : g >> 1), last_block);
    const int pk = bt[ik], pv = bt[iv];
    const bool paged = (unsigned)pv < (unsigned)a.num_blocks;
    const long hk = ((long)((unsigned)pk < (unsigned)a.num_blocks ? pk : 0) * a.nkv + kvh) * BS, hv = ((long)(paged ? pv : 0) * a.nkv + kvh) * BS;
    uint32_t kr[TL][KS][EIGHT ? 2 : 4], vr[NT][EIGHT ? (CK == 64 ? 4 : 2) : 4];
#pragma unroll
    for (int t = 0; t < TL; ++t) {
      const long row = hk + (CK == 64 ? 0 : 8 * ((rl >> 2) & 1)) + 4 * t + (rl & 3);
      if constexpr (EIGHT) {
        const uint8_t* p = (const uint8_t*)a.kc + row * D;
#pragma unroll
        for (int s = 0; s < KS; s += 2) {
          if (s + 1 < KS) {
            const uint4 v = ld16(p + 32 * s + 16 * g);
            kr[t][s][0] = v.x; kr[t][s][1] = v.y; kr[t][s + 1][0] = v.z; kr[t][s + 1][1] = v.w;
          } else {
            const uint2 v = *reinterpret_cast<const uint2*>(p + 32 * s + 8 * g);
            kr[t][s][0] = v.x; kr[t][s][1] = v.y;
          }
        }
      } else {
        const u16* p = (const u16*)a.kc + row * D + 8 * g;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          const uint4 v = ld16(p + 32 * s);
          kr[t][s][0] = v.x; kr[t][s][1] = v.y; kr[t][s][2] = v.z; kr[t][s][3] = v.w;
        }
      }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if constexpr (EIGHT) {
        const uint8_t* p = (const uint8_t*)a.vc + hv * D + (16 * n + rl) * BS;
        if constexpr (CK == 64) {
          const uint4 v = ld16(p);
          vr[n][0] = v.x; vr[n][1] = v.y; vr[n][2] = v.z; vr[n][3] = v.w;
        } else {
          const uint2 v = *reinterpret_cast<const uint2*>(p + 8 * (g & 1));
          vr[n][0] = v.x; vr[n][1] = v.y;
        }
      } else {
        const uint4 v = ld16((const u16*)a.vc + hv * D + (16 * n + rl) * BS + 8 * (g & 1));
        vr[n][0] = v.x; vr[n][1] = v.y; vr[n][2] = v.z; vr[n][3] = v.w;
      }
    }
    const bool plain = kb + CK <= base && !__any(!paged);     // every row sees the whole chunk
    bool odd = false;
    if constexpr (EIGHT) {
      // key (lane) of the chunk: 16 keys of block iv, or 8 of one half
      const int key = CK == 64 ? rl : 8 * (g & 1) + (rl & 7);
      float ks = 0.f, vs = 0.f;
      if (paged && kb + KPG * g + (CK == 64 ? rl : rl & 7) < h.ctx) { ks = a.ks[hv + key]; vs = a.vs[hv + key]; }
      if (!plain && !(fabsf(vs) < INFINITY)) { odd = true; vs = 0.f; }
      if (CK == 64 || rl < 8) {
        sm.sc[wave][0][KPG * g + rl] = ks * a.scale_log2;
        sm.sc[wave][1][KPG * g + rl] = vs;
      }
      __builtin_amdgcn_wave_barrier();
    }
    if (!plain) {
      // what no row may see (keys past ctx, pages outside the pool: stale memory) is zero in V; an infinity or NaN of a drafted token that a
      // row does not see would reach it as 0 * inf, so those are zero too and added again below, to the rows that see them
      const int n = paged ? h.ctx - kb - KPG * g : 0;         // keys of this lane that exist
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int w = 0; w < (int)(sizeof(vr[0]) / 4); ++w) {
          const int per = EIGHT ? 4 : 2, left = n - per * w;
          uint32_t x = vr[i][w];
          if (left < per) x &= left <= 0 ? 0u : (1u << ((EIGHT ? 8 : 16) * left)) - 1u;
          odd |= odd_bits<EIGHT>(x);
          vr[i][w] = tame<EIGHT>(x);
        }
    }
    f32x4 sc[RF][TL];
#pragma unroll
    for (int f = 0; f < RF; ++f)
#pragma unroll
      for (int t = 0; t < TL; ++t) sc[f][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      bf16x8 kf[TL];
#pragma unroll
      for (int t = 0; t < TL; ++t) {
        if constexpr (EIGHT) kf[t] = cvt8(make_uint2(kr[t][s][0], kr[t][s][1]));
        else kf[t] = __builtin_bit_cast(bf16x8, make_uint4(kr[t][s][0], kr[t][s][1], kr[t][s][2], kr[t][s][3]));
      }
#pragma unroll
      for (int f = 0; f < RF; ++f) {
        bf16x8 qf;
        if constexpr (F::QL) qf = __builtin_bit_cast(bf16x8, ld16(&sm.q[((f * KS + s) * 64 + lane) * 8]));
        else qf = qr[f][s];
#pragma unroll
        for (int t = 0; t < TL; ++t) sc[f][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[t], qf, sc[f][t], 0, 0, 0);
      }
    }
    bf16x8 pf[RF][CK / 32];
    uint32_t see[RF][CK / 32];
#pragma unroll
    for (int f = 0; f < RF; ++f) {
      float p[KPG];
#pragma unroll
      for (int t = 0; t < TL; ++t) {
        f32x4 ks = f32x4{a.scale_log2, a.scale_log2, a.scale_log2, a.scale_log2};
        if constexpr (EIGHT) ks = *reinterpret_cast<const f32x4*>(&sm.sc[wave][0][KPG * g + 4 * t]);
#pragma unroll
        for (int q = 0; q < 4; ++q) p[4 * t + q] = sc[f][t][q] * ks[q];
      }
      if (!plain) {
#pragma unroll
        for (int w = 0; w < CK / 32; ++w)
          see[f][w] = ok[f] ? window(a, kb + 32 * w, base, h.ctx, tok[f], (long)qstart + tok[f]) : 0u;
        const uint32_t mine = paged ? (CK == 64 ? see[f][g >> 1 & (CK / 32 - 1)] >> (16 * (g & 1)) : see[f][0] >> (8 * g)) : 0u;
#pragma unroll
        for (int j = 0; j < KPG; ++j) p[j] = (mine >> j) & 1u ? p[j] : -INFINITY;
      }
      float top = p[0];
#pragma unroll
      for (int j = 1; j < KPG; ++j) top = fmaxf(top, p[j]);
      top = lane_max(lane_max(top, 16), 32);
      if (__any(top > m[f])) {
        const float m_new = fmaxf(m[f], top), al = __builtin_amdgcn_exp2f(m[f] - (m_new == -INFINITY ? 0.f : m_new));
        m[f] = m_new;
        l[f] *= al;
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[f][n] *= al;
      }
      const float ms = m[f] == -INFINITY ? 0.f : m[f];
#pragma unroll
      for (int j = 0; j < KPG; ++j) { p[j] = __builtin_amdgcn_exp2f(p[j] - ms); l[f] += p[j]; }
      if constexpr (EIGHT) {
#pragma unroll
        for (int t = 0; t < TL; ++t) {
          const f32x4 vs = *reinterpret_cast<const f32x4*>(&sm.sc[wave][1][KPG * g + 4 * t]);
#pragma unroll
          for (int q = 0; q < 4; ++q) p[4 * t + q] *= vs[q];
        }
      }
#pragma unroll
      for (int e = 0; e < CK / 32; ++e) pf[f][e] = __builtin_bit_cast(bf16x8, pack8(p + 8 * e));
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < CK / 32; ++e) {
        bf16x8 vf;
        if constexpr (EIGHT) vf = cvt8(make_uint2(vr[n][2 * e], vr[n][2 * e + 1]));
        else vf = __builtin_bit_cast(bf16x8, make_uint4(vr[n][0], vr[n][1], vr[n][2], vr[n][3]));
#pragma unroll
        for (int f = 0; f < RF; ++f) acc[f][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[f][e], acc[f][n], 0, 0, 0);
      }
    if constexpr (EIGHT) __builtin_amdgcn_wave_barrier();     // scales are read before the next chunk's are written
    if (!plain && __any(odd)) {
      // infinities and NaN, key by key (rare): the values themselves, to the rows that see the key
      for (int j = 0; j < CK && kb + j < h.ctx; ++j) {
        const int page = bt[(kb + j) >> 4];
        if ((unsigned)page >= (unsigned)a.num_blocks) continue;
        const long at = ((long)page * a.nkv + kvh) * BS;
        const int off = (kb + j) & 15;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const long i = at * D + (16 * n + 4 * g + r) * BS + off;
            float v;
            if constexpr (EIGHT) v = __builtin_amdgcn_cvt_f32_fp8(((const uint8_t*)a.vc)[i], 0) * a.vs[at + off];
            else v = bf2f(((const u16*)a.vc)[i]);
            if (!(fabsf(v) < INFINITY)) {
#pragma unroll
              for (int f = 0; f < RF; ++f)
                if ((see[f][CK == 64 ? j >> 5 : 0] >> (j & 31)) & 1u) acc[f][n][r] += v;
            }
          }
      }
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
      float w[NW], M = -INFINITY, L = 0.f, o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < NW; ++i) M = fmaxf(M, sm.m[i][row]);
      const float Ms = M == -INFINITY ? 0.f : M;
#pragma unroll
      for (int i = 0; i < NW; ++i) {
        w[i] = __builtin_amdgcn_exp2f(sm.m[i][row] - Ms);
        L += sm.l[i][row] * w[i];
        const f32x4 x = *reinterpret_cast<const f32x4*>(&sm.o[i][row][col]), y = *reinterpret_cast<const f32x4*>(&sm.o[i][row][col + 4]);
#pragma unroll
        for (int j = 0; j < 4; ++j) { o[j] += x[j] * w[i]; o[4 + j] += y[j] * w[i]; }
      }
      if (slot >= 0) {
        const long at = (long)slot * R + 16 * f + row;
        *reinterpret_cast<f32x4*>(a.part_o + at * D + col) = f32x4{o[0], o[1], o[2], o[3]};
        *reinterpret_cast<f32x4*>(a.part_o + at * D + col + 4) = f32x4{o[4], o[5], o[6], o[7]};
        if (col == 0) { a.part_ml[2 * at] = M; a.part_ml[2 * at + 1] = L; }
        continue;
      }
      const int r = blk * R + 16 * f + row, t = r / a.G;
      const long to = (long)qstart + t;
      if (t >= h.qlen || to < 0 || to >= a.T) continue;
      const float inv = L == 0.f ? 0.f : 1.f / L;             // a row that sees nothing is zero
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] *= inv;
      st16(a.out + (to * a.nq + kvh * a.G + r % a.G) * D + col, pack8(o));
    }
  }
}

template <int D, int RF, bool EIGHT>
__global__ void __launch_bounds__(64 * NW, RF == 4 ? 2 : 1) tree_attn_kernel(TreeArgs a) {
  using F = Form<D, RF, EIGHT>;
  __shared__ TreeSmem<D, RF, EIGHT> sm;
  long incl;
  int first, count;
  const long total = scan_units(a, F::R, incl, first, count);
  if (total == 0) return;
  const long part = part_len(a, total);
  // parts in the order of the list to workgroups of one XCD, whose L2 the row blocks of a kv head then share
  const int parts = (int)((total + part - 1) / part), q8 = parts / 8, r8 = parts % 8, x = blockIdx.x % 8, i = blockIdx.x / 8;
  if (i >= q8 + (x < r8)) return;
  const int me = x * q8 + min(x, r8) + i;
  long u = me * part;
  const long end = min(total, u + part);
  Place p = place_of(a, F::R, incl, first, count, u);
  int seq = p.seq;
  long local = p.local;
  bool begun = false;
  while (u < end) {
    const Shape h = shape_of(a, seq, F::R);
    const long n = units_of(a, h);
    if (local >= n) { ++seq; local = 0; continue; }           // (units are left, so a sequence with units follows)
    const int range = (int)(local % h.nt), row = (int)(local / h.nt), blk = row % h.nb, kvh = row / h.nb;
    const int take = (int)min((long)(h.nt - range), end - u);
    const bool whole = range == 0 && take == h.nt;
    const long k0 = (long)range * a.ulen, k1 = min((long)h.ctx, k0 + (long)take * a.ulen);
    piece<D, RF, EIGHT>(a, sm, seq, h, kvh, blk, (int)k0, (int)k1, whole ? -1 : 2 * me + (begun ? 1 : 0));
    begun = true;
    u += take;
    local += take;
  }
}

// Joins the pieces of one row block that several parts hold.  The workgroup of the first cut inside a block does it: part i's start is inside
// block [b, b + nt) and part i - 1's is not.  blockIdx.y: sixteen rows of it, a wave a row at a time.
template <int D>
__global__ void __launch_bounds__(64 * NW) tree_join_kernel(TreeArgs a, int R) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  long incl;
  int first, count;
  const long total = scan_units(a, R, incl, first, count);
  const long part = total ? part_len(a, total) : 1, cut = (long)(blockIdx.x + 1) * part;
  if (cut >= total) return;
  const Place p = place_of(a, R, incl, first, count, cut);
  const Shape h = shape_of(a, p.seq, R);
  const int range = (int)(p.local % h.nt), row = (int)(p.local / h.nt), blk = row % h.nb, kvh = row / h.nb;
  const long b = cut - range;                                 // the row block's first unit
  if (range == 0 || cut - part > b) return;
  const int i0 = blockIdx.x, i1 = (int)((b + h.nt - 1) / part), qstart = a.qstart[p.seq];
  for (int r16 = wave; r16 < 16; r16 += NW) {
    const int rr = 16 * blockIdx.y + r16, r = blk * R + rr, t = r / a.G;
    const long to = (long)qstart + t;
    if (t >= h.qlen || to < 0 || to >= a.T) continue;
    // part i0's piece of this block is its last one: its second where it began in another block
    auto slot_row = [&](int i) { return ((long)2 * i + ((long)i * part < b ? 1 : 0)) * R + rr; };
    float M = -INFINITY;
    for (int i = i0 + lane; i <= i1; i += 64) M = fmaxf(M, a.part_ml[2 * slot_row(i)]);
    M = wave_max(M);
    const float Ms = M == -INFINITY ? 0.f : M;
    float L = 0.f, o0 = 0.f, o1 = 0.f;
    for (int i = i0; i <= i1; ++i) {
      const long at = slot_row(i);
      const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + 2 * at);
      const float w = __builtin_amdgcn_exp2f(ml.x - Ms);
      L += ml.y * w;
      if (2 * lane < D) {
        const float2 x = *reinterpret_cast<const float2*>(a.part_o + at * D + 2 * lane);
        o0 += x.x * w;
        o1 += x.y * w;
      }
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    if (2 * lane < D)
      *reinterpret_cast<uint32_t*>(a.out + (to * a.nq + kvh * a.G + r % a.G) * D + 2 * lane) = f2bf2(o0 * inv, o1 * inv);
  }
}

template <int D, int RF, bool EIGHT> void launch(const TreeArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((tree_attn_kernel<D, RF, EIGHT>), dim3(a.nwg), dim3(64 * NW), 0, st, a);
}
template <int D> int launch_d(const TreeArgs& a, int rf, bool join, hipStream_t st) {
  const bool e = a.ks != nullptr;
  if (rf == 1) e ? launch<D, 1, true>(a, st) : launch<D, 1, false>(a, st);
  else if (rf == 2) e ? launch<D, 2, true>(a, st) : launch<D, 2, false>(a, st);
  else e ? launch<D, 4, true>(a, st) : launch<D, 4, false>(a, st);
  if (join && a.nwg > 1) hipLaunchKernelGGL((tree_join_kernel<D>), dim3(a.nwg - 1, rf), dim3(64 * NW), 0, st, a, 16 * rf);
  return (int)hipGetLastError();
}
}  // namespace

// rf: row blocks of 16 rf rows (1, 2, 4).  ulen: keys of a unit, a multiple of 256; 0: a row block is one unit (no workspace, one launch).
extern "C" int dllm_tree_attention(const void* q, long q_ts, long q_hs, const void* kc, const void* vc, const float* ks, const float* vs,
                                   const int* bt, const int* qstart, const int* qlen, const int* ctx, const int* mask, void* out, float* part_o,
                                   float* part_ml, int W, int S, int T, int nq, int nkv, int d, int max_blocks, int num_blocks, int nwg, int ulen,
                                   int rf, float scale, hipStream_t st) {
  if (nkv < 1 || nq < nkv || nq % nkv || (rf != 1 && rf != 2 && rf != 4)) return -1;
  if ((ks == nullptr) != (vs == nullptr) || S < 1 || T < 1 || max_blocks < 1 || num_blocks < 1 || nwg < 1) return -2;
  if (ulen < 0 || ulen % 256 || (ulen && (!part_o || !part_ml))) return -3;
  TreeArgs a{(const u16*)q, q_ts, q_hs, kc, vc, ks, vs, bt, qstart, qlen, ctx, mask, (u16*)out, part_o, part_ml,
             W, S, T, nq, nkv, nq / nkv, max_blocks, num_blocks, nwg, ulen ? ulen : 0x7fffff00, scale * LOG2E};
  switch (d) {
    case 64: return launch_d<64>(a, rf, ulen != 0, st);
    case 96: return launch_d<96>(a, rf, ulen != 0, st);
    case 128: return launch_d<128>(a, rf, ulen != 0, st);
  }
  return -4;
}
