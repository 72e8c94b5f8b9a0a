// The paged cache in 8 bits: a K or V vector of one token and head is e4m3 codes (OCP: 448 the largest, no infinity) and one f32 scale.
//   scale = top / 448, code = e4m3(448 x / top), top = max |x|, at least 2^-100.
// Layouts as the bf16 cache's: K [blocks, nkv, 16, d], V [blocks, nkv, d, 16], scales [blocks, nkv, 16].
//
// 448 = 0.875 * 512, so that nothing overflows.  0.875 x is exact for a bf16 value and the quotient is rounded to f32 once ahead of the code: one that lies
// half way between two codes stays there and goes to the even one, as in exact arithmetic.  A rotated K has 24 bits and is rounded in both steps: within
// 2^-23 of a tie it may go to the other side, which is a code's half step either way.  A vector with an infinity or NaN reads back as NaN.
#include "common.h"

namespace {
constexpr int BS = 16;

struct Kv8Args {
  const u16 *x, *v;                    // rows of heads * d values: q | k | v of a token, or k (and v apart)
  long x_ld, v_ld;
  const int *pos, *slots;
  const float* cos_sin;                // [max_pos, d], null: nothing is rotated
  u16* q_out;
  uint8_t *kc, *vc;
  float *ks, *vs;
  int T, nq, nkv, d, num_blocks, max_pos;
};

// Codes of 16 values of one vector held by eight lanes (those from d / 16 on hold zeros), and its scale.
static __device__ __forceinline__ float quantise(const float* f, uint32_t* code) {
  float top = 0.f;
  bool nan = false;
#pragma unroll
  for (int j = 0; j < 16; ++j) { top = fmaxf(top, fabsf(f[j])); nan |= !(fabsf(f[j]) < INFINITY); }
  if (nan) top = INFINITY;
  top = lane_max(lane_max(lane_max(top, 1), 2), 4);
  top = fmaxf(top, 0x1p-100f);
  const float den = top * 0x1p-9f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    float y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = fminf(fmaxf(f[4 * w + j] * 0.875f / den, -448.f), 448.f);
    int c = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    code[w] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], c, true);
  }
  if (top == INFINITY) {
#pragma unroll
    for (int w = 0; w < 4; ++w) code[w] = 0x7f7f7f7fu;               // NaN
    return 1.f;
  }
  return top / 448.f;
}

// A workgroup has sixteen neighbouring tokens and two heads (of q, k and v in a row); eight lanes a vector, each with eight values of either half (i and
// i + d / 2 are rotated together).  V goes through LDS, so that a store holds neighbouring tokens of neighbouring dims, as the transposed cache has
// them: with a byte a token and dim from where it was computed 6 prompts of 300 to 2001 tokens (32 heads over 8 of 128) took 58 us, now 34.5 (3.8 TB/s of 131 MB;
// rows of two halves and the cosines beside them).  A step's 48 tokens: 4.0 us in a captured graph, a launch's own time.
constexpr int TOK = 16, HEADS = 2;

// Tokens 4 q .. 4 q + 3 have neighbouring places of one block, from a multiple of four on.
static __device__ __forceinline__ bool four(const int* slot, int q, int limit) {
  const int s = slot[4 * q];
  return s >= 0 && s < limit && !(s & 3) && slot[4 * q + 1] == s + 1 && slot[4 * q + 2] == s + 2 && slot[4 * q + 3] == s + 3;
}

__global__ void __launch_bounds__(256) kv8_write_kernel(Kv8Args a) {
#pragma clang fp contract(off)
  __shared__ alignas(16) uint8_t vt[HEADS][TOK][128 + 4];           // (rows of 33 words: sixteen tokens of one dim reach sixteen banks)
  __shared__ int slot[TOK];
  const int heads = a.nq + 2 * a.nkv, half = a.d >> 1, limit = a.num_blocks * BS;
  const int l8 = threadIdx.x & 7, i0 = 8 * l8, tok = (threadIdx.x >> 3) & (TOK - 1), hh = threadIdx.x >> 7;
  const int h = blockIdx.y * HEADS + hh;
  const long t = (long)blockIdx.x * TOK + tok;
  if (threadIdx.x < TOK) slot[threadIdx.x] = (long)blockIdx.x * TOK + threadIdx.x < a.T ? a.slots[(long)blockIdx.x * TOK + threadIdx.x] : -1;
  const bool act = t < a.T && h < heads && i0 < half;
  float f[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) f[j] = 0.f;
  if (act) {
    const u16* src = a.v && h >= a.nq + a.nkv ? a.v + t * a.v_ld + (long)(h - a.nq - a.nkv) * a.d : a.x + t * a.x_ld + (long)h * a.d;
    unpack8(ld16(src + i0), f);
    unpack8(ld16(src + half + i0), f + 8);
    if (a.cos_sin && h < a.nq + a.nkv) {
      const float* cs = a.cos_sin + (long)min(max(a.pos[t], 0), a.max_pos - 1) * a.d;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float c = cs[i0 + j], s = cs[half + i0 + j], x1 = f[j], x2 = f[8 + j];
        f[j] = x1 * c - x2 * s;
        f[8 + j] = x2 * c + x1 * s;
      }
    }
  }
  if (h < a.nq && act) {
    u16* dst = a.q_out + (t * a.nq + h) * a.d;
    st16(dst + i0, pack8(f));
    st16(dst + half + i0, pack8(f + 8));
  }
  if ((int)(blockIdx.y + 1) * HEADS <= a.nq) return;                 // q alone (the whole workgroup)
  uint32_t code[4];
  const float scale = quantise(f, code);
  __syncthreads();
  const int at = slot[tok];
  const bool is_v = h >= a.nq + a.nkv;
  if (act && h >= a.nq) {
    const int kh = h - a.nq - (is_v ? a.nkv : 0);
    if (at >= 0 && at < limit) {
      const long head = (long)(at / BS) * a.nkv + kh;
      if (l8 == 0) (is_v ? a.vs : a.ks)[head * BS + at % BS] = scale;
      if (!is_v) {
        uint8_t* dst = a.kc + (head * BS + at % BS) * a.d;
        *reinterpret_cast<uint2*>(dst + i0) = make_uint2(code[0], code[1]);
        *reinterpret_cast<uint2*>(dst + half + i0) = make_uint2(code[2], code[3]);
      }
    }
    if (is_v) {
      uint32_t* to = reinterpret_cast<uint32_t*>(&vt[hh][tok][0]);
      to[2 * l8] = code[0]; to[2 * l8 + 1] = code[1];
      to[half / 4 + 2 * l8] = code[2]; to[half / 4 + 2 * l8 + 1] = code[3];
    }
  }
  if ((int)(blockIdx.y + 1) * HEADS <= a.nq + a.nkv) return;
  __syncthreads();
  // a thread: a dim's four tokens, a wave sixteen neighbouring dims
  for (int e = threadIdx.x; e < HEADS * 4 * a.d; e += 256) {
    const int q = e & 3, dim = (e >> 2) % a.d, w = (e >> 2) / a.d, kh = (int)blockIdx.y * HEADS + w - a.nq - a.nkv;
    if (kh < 0 || kh >= a.nkv) continue;
    uint32_t c[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) c[j] = vt[w][4 * q + j][dim];
    if (four(slot, q, limit)) {
      const int s = slot[4 * q];
      *reinterpret_cast<uint32_t*>(a.vc + (((long)(s / BS) * a.nkv + kh) * a.d + dim) * BS + s % BS) = c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int s = slot[4 * q + j];
        if (s >= 0 && s < limit) a.vc[(((long)(s / BS) * a.nkv + kh) * a.d + dim) * BS + s % BS] = (uint8_t)c[j];
      }
    }
  }
}

// Tokens back as bf16 rows; a slot outside the pool gives zeros.  A workgroup has sixteen tokens of one head; V through LDS as above (4001
// tokens, 8 heads of 128: 12.4 -> 6.7 us, 3.7 TB/s).
__global__ void __launch_bounds__(256) kv8_read_kernel(const uint8_t* __restrict__ kc, const uint8_t* __restrict__ vc, const float* __restrict__ ks,
                                                       const float* __restrict__ vs, const int* __restrict__ slots, u16* __restrict__ k,
                                                       u16* __restrict__ v, int T, int nkv, int d, int num_blocks) {
  __shared__ alignas(16) uint8_t vt[TOK][128 + 4];
  __shared__ int slot[TOK];
  const int kh = blockIdx.y, limit = num_blocks * BS;
  const long t0 = (long)blockIdx.x * TOK;
  if (threadIdx.x < TOK) {
    const int s = t0 + threadIdx.x < T ? slots[t0 + threadIdx.x] : -1;
    slot[threadIdx.x] = s < limit ? s : -1;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < 4 * d; e += 256) {
    const int q = e & 3, dim = e >> 2;
    uint32_t c[4] = {0u, 0u, 0u, 0u};
    if (four(slot, q, limit)) {
      const int s = slot[4 * q];
      const uint32_t x = *reinterpret_cast<const uint32_t*>(vc + (((long)(s / BS) * nkv + kh) * d + dim) * BS + s % BS);
#pragma unroll
      for (int j = 0; j < 4; ++j) c[j] = x >> (8 * j) & 0xffu;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int s = slot[4 * q + j];
        if (s >= 0) c[j] = vc[(((long)(s / BS) * nkv + kh) * d + dim) * BS + s % BS];
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) vt[4 * q + j][dim] = (uint8_t)c[j];
  }
  __syncthreads();
  const int units = d >> 3;                                         // eight values a thread
  for (int e = threadIdx.x; e < TOK * units; e += 256) {
    const int tok = e / units, i0 = (e % units) * 8;
    const long t = t0 + tok;
    if (t >= T) continue;
    const int s = slot[tok];
    uint2 c = make_uint2(0u, 0u);
    float sk = 0.f, sv = 0.f;
    if (s >= 0) {
      const long at = ((long)(s / BS) * nkv + kh) * BS + s % BS;
      c = *reinterpret_cast<const uint2*>(kc + at * d + i0);
      sk = ks[at];
      sv = vs[at];
    }
    const uint32_t* x = reinterpret_cast<const uint32_t*>(&vt[tok][i0]);
    const uint32_t w[4] = {c.x, c.y, x[0], x[1]};
    float f[16];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(w[j], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w[j], true);
      const float m = j < 2 ? sk : sv;
      f[4 * j] = lo[0] * m; f[4 * j + 1] = lo[1] * m; f[4 * j + 2] = hi[0] * m; f[4 * j + 3] = hi[1] * m;
    }
    st16(k + (t * nkv + kh) * d + i0, pack8(f));
    st16(v + (t * nkv + kh) * d + i0, pack8(f + 8));
  }
}
}  // namespace

extern "C" int dllm_kv8_write(const void* x, long x_ld, const void* v, long v_ld, const int* pos, const float* cos_sin, int max_pos, const int* slots,
                              void* q_out, void* kc, void* vc, float* ks, float* vs, int T, int nq, int nkv, int d, int num_blocks, hipStream_t st) {
  if (T < 1 || nkv < 1 || nq < 0 || d < 16 || d > 128 || d % 16 || num_blocks < 1 || (cos_sin && (!pos || max_pos < 1)) || (nq && !q_out)) return -1;
  Kv8Args a{(const u16*)x, (const u16*)v, x_ld, v_ld, pos, slots, cos_sin, (u16*)q_out, (uint8_t*)kc, (uint8_t*)vc, ks, vs, T, nq, nkv, d, num_blocks, max_pos};
  if ((nq + 2 * nkv + 1) / 2 > 65535 || num_blocks > 0x7fffffff / BS) return -2;
  hipLaunchKernelGGL(kv8_write_kernel, dim3((T + TOK - 1) / TOK, (nq + 2 * nkv + HEADS - 1) / HEADS), dim3(256), 0, st, a);
  return (int)hipGetLastError();
}

extern "C" int dllm_kv8_read(const void* kc, const void* vc, const float* ks, const float* vs, const int* slots, void* k, void* v, int T, int nkv, int d,
                             int num_blocks, hipStream_t st) {
  if (T < 1 || nkv < 1 || d < 16 || d > 128 || d % 16 || num_blocks < 1) return -1;
  if (nkv > 65535 || num_blocks > 0x7fffffff / BS) return -2;
  hipLaunchKernelGGL(kv8_read_kernel, dim3((T + TOK - 1) / TOK, nkv), dim3(256), 0, st, (const uint8_t*)kc, (const uint8_t*)vc, ks, vs, slots, (u16*)k,
                     (u16*)v, T, nkv, d, num_blocks);
  return (int)hipGetLastError();
}
