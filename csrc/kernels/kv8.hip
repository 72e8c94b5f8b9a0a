// The paged cache in 8 bits: a K or V vector of one token and head is e4m3 codes (OCP: 448 the largest, no infinity) and one f32 scale.
//   scale = top / 448, code = e4m3(448 x / top), top = max |x|, at least 2^-100.
// Layouts as the bf16 cache's: K [blocks, nkv, 16, d], V [blocks, nkv, d, 16], scales [blocks, nkv, 16].
//
// The quotient is rounded to f32 once ahead of the code (448 = 0.875 * 512, so that nothing overflows): a bf16 value that lies half way between
// two codes stays there and goes to the even one, as in exact arithmetic.  A vector with an infinity or NaN reads back as NaN.
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

// Eight lanes a vector, each with eight values of either half (i and i + d / 2 are rotated together).
__global__ void __launch_bounds__(256) kv8_write_kernel(Kv8Args a) {
#pragma clang fp contract(off)
  const int heads = a.nq + 2 * a.nkv, half = a.d >> 1;
  const long id = (long)blockIdx.x * 32 + (threadIdx.x >> 3);
  const int l8 = threadIdx.x & 7, i0 = 8 * l8;
  const long t = id / heads;
  const int h = (int)(id % heads);
  const bool live = t < a.T, act = live && i0 < half;
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
  if (h < a.nq) {
    if (act) {
      u16* dst = a.q_out + (t * a.nq + h) * a.d;
      st16(dst + i0, pack8(f));
      st16(dst + half + i0, pack8(f + 8));
    }
  }
  uint32_t code[4];
  const float scale = quantise(f, code);
  if (!act || h < a.nq) return;
  const int slot = a.slots[t];
  if (slot < 0 || slot >= (long)a.num_blocks * BS) return;
  const bool is_v = h >= a.nq + a.nkv;
  const int kh = h - a.nq - (is_v ? a.nkv : 0), off = slot % BS;
  const long head = (long)(slot / BS) * a.nkv + kh;
  if (l8 == 0) (is_v ? a.vs : a.ks)[head * BS + off] = scale;
  if (!is_v) {
    uint8_t* dst = a.kc + (head * BS + off) * a.d;
    *reinterpret_cast<uint2*>(dst + i0) = make_uint2(code[0], code[1]);
    *reinterpret_cast<uint2*>(dst + half + i0) = make_uint2(code[2], code[3]);
  } else {
    uint8_t* dst = a.vc + head * a.d * BS + off;
#pragma unroll
    for (int j = 0; j < 16; ++j) dst[(long)((j < 8 ? i0 : half + i0 - 8) + j) * BS] = (uint8_t)(code[j >> 2] >> (8 * (j & 3)));
  }
}

// Tokens back as bf16 rows; a slot outside the pool gives zeros.
__global__ void __launch_bounds__(256) kv8_read_kernel(const uint8_t* __restrict__ kc, const uint8_t* __restrict__ vc, const float* __restrict__ ks,
                                                       const float* __restrict__ vs, const int* __restrict__ slots, u16* __restrict__ k,
                                                       u16* __restrict__ v, int T, int nkv, int d, int num_blocks) {
  const int units = d >> 3;
  const long id = (long)blockIdx.x * 256 + threadIdx.x, vec = id / units;
  const int i0 = (int)(id % units) * 8;
  const long t = vec / nkv;
  if (t >= T) return;
  const int kh = (int)(vec % nkv), slot = slots[t];
  float fk[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, fv[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (slot >= 0 && slot < (long)num_blocks * BS) {
    const long head = (long)(slot / BS) * nkv + kh;
    const int off = slot % BS;
    const float sk = ks[head * BS + off], sv = vs[head * BS + off];
    const uint2 c = *reinterpret_cast<const uint2*>(kc + (head * BS + off) * d + i0);
    const uint32_t w[2] = {c.x, c.y};
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(w[j], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w[j], true);
      fk[4 * j] = lo[0] * sk; fk[4 * j + 1] = lo[1] * sk; fk[4 * j + 2] = hi[0] * sk; fk[4 * j + 3] = hi[1] * sk;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) fv[j] = __builtin_amdgcn_cvt_f32_fp8((int)vc[(head * d + i0 + j) * BS + off], 0) * sv;
  }
  st16(k + vec * d + i0, pack8(fk));
  st16(v + vec * d + i0, pack8(fv));
}
}  // namespace

extern "C" int dllm_kv8_write(const void* x, long x_ld, const void* v, long v_ld, const int* pos, const float* cos_sin, int max_pos, const int* slots,
                              void* q_out, void* kc, void* vc, float* ks, float* vs, int T, int nq, int nkv, int d, int num_blocks, hipStream_t st) {
  if (T < 1 || nkv < 1 || nq < 0 || d < 16 || d > 128 || d % 16 || num_blocks < 1 || (cos_sin && (!pos || max_pos < 1)) || (nq && !q_out)) return -1;
  Kv8Args a{(const u16*)x, (const u16*)v, x_ld, v_ld, pos, slots, cos_sin, (u16*)q_out, (uint8_t*)kc, (uint8_t*)vc, ks, vs, T, nq, nkv, d, num_blocks, max_pos};
  const long n = (long)T * (nq + 2 * nkv);
  if ((n + 31) / 32 > 0x7fffffffL) return -2;
  hipLaunchKernelGGL(kv8_write_kernel, dim3((unsigned)((n + 31) / 32)), dim3(256), 0, st, a);
  return (int)hipGetLastError();
}

extern "C" int dllm_kv8_read(const void* kc, const void* vc, const float* ks, const float* vs, const int* slots, void* k, void* v, int T, int nkv, int d,
                             int num_blocks, hipStream_t st) {
  if (T < 1 || nkv < 1 || d < 16 || d > 128 || d % 16 || num_blocks < 1) return -1;
  const long n = (long)T * nkv * (d / 8);
  if ((n + 255) / 256 > 0x7fffffffL) return -2;
  hipLaunchKernelGGL(kv8_read_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, (const uint8_t*)kc, (const uint8_t*)vc, ks, vs, slots, (u16*)k,
                     (u16*)v, T, nkv, d, num_blocks);
  return (int)hipGetLastError();
}
