// Drafted tokens beside the attention over them: the masks of a tree, verification against the target's probabilities, and the move of the
// accepted nodes' K and V behind the committed ones.
//
// A sequence's nodes are its rows qstart .. qstart + qlen - 1, the root (the last committed token) first, every node behind its parent.
#include "common.h"

namespace {
constexpr int BS = 16;
constexpr int MAX_NODES = 1024;
constexpr int NTH = 256;

// ------------------------------------------------------------------------------------------------ masks
// Workgroup s < S: a node's word of ancestors (itself among them) and their number, from a walk up the parents in LDS; indices fall on the way,
// so a word is whole when the walk leaves it (32 trees of 20 to 40 nodes 4 us, a launch's own time).  Workgroups behind: rows that no sequence has, or that lie past 32 W nodes of it, become
// zero; a thread looks at every 256th sequence and marks what it has of the workgroup's rows (a row that looks for its sequence by itself: 512 sequences 70 us, 4 so).
__global__ void __launch_bounds__(NTH) tree_mask_kernel(const int* __restrict__ parents, const int* __restrict__ qstart, const int* __restrict__ qlen,
                                                        int* __restrict__ mask, int* __restrict__ depth, int W, int S, int T) {
  __shared__ int par[MAX_NODES];
  if ((int)blockIdx.x >= S) {
    const int t0 = (blockIdx.x - S) * NTH, t = t0 + threadIdx.x;
    par[threadIdx.x] = 0;
    __syncthreads();
    for (int s = threadIdx.x; s < S; s += NTH) {
      const int q0 = qstart[s], n = min(qlen[s], 32 * W);
      if (n <= 0 || q0 < 0 || q0 > T - n) continue;
      for (int i = max(q0, t0); i < min(q0 + n, t0 + NTH); ++i) par[i - t0] = 1;
    }
    __syncthreads();
    if (t >= T || par[threadIdx.x]) return;
    for (int w = 0; w < W; ++w) mask[(long)t * W + w] = 0;
    depth[t] = 0;
    return;
  }
  const int q0 = qstart[blockIdx.x], n = min(qlen[blockIdx.x], 32 * W);
  if (q0 < 0 || q0 > T - n) return;
  for (int i = threadIdx.x; i < n; i += NTH) par[i] = parents[q0 + i];
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += NTH) {
    int* to = mask + (long)(q0 + i) * W;
    int w = W - 1, up = -1;
    uint32_t bits = 0;
    for (int at = i; at >= 0;) {
      for (; w > (at >> 5); --w) { to[w] = (int)bits; bits = 0; }
      bits |= 1u << (at & 31);
      ++up;
      const int p = par[at];
      at = p < at ? p : -1;
    }
    for (; w >= 0; --w) { to[w] = (int)bits; bits = 0; }
    depth[q0 + i] = up;
  }
}

// ------------------------------------------------------------------------------------------------ verification
template <class T> static __device__ __forceinline__ float val(const T* p);
template <> __device__ __forceinline__ float val<float>(const float* p) { return *p; }
template <> __device__ __forceinline__ float val<u16>(const u16* p) { return bf2f(*p); }

// Four neighbouring values; `vec`: rows are 16-byte (f32) or 8-byte (bf16) aligned.
static __device__ __forceinline__ void val4(const float* p, bool vec, float* f) {
  if (vec) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = p[j];
  }
}
static __device__ __forceinline__ void val4(const u16* p, bool vec, float* f) {
  if (vec) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    f[0] = __uint_as_float(v.x << 16); f[1] = __uint_as_float(v.x & 0xffff0000u);
    f[2] = __uint_as_float(v.y << 16); f[3] = __uint_as_float(v.y & 0xffff0000u);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = bf2f(p[j]);
  }
}

struct VerifyArgs {
  const void *target, *draft;          // [T, V]; draft may be null
  long target_ld, draft_ld;
  const int *tokens, *parents;         // [T]; parents may be null (node i - 1)
  const float* uniform;                // [T]
  const int *qstart, *qlen;
  int *accepted, *next, *path;         // [S], [S], [S, N]
  double* sums;                        // [S, P, 2]
  int* found;                          // [S, P + 1, 2]: last index with weight, of each part; [P]: the path's last node, whether children were refused
  int S, T, V, N, P, part;
};

struct VerifySmem {
  int par[MAX_NODES], tok[MAX_NODES], nxt[MAX_NODES], out[MAX_NODES];
  double px[MAX_NODES];
  unsigned char ok[MAX_NODES];
  double wsum[NTH / 64][2];
  int wlast[NTH / 64][2];
  int nout;
};

static __device__ __forceinline__ int parent_of(const VerifyArgs& a, int q0, int i) {
  if (i == 0) return -1;
  const int p = a.parents ? a.parents[q0 + i] : i - 1;
  return p >= 0 && p < i ? p : -2;                                  // none: a node that cannot be reached
}

// Tokens of `last`'s children inside [v0, v1) that the last draw leaves out (trees: candidates are refused for good).
static __device__ __forceinline__ void left_out(const VerifyArgs& a, VerifySmem& sm, int n, int last, int v0, int v1) {
  if (threadIdx.x == 0) sm.nout = 0;
  __syncthreads();
  if (a.draft == nullptr)
    for (int i = threadIdx.x; i < n; i += NTH)
      if (sm.par[i] == last && sm.tok[i] >= v0 && sm.tok[i] < v1) sm.out[atomicAdd(&sm.nout, 1)] = sm.tok[i];    // (a set: its order does not matter)
  __syncthreads();
}

// p and q at v .. v + 3, zeros from `end` on (a part's end, or the row's).
template <class T> static __device__ __forceinline__ void fetch(const T* p, const T* q, int v, int end, bool vec, float* f, float* h) {
#pragma unroll
  for (int j = 0; j < 4; ++j) f[j] = h[j] = 0.f;
  if (v + 4 <= end) {
    val4(p + v, vec, f);
    if (q) val4(q + v, vec, h);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (v + j < end) {
        f[j] = val<T>(p + v + j);
        if (q) h[j] = val<T>(q + v + j);
      }
  }
}
// Weights of the last draw there: max(p - q, 0), exact in 64 bits; NaN counts as nothing.
static __device__ __forceinline__ void weights(const float* f, const float* h, int v, const VerifySmem& sm, double* w, double* pw) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const double x = (double)f[j] - (double)h[j];
    w[j] = x > 0.0 ? x : 0.0;
    pw[j] = f[j] > 0.f ? (double)f[j] : 0.0;
  }
  for (int i = 0; i < sm.nout; ++i) {
    const int k = sm.out[i] - v;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (k == j) w[j] = 0.0;
  }
}

// v of lane j (uniform)
static __device__ __forceinline__ double lane64(double v, int j) {
  return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), j), __builtin_amdgcn_readlane(__double2loint(v), j));
}
static __device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

template <class T> static __device__ __forceinline__ bool vectors(const VerifyArgs& a) {
  const uintptr_t m = 4 * sizeof(T) - 1;
  return !((uintptr_t)a.target & m) && !(a.target_ld * sizeof(T) & m) && !((uintptr_t)a.draft & m) && (!a.draft || !(a.draft_ld * sizeof(T) & m));
}

// What earlier siblings left of the target, 0 at least; a NaN among them stays one (fmax would make it 0, and any later sibling would be accepted).
static __device__ __forceinline__ double left(double mass) { return mass < 0.0 ? 0.0 : mass; }

// Where the accepted path ends, and its length, of more than 64 nodes: a thread a node, in LDS.
template <class T> static __device__ __forceinline__ void tree_walk(const VerifyArgs& a, VerifySmem& sm, int q0, int n, int& last, int& len) {
  const T *target = (const T*)a.target, *draft = (const T*)a.draft;
  const int tid = threadIdx.x;
  for (int i = tid; i < n; i += NTH) {
    const int p = parent_of(a, q0, i), x = a.tokens[q0 + i];
    sm.par[i] = p;
    sm.tok[i] = x;
    sm.nxt[i] = -1;
    sm.ok[i] = 0;
    const bool real = p >= 0 && x >= 0 && x < a.V;
    const double px = real ? (double)val<T>(target + (long)(q0 + p) * a.target_ld + x) : 0.0;
    sm.px[i] = px;
    if (draft && real) sm.ok[i] = (double)a.uniform[q0 + i] * (double)val<T>(draft + (long)(q0 + i) * a.draft_ld + x) < px;
  }
  __syncthreads();
  if (!draft) {
    bool twice[MAX_NODES / NTH];
#pragma unroll
    for (int c = 0; c < MAX_NODES / NTH; ++c) {
      const int i = tid + c * NTH;
      twice[c] = false;
      if (i < n && sm.par[i] >= 0)
        for (int j = sm.par[i] + 1; j < i; ++j) twice[c] |= sm.par[j] == sm.par[i] && sm.tok[j] == sm.tok[i];
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < MAX_NODES / NTH; ++c)
      if (twice[c]) sm.px[tid + c * NTH] = 0.0;
    __syncthreads();
    for (int i = tid; i < n; i += NTH)
      if (sm.par[i] >= 0) {
        double mass = 1.0;
        for (int j = sm.par[i] + 1; j < i; ++j)
          if (sm.par[j] == sm.par[i]) mass -= sm.px[j];
        sm.ok[i] = sm.tok[i] >= 0 && sm.tok[i] < a.V && (double)a.uniform[q0 + i] * left(mass) < sm.px[i];
      }
    __syncthreads();
  }
  for (int i = tid; i < n; i += NTH)                                 // a parent's first accepted child
    if (sm.ok[i]) {
      bool is_first = true;
      for (int j = sm.par[i] + 1; j < i; ++j) is_first &= !(sm.ok[j] && sm.par[j] == sm.par[i]);
      if (is_first) sm.nxt[sm.par[i]] = i;
    }
  __syncthreads();
  last = 0;
  len = 1;
  for (int k = sm.nxt[0]; k >= 0; k = sm.nxt[k]) { last = k; ++len; }
}

// The walk, in every workgroup of a sequence (a few dependent loads: it costs less than a launch of its own), then the weights' sum of this one's part of the
// vocabulary; the token is found by a second launch.  Node i is accepted where u q(x) < p(x) (drawn from q), or u m < p(x), m = 1 less what its earlier
// siblings held (given candidates): products of f32 and f64 values, exact or rounded once, so a token does not hang on the order of sums.
// 48 chains, 128256 tokens: 13 us of the walk's four trips to memory and 49 MB (3.8 TB/s), 7.5 for the second launch; one chain of 32000: 6.0 and 5.8.
template <class T> __global__ void __launch_bounds__(NTH) verify_walk_kernel(VerifyArgs a) {
  __shared__ VerifySmem sm;
  const int s = blockIdx.y, tid = threadIdx.x, q0 = a.qstart[s];
  int n = min(a.qlen[s], a.N);
  if (q0 < 0 || q0 > a.T - n) n = 0;
  if (n <= 0) {
    if (blockIdx.x == 0) {
      if (tid == 0) { a.accepted[s] = 0; a.found[((long)s * (a.P + 1) + a.P) * 2] = -1; }
      for (int i = tid; i < a.N; i += NTH) a.path[(long)s * a.N + i] = -1;
    }
    return;
  }
  const T *target = (const T*)a.target, *draft = (const T*)a.draft;
  int* path = a.path + (long)s * a.N;
  int last = 0, len = 1;
  bool refused;
  const int v0 = blockIdx.x * a.part, v1 = v0 + min(a.V - v0, a.part);      // (a whole last part may end past 2^31)
  if (n <= 64) {
    // a lane a node, in every wave by itself, without LDS (trees of 40 nodes: 16 us of a launch in LDS, 9 so)
    const int i = tid & 63, x = i < n ? a.tokens[q0 + i] : -1, par = i < n ? parent_of(a, q0, i) : -3;
    const bool real = par >= 0 && x >= 0 && x < a.V;
    double px = real ? (double)val<T>(target + (long)(q0 + par) * a.target_ld + x) : 0.0, mass = 1.0;
    const double u = i < n ? (double)a.uniform[q0 + i] : 0.0;
    if (a.parents)
      for (int j = 1; j < n; ++j) {                                  // siblings in order: what each held, and tokens that come again
        const int pj = __builtin_amdgcn_readlane(par, j), xj = __builtin_amdgcn_readlane(x, j);
        const double held = lane64(px, j);
        if (i > j && par == pj) {
          mass -= held;
          if (x == xj) px = 0.0;
        }
      }
    bool take = real && (draft ? u * (double)val<T>(draft + (long)(q0 + i) * a.draft_ld + x) < px : u * left(mass) < px);
    for (unsigned long long m = __ballot(take); m; m &= m - 1) {     // a parent's first accepted child
      const int j = __builtin_ctzll(m), pj = __builtin_amdgcn_readlane(par, j);
      if (i > j && par == pj) take = false;
    }
    int step = 0;
    for (unsigned long long m; (m = __ballot(take && par == last)) != 0; ++len) {
      last = __builtin_ctzll(m);
      if (i == len) step = last;
    }
    const unsigned long long kids = __ballot(par == last);
    refused = kids != 0;
    if (tid < 64) {
      const unsigned long long out = draft ? 0ull : __ballot(par == last && x >= v0 && x < v1);
      if (i == 0) sm.nout = __popcll(out);
      if (out >> i & 1) sm.out[__popcll(out & ((1ull << i) - 1))] = x;
      if (blockIdx.x == 0)
        for (int j = i; j < a.N; j += 64) path[j] = j < len ? step : -1;
    }
    __syncthreads();
  } else {
    tree_walk<T>(a, sm, q0, n, last, len);
    bool mine = false;
    for (int i = tid; i < n; i += NTH) mine |= sm.par[i] == last;
    refused = __syncthreads_or(mine);
    if (blockIdx.x == 0) {
      for (int i = len + tid; i < a.N; i += NTH) path[i] = -1;
      if (tid == 0)
        for (int i = 0, k = 0; i < len; ++i, k = sm.nxt[k]) path[i] = k;
    }
    left_out(a, sm, n, last, v0, v1);
  }
  if (blockIdx.x == 0 && tid == 0) {
    a.accepted[s] = len - 1;
    int* f = a.found + ((long)s * (a.P + 1) + a.P) * 2;
    f[0] = last;
    f[1] = refused;
  }
  const T* p = target + (long)(q0 + last) * a.target_ld;
  const T* q = draft && refused ? draft + (long)(q0 + last + 1) * a.draft_ld : nullptr;
  const bool vec = vectors<T>(a);
  double ws = 0.0, ps = 0.0;
  int wl = -1, pl = -1;
  // (four vectors asked for at once cost a workgroup on the CU: 17 us where this takes 13)
  for (int v = v0 + 4 * tid; v < v1; v += 4 * NTH) {
    float f[4], h[4];
    double w[4], pw[4];
    fetch(p, q, v, v1, vec, f, h);
    weights(f, h, v, sm, w, pw);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      ws += w[j];
      ps += pw[j];
      if (w[j] > 0.0) wl = v + j;
      if (pw[j] > 0.0) pl = v + j;
    }
  }
  ws = wave_sum64(ws);
  ps = wave_sum64(ps);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) { wl = max(wl, __shfl_xor(wl, o, 64)); pl = max(pl, __shfl_xor(pl, o, 64)); }
  if ((tid & 63) == 0) {
    sm.wsum[tid >> 6][0] = ws; sm.wsum[tid >> 6][1] = ps;
    sm.wlast[tid >> 6][0] = wl; sm.wlast[tid >> 6][1] = pl;
  }
  __syncthreads();
  if (tid < 2) {
    double t = 0.0;
    int l = -1;
    for (int i = 0; i < NTH / 64; ++i) { t += sm.wsum[i][tid]; l = max(l, sm.wlast[i][tid]); }
    a.sums[((long)s * a.P + blockIdx.x) * 2 + tid] = t;
    a.found[((long)s * (a.P + 1) + blockIdx.x) * 2 + tid] = l;
  }
}

// The next token: the smallest index whose running sum passes u times the whole; the last one with weight where rounding leaves none; weights
// that are all zero (p nowhere above q) give way to p itself, and a row without any probability to token 0.
template <class T> __global__ void __launch_bounds__(NTH) verify_pick_kernel(VerifyArgs a) {
  __shared__ VerifySmem sm;
  __shared__ double cum[NTH];
  const int s = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const int* f = a.found + ((long)s * (a.P + 1) + a.P) * 2;
  const int last = f[0];
  if (last < 0) {
    if (tid == 0) a.next[s] = -1;
    return;
  }
  const int q0 = a.qstart[s], n = min(a.qlen[s], a.N);
  if (!a.draft)
    for (int i = tid; i < n; i += NTH) { sm.par[i] = parent_of(a, q0, i); sm.tok[i] = a.tokens[q0 + i]; }
  // parts (at most NTH): running sums, whole weights first
  const double* sums = a.sums + (long)s * a.P * 2;
  const int* lasts = a.found + (long)s * (a.P + 1) * 2;
  auto scan = [&](double x) {                                        // inclusive, over the workgroup
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double y = __shfl_up(x, o, 64);
      if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 63) sm.wsum[wid][0] = x;
    __syncthreads();
    double before = 0.0;
    for (int i = 0; i < wid; ++i) before += sm.wsum[i][0];
    x += before;
    cum[tid] = x;
    __syncthreads();
    return x;
  };
  // The first thread with weight whose sum passes t, NTH if none does (not the one between two sums: rounding may leave sums of neighbours in the wrong
  // order, and a thread without weight a bit above the one before it).
  auto first_over = [&](double own, double sum, double t) {
    const unsigned long long over = __ballot(own > 0.0 && sum > t);
    if (lane == 0) sm.wlast[wid][1] = over ? 64 * wid + __builtin_ctzll(over) : NTH;
    __syncthreads();
    int m = NTH;
#pragma unroll
    for (int i = 0; i < NTH / 64; ++i) m = min(m, sm.wlast[i][1]);
    return m;
  };
  int which = 0;
  const double mine = tid < a.P ? sums[2 * tid] : 0.0, own_p = tid < a.P ? sums[2 * tid + 1] : 0.0;
  const int last_w = tid < a.P ? lasts[2 * tid] : -1, last_p = tid < a.P ? lasts[2 * tid + 1] : -1;
  double incl = scan(mine);
  if (!(cum[NTH - 1] > 0.0)) {
    which = 1;
    __syncthreads();
    incl = scan(own_p);
  }
  const double whole = cum[NTH - 1], t = (double)a.uniform[q0] * whole;
  int l = which ? last_p : last_w;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) l = max(l, __shfl_xor(l, o, 64));
  if (lane == 0) sm.wlast[wid][0] = l;
  const int part = first_over(which ? own_p : mine, incl, t);
  if (part >= a.P) {                                                 // (infinite sums, or u = 1)
    if (tid == 0) {
      int m = -1;
      for (int i = 0; i < NTH / 64; ++i) m = max(m, sm.wlast[i][0]);
      a.next[s] = max(m, 0);
    }
    return;
  }
  const double base = part ? cum[part - 1] : 0.0;
  const int v0 = part * a.part, v1 = v0 + min(a.V - v0, a.part), each = a.part / NTH;
  left_out(a, sm, which ? 0 : n, last, v0, v1);
  const T* p = (const T*)a.target + (long)(q0 + last) * a.target_ld;
  const T* q = a.draft && f[1] && !which ? (const T*)a.draft + (long)(q0 + last + 1) * a.draft_ld : nullptr;
  const bool vec = vectors<T>(a);
  const int from = v0 + tid * each, to = from + min(v1 - from, each);
  // sixteen weights of a thread stay in registers; longer rows than 16 NTH NTH read theirs again
  double w[16], pw[4], own = 0.0;
  float f4[4][4], h4[4][4];
#pragma unroll
  for (int c = 0; c < 4; ++c) fetch(p, q, from + 4 * c, to, vec, f4[c], h4[c]);
#pragma unroll
  for (int c = 0; c < 4; ++c) weights(f4[c], h4[c], from + 4 * c, sm, w + 4 * c, pw);
#pragma unroll
  for (int j = 0; j < 16; ++j) own += w[j];
  for (int v = from + 16; v < to; v += 4) {
    double x[4];
    fetch(p, q, v, to, vec, f4[0], h4[0]);
    weights(f4[0], h4[0], v, sm, x, pw);
    own += x[0]; own += x[1]; own += x[2]; own += x[3];
  }
  const double up = base + scan(own), down = tid ? base + cum[tid - 1] : base;
  const int who = first_over(own, up, t);
  if (who == NTH && tid == 0) a.next[s] = max(lasts[2 * part + which], 0);
  if (tid == who) {
    double run = down;
    int got = -1;
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (w[j] > 0.0 && (got < 0 || !(run > t))) { run += w[j]; got = from + j; }
    for (int v = from + 16; v < to; v += 4) {
      double x[4];
      fetch(p, q, v, to, vec, f4[0], h4[0]);
      weights(f4[0], h4[0], v, sm, x, pw);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (x[j] > 0.0 && (got < 0 || !(run > t))) { run += x[j]; got = v + j; }
    }
    a.next[s] = got;
  }
}

// ------------------------------------------------------------------------------------------------ keep
struct KeepArgs {
  void *kc, *vc;                       // [L, blocks, nkv, 16, d], [L, blocks, nkv, d, 16]
  float *ks, *vs;                      // [L, blocks, nkv, 16] or null
  const int *bt, *qlen, *ctx, *path, *accepted;
  int L, S, N, nkv, d, max_blocks, num_blocks;
};

// V is a column of a transposed block, two bytes of every 32: a move touches lines of 32 d bytes for 2 d, which bounds it (32 sequences, 32 layers of 8 heads of
// 128: 25 MB moved, about 100 MB of lines, each counted once however many of its tokens move, 30 us; four heads a workgroup 36).
// A workgroup: one sequence, layer and kv head.  Path indices rise and node path[j] goes to place j <= path[j]: sixteen tokens at a time are
// read, then written, and what is written lies ahead of every later source.  E: bytes of a value.
template <int E> __global__ void __launch_bounds__(NTH) keep_kernel(KeepArgs a) {
  const int s = blockIdx.y, kvh = blockIdx.x % a.nkv, layer = blockIdx.x / a.nkv, tid = threadIdx.x;
  const int base = a.ctx[s] - a.qlen[s], n = min(min(a.accepted[s], a.N - 1), a.qlen[s] - 1);
  const int* path = a.path + (long)s * a.N;
  const int* bt = a.bt + (long)s * a.max_blocks;
  const long heads = ((long)layer * a.num_blocks) * a.nkv + kvh;     // + page * nkv: a (layer, page, head)
  auto place = [&](int at, long& head, int& off) {
    const int i = base + at;
    if (at < 0 || at >= a.qlen[s] || i < 0 || i >= a.max_blocks * BS) return false;
    const int page = bt[i / BS];
    if ((unsigned)page >= (unsigned)a.num_blocks) return false;
    head = heads + (long)page * a.nkv;
    off = i % BS;
    return true;
  };
  __shared__ long from[16], to[16];                                  // head * 16 + offset
  __shared__ int moves;
  for (int j0 = 1; j0 <= n; j0 += 16) {
    __syncthreads();
    if (tid == 0) moves = 0;
    __syncthreads();
    if (tid < 16) {
      const int j = j0 + tid;
      long h0 = 0, h1 = 0;
      int o0 = 0, o1 = 0;
      const bool move = j <= n && path[j] > j && place(path[j], h0, o0) && place(j, h1, o1);
      from[tid] = move ? h0 * BS + o0 : -1;
      to[tid] = h1 * BS + o1;
      if (move) moves = 1;
    }
    __syncthreads();
    if (!moves) continue;
    const int kv = a.d * E / 16;                                     // 16-byte vectors of a K row
    constexpr int KM = 128 * E / 16 * 16 / NTH > 0 ? 128 * E / 16 * 16 / NTH : 1, VM = 128 * 16 / NTH;
    uint4 kr[KM];
    uint32_t vr[VM];
    float sr[2] = {0.f, 0.f};
#pragma unroll
    for (int c = 0; c < KM; ++c) {
      const int e = tid + c * NTH, j = e / kv;
      if (j < 16 && from[j] >= 0) kr[c] = ld16((const uint8_t*)a.kc + from[j] * a.d * E + (e % kv) * 16);
    }
#pragma unroll
    for (int c = 0; c < VM; ++c) {
      const int e = tid + c * NTH, j = e / a.d, i = e % a.d;
      if (j < 16 && from[j] >= 0) {
        const long at = ((from[j] / BS) * a.d + i) * BS + from[j] % BS;
        vr[c] = E == 2 ? ((const u16*)a.vc)[at] : ((const uint8_t*)a.vc)[at];
      }
    }
    if (a.ks && tid < 16 && from[tid] >= 0) { sr[0] = a.ks[from[tid]]; sr[1] = a.vs[from[tid]]; }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < KM; ++c) {
      const int e = tid + c * NTH, j = e / kv;
      if (j < 16 && from[j] >= 0) st16((uint8_t*)a.kc + to[j] * a.d * E + (e % kv) * 16, kr[c]);
    }
#pragma unroll
    for (int c = 0; c < VM; ++c) {
      const int e = tid + c * NTH, j = e / a.d, i = e % a.d;
      if (j < 16 && from[j] >= 0) {
        const long at = ((to[j] / BS) * a.d + i) * BS + to[j] % BS;
        if (E == 2) ((u16*)a.vc)[at] = (u16)vr[c];
        else ((uint8_t*)a.vc)[at] = (uint8_t)vr[c];
      }
    }
    if (a.ks && tid < 16 && from[tid] >= 0) { a.ks[to[tid]] = sr[0]; a.vs[to[tid]] = sr[1]; }
  }
}
}  // namespace

extern "C" int dllm_tree_mask(const int* parents, const int* qstart, const int* qlen, int* mask, int* depth, int W, int S, int T, hipStream_t st) {
  if (W < 1 || W > MAX_NODES / 32 || S < 0 || T < 1) return -1;
  hipLaunchKernelGGL(tree_mask_kernel, dim3(S + (T + NTH - 1) / NTH), dim3(NTH), 0, st, parents, qstart, qlen, mask, depth, W, S, T);
  return (int)hipGetLastError();
}

// Parts of a row: `part` values each, at most NTH of them.
extern "C" int dllm_verify_parts(int V, int* part) {
  int p = 16 * NTH;
  while (((long)V + p - 1) / p > NTH) p *= 2;
  *part = p;
  return (int)(((long)V + p - 1) / p);
}

extern "C" int dllm_verify(const void* target, long target_ld, const void* draft, long draft_ld, int bf16, const int* tokens, const int* parents,
                           const float* uniform, const int* qstart, const int* qlen, int* accepted, int* next, int* path, double* sums, int* found, int S,
                           int T, int V, int N, hipStream_t st) {
  if (S < 1 || S > 65535 || T < 1 || V < 1 || N < 1 || N > MAX_NODES || (draft && parents)) return -1;
  VerifyArgs a{target, draft, target_ld, draft_ld, tokens, parents, uniform, qstart, qlen, accepted, next, path, sums, found, S, T, V, N, 0, 0};
  a.P = dllm_verify_parts(V, &a.part);
  if (bf16) {
    hipLaunchKernelGGL(verify_walk_kernel<u16>, dim3(a.P, S), dim3(NTH), 0, st, a);
    hipLaunchKernelGGL(verify_pick_kernel<u16>, dim3(S), dim3(NTH), 0, st, a);
  } else {
    hipLaunchKernelGGL(verify_walk_kernel<float>, dim3(a.P, S), dim3(NTH), 0, st, a);
    hipLaunchKernelGGL(verify_pick_kernel<float>, dim3(S), dim3(NTH), 0, st, a);
  }
  return (int)hipGetLastError();
}

extern "C" int dllm_keep(void* kc, void* vc, float* ks, float* vs, const int* bt, const int* qlen, const int* ctx, const int* path, const int* accepted,
                         int L, int S, int N, int nkv, int d, int max_blocks, int num_blocks, int bytes, hipStream_t st) {
  if (L < 1 || S < 1 || S > 65535 || N < 1 || nkv < 1 || d < 16 || d > 128 || d % 16 || max_blocks < 1 || num_blocks < 1) return -1;
  if ((bytes != 1 && bytes != 2) || (ks == nullptr) != (bytes == 2) || (vs == nullptr) != (bytes == 2)) return -2;
  if ((long)L * nkv > 0x7fffffffL) return -3;
  KeepArgs a{kc, vc, ks, vs, bt, qlen, ctx, path, accepted, L, S, N, nkv, d, max_blocks, num_blocks};
  if (bytes == 2) hipLaunchKernelGGL(keep_kernel<2>, dim3(L * nkv, S), dim3(NTH), 0, st, a);
  else hipLaunchKernelGGL(keep_kernel<1>, dim3(L * nkv, S), dim3(NTH), 0, st, a);
  return (int)hipGetLastError();
}
