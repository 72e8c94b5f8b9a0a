// Bindings of the operators of a speculative step (csrc/kernels/tree_attn.hip, draft.hip) and of the 8-bit cache (kv8.hip).
//
// Arguments are checked here, with the words that distributed_llm_amd/ops/draft.py and kv8.py use for CPU tensors; launches go to the current
// stream of the tensors' device, whichever device is current.
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/extension.h>

#include <algorithm>
#include <array>

extern "C" {
int dllm_tree_attention(const void*, long, long, const void*, const void*, const float*, const float*, const int*, const int*, const int*, const int*,
                        const int*, void*, float*, float*, int*, int, int, int, int, int, int, int, int, int, int, int, int, int, int, int, float, hipStream_t);
int dllm_tree_mask(const int*, const int*, const int*, int*, int*, int, int, int, hipStream_t);
int dllm_verify_parts(int, int*);
int dllm_verify(const void*, long, const void*, long, int, const int*, const int*, const float*, const int*, const int*, int*, int*, int*, double*, int*,
                int, int, int, int, hipStream_t);
int dllm_keep(void*, void*, float*, float*, const int*, const int*, const int*, const int*, const int*, int, int, int, int, int, int, int, int,
              hipStream_t);
int dllm_kv8_write(const void*, long, const void*, long, const int*, const float*, int, const int*, void*, void*, void*, float*, float*, int, int, int,
                   int, int, hipStream_t);
int dllm_kv8_read(const void*, const void*, const float*, const float*, const int*, void*, void*, int, int, int, int, hipStream_t);
}

namespace {
using at::Tensor;
using OptTensor = c10::optional<Tensor>;
constexpr int64_t BS = 16, MAX_NODES = 1024;

#define NEED(cond, ...) TORCH_CHECK_VALUE(cond, __VA_ARGS__)

hipStream_t stream() { return c10::hip::getCurrentHIPStream().stream(); }
void launched(int rc, const char* what) { TORCH_CHECK(rc == 0, what, " launch failed, code ", rc); }

void same_device(const Tensor& a, const Tensor& t, const char* name) { NEED(t.device() == a.device(), name, " is on another device"); }
void vec_i32(const Tensor& a, const Tensor& t, const char* name, int64_t n) {
  same_device(a, t, name);
  NEED(t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == n && t.is_contiguous(), name, ": contiguous int32 [", n, "]");
}
bool aligned(const Tensor& t, uintptr_t n) { return (uintptr_t)t.data_ptr() % n == 0; }
bool overlap(const Tensor& a, const Tensor& b) {
  const char *pa = (const char*)a.data_ptr(), *pb = (const char*)b.data_ptr();
  auto bytes = [](const Tensor& t) {
    int64_t n = 1;
    for (int64_t i = 0; i < t.dim(); ++i) n += (t.size(i) - 1) * t.stride(i);
    return n * (int64_t)t.element_size();
  };
  return pa < pb + bytes(b) && pb < pa + bytes(a);
}

struct CacheDims {
  int64_t blocks, nkv, d;
  bool eight;
};
// K [.., blocks, nkv, 16, d], V [.., blocks, nkv, d, 16]; with scales [.., blocks, nkv, 16] both are e4m3.
CacheDims check_cache(const Tensor& a, const Tensor& k, const Tensor& v, const OptTensor& ks, const OptTensor& vs, int64_t lead) {
  same_device(a, k, "k_cache");
  same_device(a, v, "v_cache");
  NEED(k.dim() == 4 + lead && v.dim() == 4 + lead && k.is_contiguous() && v.is_contiguous() && k.size(lead + 2) == BS && v.size(lead + 3) == BS &&
           v.size(lead + 2) == k.size(lead + 3) && v.size(lead + 1) == k.size(lead + 1) && v.size(lead) == k.size(lead) && (!lead || k.size(0) == v.size(0)),
       "cache layout: contiguous K [blocks, nkv, 16, d], V [blocks, nkv, d, 16]");
  CacheDims c{k.size(lead), k.size(lead + 1), k.size(lead + 3), ks.has_value()};
  NEED(ks.has_value() == vs.has_value(), "k_scale and v_scale come together");
  const auto type = c.eight ? at::kFloat8_e4m3fn : at::kBFloat16;
  NEED(k.scalar_type() == type && v.scalar_type() == type, c.eight ? "a cache with scales is float8_e4m3fn" : "a cache without scales is bfloat16");
  NEED(aligned(k, 16) && aligned(v, 16), "caches must be 16-byte aligned");
  if (c.eight)
    for (const Tensor& t : {*ks, *vs}) {
      same_device(a, t, "scales");
      NEED(t.scalar_type() == at::kFloat && t.is_contiguous() && t.dim() == 3 + lead && t.size(lead) == c.blocks && t.size(lead + 1) == c.nkv &&
               t.size(lead + 2) == BS && (!lead || t.size(0) == k.size(0)),
           "scales: contiguous f32 [blocks, nkv, 16]");
    }
  return c;
}
void check_int(int64_t n, const char* name) { NEED(n <= 0x7fff0000, name, ": too many"); }      // (with room to round up in 32 bits)

int cus(const Tensor& t) {
  static std::array<int, 64> known{};
  const int i = t.device().index();
  if (i < 0 || i >= 64) return 256;
  if (!known[i]) {
    int n = 0;
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, i) != hipSuccess || n < 8) n = 256;
    known[i] = n;
  }
  return known[i];
}

Tensor tree_attention(Tensor q, Tensor k, Tensor v, Tensor bt, Tensor qstart, Tensor qlen, Tensor ctx, OptTensor mask, double scale, OptTensor ks,
                      OptTensor vs, int64_t max_qlen, int64_t max_ctx, OptTensor out) {
  NEED(q.dim() == 3 && q.scalar_type() == at::kBFloat16 && q.stride(2) == 1 && q.stride(0) % 8 == 0 && q.stride(1) % 8 == 0 && aligned(q, 16),
       "q: bfloat16 [T, nq, d] with rows of 16-byte alignment");
  const int64_t T = q.size(0), nq = q.size(1), d = q.size(2);
  const CacheDims c = check_cache(q, k, v, ks, vs, 0);
  NEED(c.d == d && (d == 64 || d == 96 || d == 128), "head_dim must be 64, 96 or 128, and the cache's");
  NEED(c.nkv >= 1 && nq >= 1 && nq % c.nkv == 0, "query heads must be a multiple of the cache's");
  same_device(q, bt, "block_tables");
  NEED(bt.dim() == 2 && bt.scalar_type() == at::kInt && bt.is_contiguous(), "block_tables: contiguous int32 [num_seqs, max_blocks]");
  const int64_t S = bt.size(0), max_blocks = c.blocks ? bt.size(1) : 0;      // (an empty pool has no key for any table)
  vec_i32(q, qstart, "seq_qstart", S);
  vec_i32(q, qlen, "seq_qlen", S);
  vec_i32(q, ctx, "seq_ctx", S);
  NEED(max_qlen >= 0 && max_ctx >= 0, "max_qlen and max_ctx: 0 (unknown) or more");
  int64_t W = 0;
  if (mask) {
    same_device(q, *mask, "mask");
    NEED(mask->dim() == 2 && mask->scalar_type() == at::kInt && mask->is_contiguous() && mask->size(0) == T && mask->size(1) >= 1,
         "mask: contiguous int32 [T, words]");
    W = mask->size(1);
  }
  if (out) {
    same_device(q, *out, "out");
    NEED(out->sizes() == q.sizes() && out->scalar_type() == at::kBFloat16 && out->is_contiguous() && aligned(*out, 16),
         "out: contiguous bfloat16 like q, 16-byte aligned");
    NEED(T == 0 || !overlap(*out, q), "out overlaps q");
  }
  for (int64_t n : {T, nq, S, max_blocks * BS, c.blocks}) check_int(n, "tree_attention");
  const c10::OptionalDeviceGuard guard(q.device());
  Tensor o = out ? *out : at::empty({T, nq, d}, q.options());
  if (T == 0 || S == 0) return o;
  const int64_t G = nq / c.nkv;
  const int64_t most = std::min(max_qlen ? max_qlen : S == 1 ? T : W ? 32 * W : T, T) * G;
  const int64_t keys = std::min(max_ctx ? max_ctx : max_blocks * BS, max_blocks * BS);
  // Rows of a wave, and whether four waves have rows of their own over shared keys (bf16).  us, sequences of 200 to 3000 keys, 8 kv heads of 128, one
  // wave's 16 / 32 / 48 rows, four waves' 64 / 128: 48 rows 65 / 61 / 58, 54 / 63; 80 to 160 rows 163 / 117 / 115, 104 / 82; 512 rows of 8000 to 32000
  // keys 940 / 389 / 327, 281 / 203 (four waves' after that, with one address a chunk and finer units: 48 rows 42, then 65 and 178).  e4m3 keys cost conversions in every wave that shares them, or LDS bandwidth as bf16: the last one 488 / 217 / 182
  // and 286 / 211, 48 rows 46 / 41 / 37 and 43 / 51.
  // What fits the chip at once in 16-row blocks is cut that fine, for the shortest way through (one chat of 437 keys, 40 rows, in two launches: 12.2 us, 10.4 so).
  const int64_t fine = S * c.nkv * ((most + 15) / 16) * ((keys + 255) / 256);
  const bool wide = !c.eight && most > 32 && fine > cus(q);
  const int rf = wide ? (most <= 64 ? 1 : 2) : most <= 16 || fine <= cus(q) ? 1 : most <= 32 ? 2 : 3;
  int64_t nwg = (int64_t)cus(q) * 2 / 8 * 8;      // two workgroups a CU (three: 70 -> 81 us for single tokens over 8 bits)
  const int64_t R = 16 * rf * (wide ? 4 : 1);
  const int64_t blocks = S * c.nkv * ((most + R - 1) / R);      // row blocks, at most
  // Keys of a unit (of whole rounds of a workgroup's chunks), units that a row block's way in and out counts for, and units of a part, at least: short
  // parts of long contexts leave many pieces to join.  us with a way of 0 / 2 / 3 / 4 / 6 units: ragged trees of 80 to 160 rows 94 / 78 / 75 / 74 / 75, 160
  // rows of a chain 108 / 91 / 87 / 86 / 92; 48 rows over e4m3 39 / 37 / 35 / 35 / 36; 16 rows are bound by memory, 64 single tokens of up to 6000 keys
  // 113 / 116 / 118 (0 / 1 / 2 units where contexts are shorter: 512 of 200 to 1000 keys, 4 kv heads of 64, 68 / 65 / 65; 2000 of 100 to 400 146 / 141 / 140;
  // 0 / 1 for even and for ragged contexts: 32 of 1500 45 / 48, of 200 to 1500 24 / 24; 8 of 1000 14 / 16, of 300 to 1000 15 / 13; 128 of 1500 149 / 150, of 200
  // to 1500 88 / 85, 4 kv heads of 64 48 / 49 and 25 / 23).
  // With units of 256 keys and no way 82, 100, 37, 113.  Parts of 512 keys and more from 4096 on: one sequence of 16000 65 -> 55.  A context of up to
  // 512 keys is one unit, not split: one launch (us in a graph with a bound of 256 / 512 / 1024 keys: one chat of 437, masks beside it, 10.7 / 9.0 / 9.0; 64 of
  // 300 to 500 20 / 16.5 / 16.4; one of 800 and 40 nodes 22 / 22 / 33; 512 of up to 1000 and 5 nodes 86 / 86 / 101).  Parts are then of whole row blocks, as
  // uneven as their lengths, so from more than five row blocks a workgroup on contexts of more than 256 keys are cut after all.  us whole / cut, 8 kv heads of
  // 128, one token, bf16 and e4m3: 96 sequences of 500 keys 48 / 50 and 29 / 32, 128 of 300 to 500 48 / 54 and 31 / 33, of 20 to 500 27 / 27 and 21 / 27, 256 of
  // those 59 / 53 and 39 / 42, 384 91 / 76 and 62 / 61, 512 117 / 96 and 84 / 79; 384 of 500 159 / 162 and 105 / 109.  48 trees of 40 nodes 36 / 51.
  const int64_t listed = c.nkv * (T * G / R + S);      // row blocks, at most, however long the longest
  int64_t ulen = keys <= 256 || (keys <= 512 && std::min(blocks, listed) <= 5 * nwg) ? 0 : wide ? 64 : c.eight && rf == 1 ? 256 : 128;
  const int64_t way = wide ? 4 : rf > 1 ? 3 : c.eight || keys <= 4096 ? 1 : 0, least = ulen ? (keys > 4096 ? 512 : 256) / ulen : 1;
  // the list of units is counted in 32 bits
  NEED(c.nkv < (1 << 20), "tree_attention: too many heads");
  NEED(T * nq <= 0x7fffffff && listed < (1 << 30), "tree_attention: too many");
  while (ulen && listed * (max_blocks * BS / ulen + 1 + way) >= (1 << 30)) ulen *= 2;
  nwg = std::min(nwg, (blocks * (ulen ? (keys + ulen - 1) / ulen : 1) + 7) / 8 * 8);
  Tensor part;
  float *po = nullptr, *pml = nullptr;
  int* joins = nullptr;
  if (ulen) {
    const int64_t rows = 2 * nwg * R;
    part = at::empty({rows * (d + 2) + 8 * nwg + 1}, q.options().dtype(at::kFloat));
    po = part.data_ptr<float>();
    pml = po + rows * d;
    joins = reinterpret_cast<int*>(pml + rows * 2);
  }
  const int64_t join_rows = std::min(R, most);
  launched(dllm_tree_attention(q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), v.data_ptr(), ks ? ks->data_ptr<float>() : nullptr,
                               vs ? vs->data_ptr<float>() : nullptr, bt.data_ptr<int>(), qstart.data_ptr<int>(), qlen.data_ptr<int>(), ctx.data_ptr<int>(),
                               mask ? mask->data_ptr<int>() : nullptr, o.data_ptr(), po, pml, joins, (int)W, (int)S, (int)T, (int)nq, (int)c.nkv, (int)d,
                               (int)max_blocks, (int)c.blocks, (int)nwg, (int)ulen, (int)way, (int)least, rf, wide, (int)join_rows, (float)scale, stream()),
           "tree_attention");
  return o;
}

std::tuple<Tensor, Tensor> tree_mask(Tensor parents, Tensor qstart, Tensor qlen, int64_t max_nodes) {
  NEED(parents.dim() == 1 && parents.scalar_type() == at::kInt && parents.is_contiguous(), "parents: contiguous int32 [T]");
  NEED(max_nodes >= 1 && max_nodes <= MAX_NODES, "max_nodes must be 1 to ", MAX_NODES);
  const int64_t T = parents.size(0), S = qstart.numel(), W = (max_nodes + 31) / 32;
  vec_i32(parents, qstart, "seq_qstart", S);
  vec_i32(parents, qlen, "seq_qlen", S);
  check_int(T, "tree_mask");
  check_int(S, "tree_mask");
  const c10::OptionalDeviceGuard guard(parents.device());
  Tensor mask = at::empty({T, W}, parents.options()), depth = at::empty({T}, parents.options());
  if (T) launched(dllm_tree_mask(parents.data_ptr<int>(), qstart.data_ptr<int>(), qlen.data_ptr<int>(), mask.data_ptr<int>(), depth.data_ptr<int>(), (int)W, (int)S, (int)T, stream()), "tree_mask");
  return {mask, depth};
}

std::tuple<Tensor, Tensor, Tensor> verify(Tensor target, Tensor tokens, Tensor uniform, Tensor qstart, Tensor qlen, int64_t max_nodes, OptTensor parents,
                                          OptTensor draft) {
  NEED(target.dim() == 2 && (target.scalar_type() == at::kFloat || target.scalar_type() == at::kBFloat16) && target.size(1) >= 1 &&
           (target.stride(1) == 1 || target.size(1) == 1), "target: float32 or bfloat16 [T, vocab]");
  const int64_t T = target.size(0), V = target.size(1), S = qstart.numel();
  vec_i32(target, tokens, "tokens", T);
  same_device(target, uniform, "uniform");
  NEED(uniform.scalar_type() == at::kFloat && uniform.dim() == 1 && uniform.size(0) == T && uniform.is_contiguous(), "uniform: contiguous float32 [T]");
  vec_i32(target, qstart, "seq_qstart", S);
  vec_i32(target, qlen, "seq_qlen", S);
  NEED(max_nodes >= 1 && max_nodes <= MAX_NODES, "max_nodes must be 1 to ", MAX_NODES);
  NEED(!(parents && draft), "a tree's candidates are given, not drawn: parents or draft, not both");
  if (parents) vec_i32(target, *parents, "parents", T);
  if (draft) {
    same_device(target, *draft, "draft");
    NEED(draft->sizes() == target.sizes() && draft->scalar_type() == target.scalar_type() && (draft->stride(1) == 1 || V == 1), "draft: like target");
  }
  NEED(S <= 65535, "at most 65535 sequences");
  check_int(T, "verify");
  check_int(V, "verify");
  const c10::OptionalDeviceGuard guard(target.device());
  const auto i32 = qstart.options();
  Tensor accepted = at::empty({S}, i32), next = at::empty({S}, i32), path = at::empty({S, max_nodes}, i32);
  if (S == 0) return {accepted, next, path};
  if (T == 0) {
    accepted.zero_();
    next.fill_(-1);
    path.fill_(-1);
    return {accepted, next, path};
  }
  int part = 0;
  const int64_t P = dllm_verify_parts((int)V, &part);
  Tensor sums = at::empty({S * P * 2}, target.options().dtype(at::kDouble)), found = at::empty({S * (P + 1) * 2}, i32);
  launched(dllm_verify(target.data_ptr(), target.stride(0), draft ? draft->data_ptr() : nullptr, draft ? draft->stride(0) : 0,
                       target.scalar_type() == at::kBFloat16, tokens.data_ptr<int>(), parents ? parents->data_ptr<int>() : nullptr,
                       uniform.data_ptr<float>(), qstart.data_ptr<int>(), qlen.data_ptr<int>(), accepted.data_ptr<int>(), next.data_ptr<int>(),
                       path.data_ptr<int>(), sums.data_ptr<double>(), found.data_ptr<int>(), (int)S, (int)T, (int)V, (int)max_nodes, stream()),
           "verify");
  return {accepted, next, path};
}

void keep(Tensor k, Tensor v, Tensor bt, Tensor qlen, Tensor ctx, Tensor path, Tensor accepted, OptTensor ks, OptTensor vs) {
  NEED(k.dim() == 4 || k.dim() == 5, "caches: one layer's or [layers, ...]");
  const int64_t lead = k.dim() - 4;
  const CacheDims c = check_cache(k, k, v, ks, vs, lead);
  NEED(c.d >= 16 && c.d <= 128 && c.d % 16 == 0, "head_dim must be a multiple of 16, at most 128");
  same_device(k, bt, "block_tables");
  NEED(bt.dim() == 2 && bt.scalar_type() == at::kInt && bt.is_contiguous(), "block_tables: contiguous int32 [num_seqs, max_blocks]");
  const int64_t S = bt.size(0), max_blocks = bt.size(1), L = lead ? k.size(0) : 1;
  vec_i32(k, qlen, "seq_qlen", S);
  vec_i32(k, ctx, "seq_ctx", S);
  vec_i32(k, accepted, "accepted", S);
  same_device(k, path, "path");
  NEED(path.dim() == 2 && path.scalar_type() == at::kInt && path.is_contiguous() && path.size(0) == S && path.size(1) >= 1,
       "path: contiguous int32 [num_seqs, max_nodes]");
  NEED(S <= 65535, "at most 65535 sequences");
  for (int64_t n : {path.size(1), L * c.nkv, max_blocks * BS, c.blocks}) check_int(n, "keep");
  if (S == 0 || L == 0 || c.blocks == 0 || c.nkv == 0 || max_blocks == 0) return;
  const c10::OptionalDeviceGuard guard(k.device());
  launched(dllm_keep(k.data_ptr(), v.data_ptr(), ks ? ks->data_ptr<float>() : nullptr, vs ? vs->data_ptr<float>() : nullptr, bt.data_ptr<int>(),
                     qlen.data_ptr<int>(), ctx.data_ptr<int>(), path.data_ptr<int>(), accepted.data_ptr<int>(), (int)L, (int)S, (int)path.size(1),
                     (int)c.nkv, (int)c.d, (int)max_blocks, (int)c.blocks, c.eight ? 1 : 2, stream()),
           "keep");
}

CacheDims check_kv8(const Tensor& a, const Tensor& k, const Tensor& v, const Tensor& ks, const Tensor& vs) {
  const CacheDims c = check_cache(a, k, v, ks, vs, 0);
  NEED(c.d >= 16 && c.d <= 128 && c.d % 16 == 0, "head_dim must be a multiple of 16, at most 128");
  check_int(c.blocks * BS, "slots");
  return c;
}

Tensor kv8_rope(Tensor qkv, Tensor pos, Tensor cos_sin, Tensor slots, Tensor k, Tensor v, Tensor ks, Tensor vs, int64_t nq, int64_t nkv, int64_t d,
                OptTensor out) {
  NEED(qkv.dim() == 2 && qkv.scalar_type() == at::kBFloat16 && qkv.stride(1) == 1 && qkv.stride(0) % 8 == 0 && aligned(qkv, 16),
       "qkv: bfloat16 [T, (nq + 2 nkv) d] with rows of 16-byte alignment");
  const CacheDims c = check_kv8(qkv, k, v, ks, vs);
  NEED(c.nkv == nkv && c.d == d && nq >= 0 && nkv >= 1 && qkv.size(1) >= (nq + 2 * nkv) * d, "qkv and cache disagree on heads or head_dim");
  const int64_t T = qkv.size(0);
  vec_i32(qkv, pos, "positions", T);
  vec_i32(qkv, slots, "slots", T);
  same_device(qkv, cos_sin, "cos_sin");
  NEED(cos_sin.dim() == 2 && cos_sin.scalar_type() == at::kFloat && cos_sin.is_contiguous() && cos_sin.size(1) == d && cos_sin.size(0) >= 1,
       "cos_sin: contiguous float32 [max_pos, d]");
  check_int(cos_sin.size(0), "positions");
  check_int(T, "tokens");
  if (out) {
    same_device(qkv, *out, "q_out");
    NEED(out->dim() == 3 && out->size(0) == T && out->size(1) == nq && out->size(2) == d && out->scalar_type() == at::kBFloat16 && out->is_contiguous() &&
             aligned(*out, 16), "q_out: contiguous bfloat16 [T, nq, d], 16-byte aligned");
    NEED(T == 0 || nq == 0 || !overlap(*out, qkv), "q_out overlaps qkv");
  }
  const c10::OptionalDeviceGuard guard(qkv.device());
  Tensor q = out ? *out : at::empty({T, nq, d}, qkv.options());
  if (T == 0 || c.blocks == 0) { NEED(T == 0, "the cache has no blocks"); return q; }
  launched(dllm_kv8_write(qkv.data_ptr(), qkv.stride(0), nullptr, 0, pos.data_ptr<int>(), cos_sin.data_ptr<float>(), (int)cos_sin.size(0),
                          slots.data_ptr<int>(), q.data_ptr(), k.data_ptr(), v.data_ptr(), ks.data_ptr<float>(), vs.data_ptr<float>(), (int)T, (int)nq,
                          (int)nkv, (int)d, (int)c.blocks, stream()),
           "kv8_write");
  return q;
}

void kv8_write(Tensor x, Tensor y, Tensor slots, Tensor k, Tensor v, Tensor ks, Tensor vs) {
  for (const Tensor& t : {x, y})
    NEED(t.dim() == 3 && t.scalar_type() == at::kBFloat16 && t.sizes() == x.sizes() && t.stride(2) == 1 && (t.stride(1) == t.size(2) || t.size(1) == 1) &&
             t.stride(0) % 8 == 0 && aligned(t, 16), "k, v: bfloat16 [T, nkv, d] with rows of 16-byte alignment");
  same_device(x, y, "v");
  const CacheDims c = check_kv8(x, k, v, ks, vs);
  NEED(c.nkv == x.size(1) && c.d == x.size(2) && c.nkv >= 1, "k, v and cache disagree on heads or head_dim");
  const int64_t T = x.size(0);
  vec_i32(x, slots, "slots", T);
  check_int(T, "tokens");
  if (T == 0) return;
  NEED(c.blocks >= 1, "the cache has no blocks");
  const c10::OptionalDeviceGuard guard(x.device());
  launched(dllm_kv8_write(x.data_ptr(), x.stride(0), y.data_ptr(), y.stride(0), nullptr, nullptr, 0, slots.data_ptr<int>(), nullptr, k.data_ptr(),
                          v.data_ptr(), ks.data_ptr<float>(), vs.data_ptr<float>(), (int)T, 0, (int)c.nkv, (int)c.d, (int)c.blocks, stream()),
           "kv8_write");
}

std::tuple<Tensor, Tensor> kv8_read(Tensor k, Tensor v, Tensor ks, Tensor vs, Tensor slots) {
  const CacheDims c = check_kv8(k, k, v, ks, vs);
  NEED(slots.dim() == 1, "slots: contiguous int32 [T]");
  const int64_t T = slots.size(0);
  vec_i32(k, slots, "slots", T);
  check_int(T, "tokens");
  const c10::OptionalDeviceGuard guard(k.device());
  const auto bf = k.options().dtype(at::kBFloat16);
  Tensor x = at::empty({T, c.nkv, c.d}, bf), y = at::empty({T, c.nkv, c.d}, bf);
  if (T == 0 || c.nkv == 0) return {x, y};
  NEED(c.blocks >= 1, "the cache has no blocks");
  launched(dllm_kv8_read(k.data_ptr(), v.data_ptr(), ks.data_ptr<float>(), vs.data_ptr<float>(), slots.data_ptr<int>(), x.data_ptr(), y.data_ptr(), (int)T,
                         (int)c.nkv, (int)c.d, (int)c.blocks, stream()),
           "kv8_read");
  return {x, y};
}
}  // namespace

void bind_draft(pybind11::module_& m) {
  m.def("tree_attention", &tree_attention);
  m.def("tree_mask", &tree_mask);
  m.def("verify_drafts", &verify);
  m.def("keep_drafts", &keep);
  m.def("kv8_rope", &kv8_rope);
  m.def("kv8_write", &kv8_write);
  m.def("kv8_read", &kv8_read);
}
