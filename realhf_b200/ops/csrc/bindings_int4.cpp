// torch bindings for the kernels over 4-bit groups: the cache, its decode attention, weights and their products.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/library.h>
#include <torch/types.h>

#include <limits>

using at::Tensor;
using OptT = c10::optional<Tensor>;

extern "C" {
int rb_int4_cache_rows(void* k, void* v, int64_t kt, int64_t kh, int64_t vt, int64_t vh, void* cache, const int* cu, const int* slots, const int* start, int n, int nkv,
                       int hd, int n_slots, int room, int T, int longest, int store, int dt, cudaStream_t s);
int rb_decode_attention_int4(const void* qkv, void* cache, const int* lens, void* out, const float* cos, const float* sin, int64_t qkv_stride, int B, int nq, int nkv,
                             int hd, int room, int rot_dim, int interleaved, float scale, int dt, cudaStream_t s);
int rb_int4_quantize(const void* w, void* q, int N, int K, int64_t ld, int group, int dt, cudaStream_t s);
int rb_int4_pack(const void* codes, const void* scale, const void* low, void* q, int N, int K, int group, cudaStream_t s);
int rb_int4_linear(const void* x, const void* q, const void* bias, void* y, int M, int N, int K, int64_t ldx, int64_t ldy, int group, int dt, cudaStream_t s);
}

void attn_check();

namespace {

constexpr int64_t kInt = std::numeric_limits<int>::max();

int type_of(const Tensor& t, const char* op) {
  TORCH_CHECK_VALUE(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf, op, ": bfloat16 or float16 expected, not ", t.scalar_type());
  return t.scalar_type() == at::kBFloat16 ? 1 : 2;
}
bool on16(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }
// t itself if its rows lie on 16 bytes with unit inner stride, else a packed copy (not `contiguous()`: a slice of one row counts as that wherever it starts)
Tensor rows16(const Tensor& t) {
  bool ok = t.numel() == 0 || (t.stride(-1) == 1 && on16(t));
  for (int64_t i = 0; ok && t.numel() > 0 && i + 1 < t.dim(); ++i) ok = t.stride(i) % 8 == 0;
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

// int32 [n] on the device of `like`, or null
const int* whole(const OptT& t, int64_t n, const Tensor& like, const char* op, const char* what) {
  if (!t.has_value()) return nullptr;
  TORCH_CHECK_VALUE(t->scalar_type() == at::kInt && t->dim() == 1 && t->size(0) == n && t->is_contiguous() && t->device() == like.device(), op, ": ", what,
                    " is a contiguous int32 vector of ", n, " numbers beside the cache");
  return t->data_ptr<int>();
}

struct CacheDims { int64_t slots, nkv, tiles; };
CacheDims cache_dims(const Tensor& cache, int64_t room, int64_t hd, const char* op) {
  TORCH_CHECK_VALUE(hd == 64 || hd == 128, op, ": heads of 64 or 128 channels, not ", hd);
  const int64_t words = 16 * (hd / 4) + 16 * (hd / 32 + hd / 64);
  TORCH_CHECK_VALUE(cache.is_cuda() && cache.scalar_type() == at::kInt && cache.dim() == 4 && cache.is_contiguous() && cache.size(3) == words && room >= 0 &&
                        room <= kInt - 16 && cache.size(2) == (room + 15) / 16 && cache.size(0) <= kInt && cache.size(1) <= 65535 && on16(cache),
                    op, ": a cache is an int32 tensor [slots, heads, tiles, ", words, "] on a CUDA device");
  return {cache.size(0), cache.size(1), cache.size(2)};
}

void cache_rows(Tensor k, Tensor v, Tensor cache, const Tensor& cu, const OptT& slots, const OptT& start, int64_t room, int64_t hd, int64_t longest, bool store,
                const char* op) {
  TORCH_CHECK_VALUE(k.dim() == 3 && v.dim() == 3 && k.sizes() == v.sizes() && k.scalar_type() == v.scalar_type() && k.device() == cache.device() &&
                        v.device() == cache.device(), op, ": keys and values [tokens, heads, channels] of one type beside the cache");
  const int dt = type_of(k, op);
  const auto d = cache_dims(cache, room, hd, op);
  TORCH_CHECK_VALUE(k.size(1) == d.nkv && k.size(2) == hd && k.size(0) <= kInt, op, ": ", k.size(1), " heads of ", k.size(2), " channels for a cache of ", d.nkv, " of ", hd);
  TORCH_CHECK_VALUE(cu.dim() == 1 && cu.size(0) >= 1, op, ": cu_seqlens holds one number more than there are sequences");
  const int64_t n = cu.size(0) - 1;
  const int *cp = whole(cu, n + 1, cache, op, "cu_seqlens"), *sp = whole(slots, n, cache, op, "slots"), *bp = whole(start, n, cache, op, "start");
  c10::cuda::CUDAGuard guard(cache.device());
  if (store) {
    k = rows16(k);
    v = rows16(v);
  }
  if (longest <= 0) longest = k.size(0) / std::max<int64_t>(n, 1);
  const int rc = rb_int4_cache_rows(k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), v.stride(0), v.stride(1), cache.data_ptr(), cp, sp, bp, (int)n, (int)d.nkv,
                                    (int)k.size(2), (int)d.slots, (int)room, (int)k.size(0), (int)std::min(std::max<int64_t>(longest, 1), kInt), store, dt,
                                    at::cuda::getCurrentCUDAStream().stream());
  TORCH_CHECK(rc == 0, op, ": the kernel could not be launched (", rc, ")");
}

void int4_cache_store(const Tensor& k, const Tensor& v, Tensor cache, const Tensor& cu, const OptT& slots, const OptT& start, int64_t room, int64_t hd,
                      int64_t longest) {
  cache_rows(k, v, cache, cu, slots, start, room, hd, longest, true, "int4_cache_store");
}

// Tokens that belong to no sequence, or whose row or slot is not there, are 0.
std::vector<Tensor> int4_cache_load(const Tensor& cache, const Tensor& cu, const OptT& slots, const OptT& start, int64_t room, int64_t hd, int64_t tokens, int64_t longest,
                                    at::ScalarType dtype) {
  cache_dims(cache, room, hd, "int4_cache_load");
  TORCH_CHECK_VALUE(tokens >= 0, "int4_cache_load: ", tokens, " tokens");
  c10::cuda::CUDAGuard guard(cache.device());
  auto k = at::empty({tokens, cache.size(1), hd}, cache.options().dtype(dtype)), v = at::empty_like(k);
  cache_rows(k, v, cache, cu, slots, start, room, hd, longest, false, "int4_cache_load");
  if (cu.size(0) == 1) {   // (no sequence: no block wrote anything)
    k.zero_();
    v.zero_();
  }
  return {k, v};
}

Tensor decode_attention_int4(const Tensor& qkv, Tensor cache, const Tensor& lens, int64_t nq, int64_t nkv, int64_t hd, int64_t room, double scale, const OptT& cos,
                             const OptT& sin, int64_t rot_dim, bool interleaved) {
  const char* op = "decode_attention_int4";
  const auto d = cache_dims(cache, room, hd, op);
  const int dt = type_of(qkv, op);
  TORCH_CHECK_VALUE(nkv == d.nkv && nkv > 0 && nq > 0 && nq % nkv == 0 && nq <= 65535, op, ": ", nq, " query heads over ", nkv, " key heads, a cache of ", d.nkv);
  TORCH_CHECK_VALUE(qkv.dim() == 2 && qkv.device() == cache.device() && qkv.size(0) == d.slots && qkv.size(1) == (nq + 2 * nkv) * hd, op,
                    ": the fused projection's output [slots, (n_q + 2 n_kv) * hd] beside the cache");
  const int* lp = whole(lens, d.slots, cache, op, "cache_lens");
  TORCH_CHECK_VALUE(cos.has_value() == sin.has_value(), op, ": cosines and sines go together");
  if (cos.has_value()) {
    TORCH_CHECK_VALUE(rot_dim > 0 && rot_dim <= hd && rot_dim % (interleaved ? 2 : 16) == 0, op, ": ", rot_dim, " rotated channels");
    for (const Tensor& t : {*cos, *sin})
      TORCH_CHECK_VALUE(t.scalar_type() == at::kFloat && t.dim() == 2 && t.is_contiguous() && t.size(0) >= room && t.size(1) == rot_dim / 2 && t.device() == cache.device(), op,
                        ": cosines and sines are contiguous float32 tables [at least ", room, ", ", rot_dim / 2, "]");
  }
  attn_check();
  c10::cuda::CUDAGuard guard(qkv.device());
  const Tensor rows = rows16(qkv);
  auto out = at::empty({qkv.size(0), nq * hd}, qkv.options());
  const int rc = rb_decode_attention_int4(rows.data_ptr(), cache.data_ptr(), lp, out.data_ptr(), cos.has_value() ? cos->data_ptr<float>() : nullptr,
                                          sin.has_value() ? sin->data_ptr<float>() : nullptr, rows.stride(0), (int)qkv.size(0), (int)nq, (int)nkv, (int)hd, (int)room,
                                          (int)rot_dim, interleaved, (float)scale, dt, at::cuda::getCurrentCUDAStream().stream());
  TORCH_CHECK(rc == 0, op, ": the kernel could not be launched (", rc, ")");
  return out;
}

int64_t weight_words(int64_t N, int64_t K, int64_t group) { return (N + 127) / 128 * 8 * ((K + 127) / 128) * (256 + 16 * (128 / group)); }

void check_weight(const Tensor& q, int64_t N, int64_t K, int64_t group, const char* op) {
  TORCH_CHECK_VALUE(group == 32 || group == 64 || group == 128, op, ": groups of 32, 64 or 128, not ", group);
  TORCH_CHECK_VALUE(N > 0 && N <= kInt - 256 && K > 0 && K <= kInt - 256 && K % group == 0, op, ": a weight [", N, ", ", K, "] in groups of ", group);
  TORCH_CHECK_VALUE(q.is_cuda() && q.scalar_type() == at::kInt && q.is_contiguous() && q.numel() == weight_words(N, K, group) && on16(q), op,
                    ": the packed weight is a contiguous int32 tensor of ", weight_words(N, K, group), " words on a CUDA device");
}

void int4_quantize(const Tensor& w, Tensor q, int64_t group) {
  const char* op = "int4_quantize";
  TORCH_CHECK_VALUE(w.dim() == 2 && w.device() == q.device(), op, ": a weight [N, K] beside its packed form");
  const int dt = type_of(w, op);
  check_weight(q, w.size(0), w.size(1), group, op);
  c10::cuda::CUDAGuard guard(w.device());
  const Tensor rows = rows16(w);
  const int rc = rb_int4_quantize(rows.data_ptr(), q.data_ptr(), (int)w.size(0), (int)w.size(1), rows.stride(0), (int)group, dt, at::cuda::getCurrentCUDAStream().stream());
  TORCH_CHECK(rc == 0, op, ": the kernel could not be launched (", rc, ")");
}

void int4_pack(const Tensor& codes, const Tensor& scale, const Tensor& low, Tensor q, int64_t group) {
  const char* op = "int4_pack";
  TORCH_CHECK_VALUE(codes.dim() == 2 && codes.scalar_type() == at::kByte && codes.device() == q.device(), op, ": codes uint8 [N, K] beside the packed form");
  check_weight(q, codes.size(0), codes.size(1), group, op);
  type_of(scale, op);
  for (const Tensor& t : {scale, low})
    TORCH_CHECK_VALUE(t.scalar_type() == scale.scalar_type() && t.dim() == 2 && t.size(0) == codes.size(0) && t.size(1) == codes.size(1) / group && t.device() == q.device(), op,
                      ": steps and lowest values [N, K / group] of one 16-bit type beside the codes");
  c10::cuda::CUDAGuard guard(q.device());
  const Tensor c = codes.is_contiguous() && (reinterpret_cast<uintptr_t>(codes.data_ptr()) & 7) == 0 ? codes : codes.clone(at::MemoryFormat::Contiguous);
  const Tensor s = scale.contiguous(), l = low.contiguous();
  const int rc = rb_int4_pack(c.data_ptr(), s.data_ptr(), l.data_ptr(), q.data_ptr(), (int)codes.size(0), (int)codes.size(1), (int)group, at::cuda::getCurrentCUDAStream().stream());
  TORCH_CHECK(rc == 0, op, ": the kernel could not be launched (", rc, ")");
}

Tensor int4_linear(const Tensor& x, const Tensor& q, const OptT& bias, int64_t N, int64_t group) {
  const char* op = "int4_linear";
  TORCH_CHECK_VALUE(x.dim() == 2 && x.device() == q.device() && x.size(0) <= kInt - 256, op, ": rows [M, K] beside the weight");
  const int dt = type_of(x, op);
  const int64_t M = x.size(0), K = x.size(1);
  check_weight(q, N, K, group, op);
  TORCH_CHECK_VALUE(!bias.has_value() || (bias->scalar_type() == x.scalar_type() && bias->dim() == 1 && bias->size(0) == N && bias->is_contiguous() && bias->device() == x.device()),
                    op, ": a bias [", N, "] of the rows' type");
  attn_check();
  c10::cuda::CUDAGuard guard(x.device());
  // (a row repeated by a stride of 0, or rows that overlap, are copied: a tensor map does not take them)
  const Tensor rows = M > 1 && x.stride(0) < K ? x.clone(at::MemoryFormat::Contiguous) : rows16(x);
  auto y = at::empty({M, N}, x.options());
  const int rc = rb_int4_linear(rows.data_ptr(), q.data_ptr(), bias.has_value() ? bias->data_ptr() : nullptr, y.data_ptr(), (int)M, (int)N, (int)K, rows.stride(0), N, (int)group, dt,
                                at::cuda::getCurrentCUDAStream().stream());
  TORCH_CHECK(rc == 0, op, ": the kernel could not be launched (", rc, ")");
  return y;
}

}  // namespace

void register_int4_ops(torch::Library& m) {
  m.def("int4_cache_store(Tensor k, Tensor v, Tensor(a!) cache, Tensor cu_seqlens, Tensor? slots, Tensor? start, int room, int hd, int longest) -> ()", &int4_cache_store);
  m.def("int4_cache_load(Tensor cache, Tensor cu_seqlens, Tensor? slots, Tensor? start, int room, int hd, int tokens, int longest, ScalarType dtype) -> Tensor[]",
        &int4_cache_load);
  m.def("decode_attention_int4(Tensor qkv, Tensor(a!) cache, Tensor cache_lens, int nq, int nkv, int hd, int room, float scale, Tensor? cos, Tensor? sin, int rot_dim, "
        "bool interleaved) -> Tensor", &decode_attention_int4);
  m.def("int4_quantize(Tensor w, Tensor(a!) q, int group) -> ()", &int4_quantize);
  m.def("int4_pack(Tensor codes, Tensor scale, Tensor low, Tensor(a!) q, int group) -> ()", &int4_pack);
  m.def("int4_linear(Tensor x, Tensor q, Tensor? bias, int n, int group) -> Tensor", &int4_linear);
}
