// The checks and calls of paged.py's entry points, on ATen tensors.
//
// A decoding step over a paged cache takes a few microseconds of GPU time, less than the
// same checks take in Python (about 20 us a call; 5 here), so they are compiled.  This
// file holds no computation: it checks the arguments, allocates what is returned, keeps the
// workspaces and calls the C entry points of include/reworld_b200.h on the current stream.
//
// Workspaces are kept for each stream, since calls on different streams may
// overlap; a call that is captured into a graph gets its own, of the graph's memory, so
// graphs share nothing.  The interpreter lock is held throughout, so that two host threads
// that use one stream cannot put their launches between each other's.
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/utils/pybind.h>

#include <cmath>
#include <map>
#include <optional>
#include <string>
#include <utility>

#include "../../include/reworld_b200.h"

namespace py = pybind11;
using at::Tensor;
using std::optional;

namespace {

#define CHECK_VALUE(cond, ...) TORCH_CHECK_VALUE(cond, __VA_ARGS__)

void check_code(int code, const char* what) {
  if (code == RW_OK) return;
  throw std::runtime_error(std::string(what) + " failed: " + rw_error_string(code) + " (code " + std::to_string(code) +
                           ")");
}

int dtype_code(at::ScalarType t) { return t == at::kBFloat16 ? RW_DTYPE_BF16 : (t == at::kHalf ? RW_DTYPE_FP16 : -1); }

// A new tensor beside `like` (at::empty's dispatch costs as much again as the allocation: 0.4 us a tensor).
Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) {
  return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);
}

struct Heads {
  void* ptr;
  int64_t sl, sh;
};

bool heads_ok(const Tensor& t) {
  if (t.stride(2) != 1 || reinterpret_cast<uintptr_t>(t.data_ptr()) % 16) return false;
  for (int d = 0; d < 2; ++d)
    if (t.size(d) > 1 && (t.stride(d) <= 0 || t.stride(d) % 8)) return false;
  return true;
}

void check_kind(const Tensor& t, const char* name, const Tensor& like) {
  CHECK_VALUE(t.dim() == 3 && t.scalar_type() == like.scalar_type() && t.device() == like.device(), name, " must be a ",
              like.scalar_type(), " [T, heads, D] tensor on ", like.device());
}

// Strides of a dimension of one are never used, but have to be valid.
Heads heads_of(const Tensor& t) {
  return {t.data_ptr(), t.size(0) > 1 ? t.stride(0) : 8, t.size(1) > 1 ? t.stride(1) : 8};
}

// A packed [T, heads, D] input; one that the kernels cannot read as it is gets copied to `copy`.
Heads input(const Tensor& t, const char* name, const Tensor& like, Tensor& copy) {
  check_kind(t, name, like);
  if (heads_ok(t)) return heads_of(t);
  copy = t.clone(at::MemoryFormat::Contiguous);
  CHECK_VALUE(heads_ok(copy), name, ": channels must be a multiple of 8");
  return heads_of(copy);
}

// Whether two packed tensors may share bytes (heads [i, j) and [k, l) of the same packed rows do not).
bool meet(const Tensor& a, const Tensor& b) {
  if (a.numel() == 0 || b.numel() == 0) return false;
  const int64_t es = a.element_size();
  auto span = [&](const Tensor& t, int from) {
    int64_t n = 1;
    for (int d = from; d < 3; ++d) n += (t.size(d) - 1) * t.stride(d);
    return n * es;
  };
  const auto pa = reinterpret_cast<uintptr_t>(a.data_ptr()), pb = reinterpret_cast<uintptr_t>(b.data_ptr());
  if (pa + span(a, 0) <= pb || pb + span(b, 0) <= pa) return false;
  if (a.size(0) == b.size(0) && a.size(0) > 1 && a.stride(0) == b.stride(0)) {
    const int64_t row = a.stride(0) * es, d = pa < pb ? pb - pa : pa - pb;
    const int64_t lo = span(pa < pb ? a : b, 1), hi = span(pa < pb ? b : a, 1);
    return !(lo <= d && d + hi <= row);
  }
  return true;
}

// Whether an output may lie among a pool's pages: between its first and its last byte.
bool among(const Tensor& out, const Tensor& pool) {
  if (out.numel() == 0) return false;
  auto span = [](const Tensor& t) {
    int64_t n = 1;
    for (int64_t d = 0; d < t.dim(); ++d) n += (t.size(d) - 1) * t.stride(d);
    return n * t.element_size();
  };
  const auto a = reinterpret_cast<uintptr_t>(out.data_ptr()), b = reinterpret_cast<uintptr_t>(pool.data_ptr());
  return a < b + span(pool) && b < a + span(out);
}

// An output of the caller's: the input itself, or apart from it.
Heads output(const Tensor& t, const char* name, const Tensor& like, at::IntArrayRef shape, const Tensor& given) {
  check_kind(t, name, like);
  CHECK_VALUE(t.sizes() == shape, name, " must have the shape ", shape);
  CHECK_VALUE(heads_ok(t), name, ": channels must be contiguous, 16-byte aligned, other strides multiples of 8");
  const bool same = t.data_ptr() == given.data_ptr() && t.sizes() == given.sizes() && t.strides() == given.strides();
  CHECK_VALUE(same || !meet(t, given), name, " overlaps its input without being it");
  return heads_of(t);
}

const int* ints(const Tensor& t, const char* name, int64_t n, const Tensor& like) {
  CHECK_VALUE(t.scalar_type() == at::kInt && t.device() == like.device() && t.dim() == 1 && t.size(0) == n &&
                  (n < 2 || t.stride(0) == 1),
              name, " must be a contiguous int32 [", n, "] tensor on ", like.device());
  return t.data_ptr<int>();
}

struct Table {
  int64_t B, width, stride;
  const int* ptr;
};

Table table_of(const Tensor& t, const char* name, const Tensor& like) {
  CHECK_VALUE(t.scalar_type() == at::kInt && t.device() == like.device() && t.dim() == 2, name,
              " must be an int32 [B, pages] tensor on ", like.device());
  const int64_t B = t.size(0), w = t.size(1), s = t.stride(0);
  CHECK_VALUE((w < 2 || t.stride(1) == 1) && (B < 2 || s >= w), name,
              ": a sequence's pages must be contiguous, and rows apart");
  return {B, w, B > 1 && s > w ? s : w, t.data_ptr<int>()};
}

rw_paged_t cache_of(const Tensor& k, const Tensor& v, const Tensor& block_table, const Tensor& kv_lens,
                    const Tensor* q_starts) {
  CHECK_VALUE(k.is_cuda(), "a paged cache lives on a CUDA device, not on ", k.device());
  const int code = dtype_code(k.scalar_type());
  CHECK_VALUE(code >= 0, "a paged cache is bf16 or fp16");
  CHECK_VALUE(k.dim() == 4 && v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type() && v.device() == k.device(),
              "k_pages and v_pages must be alike, [num_pages, page_size, Hkv, D]");
  const int64_t n = k.size(0), page = k.size(1), hkv = k.size(2), D = k.size(3);
  TORCH_CHECK_NOT_IMPLEMENTED(D == 64 || D == 128, "head_dim ", D, ": the paged kernels have 64 and 128");
  TORCH_CHECK_NOT_IMPLEMENTED(page >= 8 && page <= (1 << 20) && (page & (page - 1)) == 0, "page_size ", page,
                              ": must be a power of two >= 8");
  CHECK_VALUE(n > 0 && hkv > 0 && n <= INT32_MAX && hkv <= 65535, "the pools have no pages or heads, or too many");
  for (const Tensor* t : {&k, &v}) {
    bool ok = t->stride(3) == 1 && reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0;
    for (int d = 0; d < 3; ++d) ok = ok && t->stride(d) > 0 && t->stride(d) % 8 == 0;
    CHECK_VALUE(ok, "k_pages, v_pages: channels must be contiguous, 16-byte aligned, other strides multiples of 8");
  }
  const Table bt = table_of(block_table, "block_table", k);
  CHECK_VALUE(bt.B <= 65535 && bt.width * page <= (1ll << 30), "block_table: more than 65535 sequences or 2^30 rows");
  rw_paged_t c{};
  c.k = k.data_ptr();
  c.v = v.data_ptr();
  c.k_sp = k.stride(0); c.k_sl = k.stride(1); c.k_sh = k.stride(2);
  c.v_sp = v.stride(0); c.v_sl = v.stride(1); c.v_sh = v.stride(2);
  c.num_pages = (int)n; c.page_size = (int)page; c.Hkv = (int)hkv; c.D = (int)D; c.dtype = code;
  c.B = (int)bt.B; c.table_width = (int)bt.width;
  c.table_stride = bt.stride;
  // (empty tensors have no address; the library wants one although it reads nothing there)
  const int* some = static_cast<const int*>(c.k);
  c.block_table = bt.ptr ? bt.ptr : some;
  c.kv_lens = ints(kv_lens, "kv_lens", bt.B, k);
  if (!c.kv_lens) c.kv_lens = some;
  c.q_starts = q_starts ? ints(*q_starts, "q_starts", bt.B + 1, k) : nullptr;
  return c;
}

struct RotaryTable {
  const float* ptr = nullptr;
  int max_pos = 0, rot = 0;
};

RotaryTable rotary_of(const Tensor& t, int64_t D, const Tensor& like) {
  CHECK_VALUE(t.scalar_type() == at::kFloat && t.dim() == 3 && t.size(2) == 2 && t.is_contiguous() &&
                  t.device() == like.device() && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0,
              "table must be a contiguous fp32 [max_pos, rotary_dim / 2, 2] tensor on ", like.device());
  const int64_t rot = 2 * t.size(1);
  CHECK_VALUE(rot >= 16 && rot % 16 == 0 && rot <= D && t.size(0) > 0 && t.size(0) <= INT32_MAX, "rotary_dim ", rot,
              ": a multiple of 16 up to the head dim (", D, ") is needed");
  return {t.data_ptr<float>(), (int)t.size(0), (int)rot};
}

int count(int64_t n, const char* what) {
  CHECK_VALUE(n <= INT32_MAX / 2, "too many ", what);
  return (int)n;
}

// The per-device status word (_native.status_tensor), asked for once.  The first call on a device may be a captured
// one: its word would be the graph's, so that call reports nothing.
int* status_word(int device) {
  static int* word[64] = {};
  if (device < 0 || device >= 64) return nullptr;
  if (!word[device] && c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None)
    word[device] = reinterpret_cast<int*>(
        py::module_::import("reworld_b200._native").attr("status_tensor")(device).attr("data_ptr")().cast<uintptr_t>());
  return word[device];
}

Tensor scratch_for(const Tensor& like, cudaStream_t stream, int64_t bytes) {
  // (a large one is not worth keeping: its allocation is nothing beside the call)
  if (bytes > (64 << 20) || c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None)
    return fresh({bytes}, at::kByte, like);
  // never destroyed: at exit the device may be gone before it
  static auto* kept = new std::map<std::pair<int, cudaStream_t>, Tensor>();
  Tensor& s = (*kept)[{like.device().index(), stream}];
  if (!s.defined() || s.numel() < bytes) s = fresh({bytes}, at::kByte, like);
  return s;
}

Tensor rotary(const Tensor& x, const Tensor& table, const Tensor& positions, bool interleaved,
              const optional<Tensor>& out) {
  const int code = dtype_code(x.scalar_type());
  CHECK_VALUE(x.is_cuda() && code >= 0 && x.dim() == 3, "rotary runs on bf16 or fp16 CUDA tensors [T, heads, D], not on ",
              x.scalar_type(), " ", x.sizes(), " on ", x.device());
  const int64_t T = x.size(0), H = x.size(1), D = x.size(2);
  TORCH_CHECK_NOT_IMPLEMENTED(D == 64 || D == 128, "head_dim ", D, ": the rotary kernel has 64 and 128");
  const RotaryTable tab = rotary_of(table, D, x);
  const int* pos = ints(positions, "positions", T, x);
  const c10::cuda::CUDAGuard guard(x.device());
  Tensor copy;
  const Heads in = input(x, "x", x, copy);
  const Tensor y = out ? *out : fresh({T, H, D}, x.scalar_type(), x);
  const Heads o = out ? output(y, "out", x, x.sizes(), x) : heads_of(y);
  if (T && H)
    check_code(rw_rotary(in.ptr, o.ptr, count(T, "tokens"), count(H, "heads"), (int)D, code, in.sl, in.sh, o.sl, o.sh,
                         tab.ptr, tab.max_pos, tab.rot, interleaved, pos, status_word(x.device().index()),
                         c10::cuda::getCurrentCUDAStream(x.device().index()).stream()),
               "rw_rotary");
  return y;
}

optional<Tensor> store(const Tensor& k, const Tensor& v, const Tensor& k_pages, const Tensor& v_pages,
                       const Tensor& block_table, const Tensor& q_starts, const Tensor& kv_lens,
                       const optional<Tensor>& table, const optional<Tensor>& positions, const optional<Tensor>& q,
                       const optional<Tensor>& q_out, bool interleaved) {
  const rw_paged_t c = cache_of(k_pages, v_pages, block_table, kv_lens, &q_starts);
  const c10::cuda::CUDAGuard guard(k_pages.device());
  Tensor kc, vc, qc;
  const Heads hk = input(k, "k", k_pages, kc), hv = input(v, "v", k_pages, vc);
  const int64_t T = k.size(0);
  CHECK_VALUE(k.size(1) == c.Hkv && k.size(2) == c.D && v.sizes() == k.sizes(), "k and v must be [T, ", c.Hkv, ", ",
              c.D, "], as the pools");
  CHECK_VALUE(q || !q_out, "q_out needs q");
  int64_t Hq = 0;
  Heads hq{nullptr, 0, 0}, ho{nullptr, 0, 0};
  optional<Tensor> y;
  if (q) {
    hq = input(*q, "q", k_pages, qc);
    Hq = q->size(1);
    CHECK_VALUE(q->size(0) == T && q->size(2) == c.D, "q must be [", T, ", heads, ", c.D, "]");
    if (q_out) {
      y = *q_out;
      ho = output(*y, "q_out", k_pages, q->sizes(), *q);
      CHECK_VALUE(!meet(*y, k) && !meet(*y, v), "q_out overlaps k or v");
      CHECK_VALUE(!among(*y, k_pages) && !among(*y, v_pages), "q_out lies in the pools");
    } else {
      y = fresh({T, Hq, (int64_t)c.D}, k_pages.scalar_type(), k_pages);
      ho = heads_of(*y);
    }
    if (Hq == 0) hq.ptr = ho.ptr = nullptr;
  }
  const RotaryTable tab = table ? rotary_of(*table, c.D, k_pages) : RotaryTable{};
  const int* pos = positions ? ints(*positions, "positions", T, k_pages) : nullptr;
  const int dev = k_pages.device().index();
  if (T && c.B)
    check_code(rw_paged_rotary_store(&c, hk.ptr, hv.ptr, hq.ptr, ho.ptr, count(T, "tokens"), count(Hq, "heads"), hk.sl,
                                     hk.sh, hv.sl, hv.sh, hq.sl, hq.sh, ho.sl, ho.sh, tab.ptr, tab.max_pos, tab.rot,
                                     interleaved, pos, status_word(dev),
                                     c10::cuda::getCurrentCUDAStream(dev).stream()),
               "rw_paged_rotary_store");
  return y;
}

struct Sums {
  float* ptr;
  int64_t sb, sh, cap;
};

Sums sums_of(const Tensor& w, const rw_paged_t& c, int64_t rows, const Tensor& like) {
  CHECK_VALUE(w.scalar_type() == at::kFloat && w.device() == like.device() && w.dim() == 3 && w.size(0) == c.B &&
                  w.size(1) == c.Hkv && w.size(2) >= rows && (w.size(2) < 2 || w.stride(2) == 1),
              "weight_sums must be fp32 [", c.B, ", ", c.Hkv, ", >= ", rows, "] on ", like.device());
  const int64_t n = w.size(0), h = w.size(1), cap = w.size(2), s0 = w.stride(0), s1 = w.stride(1);
  bool apart = (h < 2 || s1 >= cap) && (n < 2 || s0 >= cap);
  if (n > 1 && h > 1) apart = apart && (s0 >= (h - 1) * s1 + cap || s1 >= (n - 1) * s0 + cap);
  CHECK_VALUE(apart, "weight_sums: rows overlap");
  return {w.data_ptr<float>(), s0, s1, cap};
}

py::object attention(const Tensor& q, const Tensor& k_pages, const Tensor& v_pages, const Tensor& block_table,
                     const Tensor& q_starts, const Tensor& kv_lens, optional<int64_t> max_q_len, bool causal,
                     optional<double> softmax_scale, const optional<Tensor>& weight_sums, bool return_lse,
                     const optional<Tensor>& out) {
  const rw_paged_t c = cache_of(k_pages, v_pages, block_table, kv_lens, &q_starts);
  const c10::cuda::CUDAGuard guard(k_pages.device());
  Tensor copy;
  const Heads hq = input(q, "q", k_pages, copy);
  const int64_t T = q.size(0), Hq = q.size(1), D = q.size(2), rows = (int64_t)c.table_width * c.page_size;
  CHECK_VALUE(D == c.D && Hq > 0 && Hq % c.Hkv == 0, "q must be [T, heads, ", c.D, "] with a multiple of ", c.Hkv,
              " heads");
  TORCH_CHECK_NOT_IMPLEMENTED(Hq / c.Hkv <= 128, "more than 128 query heads share a key head");
  Tensor y;
  Heads ho;
  if (out) {
    y = *out;
    ho = output(y, "out", k_pages, q.sizes(), q);
    CHECK_VALUE(y.numel() == 0 || y.data_ptr() != q.data_ptr(), "out overlaps q");
    CHECK_VALUE(!among(y, k_pages) && !among(y, v_pages), "out lies in the pools");
  } else {
    y = fresh({T, Hq, D}, k_pages.scalar_type(), k_pages);
    ho = heads_of(y);
  }
  const double scale = softmax_scale ? *softmax_scale : 1.0 / std::sqrt((double)D);
  CHECK_VALUE(scale > 0.0 && scale < 1e30, "softmax_scale must be positive and finite");
  const int64_t longest = max_q_len ? std::min(*max_q_len, T) : T;
  CHECK_VALUE(longest >= 0, "max_q_len must not be negative");
  Sums w{nullptr, 0, 0, 0};
  if (weight_sums) w = sums_of(*weight_sums, c, rows, k_pages);
  Tensor lse;
  if (return_lse) lse = fresh({T, Hq}, at::kFloat, k_pages);
  if (T && c.B && longest) {
    const int dev = k_pages.device().index();
    cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev).stream();
    const int t = count(T, "tokens"), h = count(Hq, "heads");
    const long long need = rw_paged_attn_workspace_bytes(t, h, c.Hkv, c.D, c.B, (int)longest, rows, w.ptr != nullptr);
    const Tensor ws = scratch_for(k_pages, stream, need);
    check_code(rw_paged_attn(&c, hq.ptr, ho.ptr, return_lse ? lse.data_ptr<float>() : nullptr, t, h, (int)longest,
                             hq.sl, hq.sh, ho.sl, ho.sh, causal, (float)scale, w.ptr, w.sb, w.sh, ws.data_ptr(),
                             need, status_word(dev), stream),
               "rw_paged_attn");
  }
  if (return_lse) return py::make_tuple(y, lse);
  return py::cast(y);
}

py::tuple evict(const Tensor& k_pages, const Tensor& v_pages, const Tensor& block_table, const Tensor& kv_lens,
                const Tensor& weight_sums, int64_t keep, const Tensor& dst_table, int64_t n_sink, int64_t n_recent) {
  const rw_paged_t c = cache_of(k_pages, v_pages, block_table, kv_lens, nullptr);
  CHECK_VALUE(keep >= 1 && keep <= (1ll << 30) && n_sink >= 0 && n_recent >= 0 && n_sink + n_recent <= keep,
              "keep must be positive and hold n_sink + n_recent rows");
  const int64_t rows = std::max((int64_t)c.table_width * c.page_size, keep);
  const Sums w = sums_of(weight_sums, c, rows, k_pages);
  const Table dst = table_of(dst_table, "dst_table", k_pages);
  CHECK_VALUE(dst.B == c.B, "dst_table must be an int32 [", c.B, ", pages] tensor");
  CHECK_VALUE(dst.width * c.page_size >= keep, "dst_table holds ", dst.width * c.page_size, " rows, ", keep,
              " are kept");
  const c10::cuda::CUDAGuard guard(k_pages.device());
  const Tensor kept = fresh({c.B, c.Hkv, keep}, at::kInt, k_pages), lens = fresh({c.B}, at::kInt, k_pages),
               sums = fresh({c.B, c.Hkv, w.cap}, at::kFloat, k_pages);
  const int dev = k_pages.device().index();
  if (c.B)
    check_code(rw_paged_evict(&c, w.ptr, w.sb, w.sh, sums.data_ptr<float>(), w.cap, kept.data_ptr<int>(),
                              lens.data_ptr<int>(), (int)keep, (int)n_sink, (int)n_recent, dst.ptr, dst.stride,
                              (int)dst.width, status_word(dev), c10::cuda::getCurrentCUDAStream(dev).stream()),
               "rw_paged_evict");
  return py::make_tuple(kept, lens, sums);
}

}  // namespace

PYBIND11_MODULE(paged_bind, m) {
  m.def("abi_version", &rw_abi_version);
  m.def("rotary", &rotary);
  m.def("store", &store);
  m.def("attention", &attention);
  m.def("evict", &evict);
}
