// The Python face of the operators of bounded caches, as a small extension module: argument checks,
// outputs and scratch memory from torch's allocator, and the launches (api.h).  A decode step's
// attention or a choice among a layer's entries is done on the GPU in 4 to 8 microseconds; the same checks and
// allocations in Python, and thirty arguments through ctypes, took 12 to 23.
//
// Every function raises the library's KernelError (given to `init`) for an argument that it does not
// take, before anything is launched.
#include <Python.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <climits>
#include <map>
#include <string>
#include <utility>

#include "api.h"

namespace {

constexpr long PAGE = 64;
constexpr long MAX_DECODE_SEQS = 1024;   // sequences of a decode step that the single-token kernels take
constexpr long SUMS_KEYS = 256;          // keys of a segment of attention_sums_tc.cu
PyObject* kernel_error = nullptr;

struct Refused {};                        // a Python exception has been set

[[noreturn]] void refuse(const std::string& what) {
  PyErr_SetString(kernel_error ? kernel_error : PyExc_RuntimeError, what.c_str());
  throw Refused();
}
void launched(const char* name, int rc) {
  if (rc == 0) return;
  const char* what = rc == 1001 ? "bad argument" : rc == 1002 ? "unsupported size"
                     : rc == 1003 ? "size beyond the stated maximum" : nullptr;
  refuse(std::string(name) + ": " + (what ? std::string(what) : "CUDA error " + std::to_string(rc)));
}

int as_int(long v, const char* name) {
  if (v < 0 || v > 0x7fffffff) refuse(std::string(name) + " is out of range");
  return (int)v;
}

struct Args {
  PyObject* const* a;
  const at::Tensor& tensor(int i, const char* name) const {
    if (!THPVariable_Check(a[i])) refuse(std::string(name) + " must be a tensor");
    return THPVariable_Unpack(a[i]);
  }
  bool none(int i) const { return a[i] == Py_None; }
  // (a number that is none raises the library's error like any other argument that is not taken)
  long number(int i, const char* name) const {
    const long v = PyLong_AsLong(a[i]);
    if (v == -1 && PyErr_Occurred()) not_taken(name, "a whole number");
    return v;
  }
  double real(int i, const char* name) const {
    const double v = PyFloat_AsDouble(a[i]);
    if (v == -1.0 && PyErr_Occurred()) not_taken(name, "a number");
    return v;
  }
  int integer(int i, const char* name, long most = LONG_MAX) const {
    return as_int(std::min(number(i, name), most), name);
  }

 private:
  [[noreturn]] static void not_taken(const char* name, const char* what) {
    if (!PyErr_ExceptionMatches(PyExc_TypeError) && !PyErr_ExceptionMatches(PyExc_OverflowError)) throw Refused();
    PyErr_Clear();
    refuse(std::string(name) + " must be " + what);
  }
};

bool is(const at::Tensor& t, at::ScalarType type, long numel, int device) {
  return t.scalar_type() == type && t.numel() == numel && t.is_cuda() && t.get_device() == device && t.is_contiguous();
}
void need_ints(const at::Tensor& t, const char* name, long n, int device) {
  if (!is(t, at::kInt, n, device))
    refuse(std::string(name) + " must be contiguous int32 of " + std::to_string(n) + " elements on cuda:" + std::to_string(device));
}
int current_device_of(const at::Tensor& t, const char* name) {
  if (!t.is_cuda()) refuse(std::string(name) + " must be on a CUDA device");
  const int device = t.get_device(), current = c10::cuda::current_device();
  if (device != current)
    refuse("the tensors lie on cuda:" + std::to_string(device) + ", but the current device is cuda:" + std::to_string(current));
  return device;
}
uintptr_t address(const at::Tensor& t) { return (uintptr_t)t.data_ptr(); }

at::Tensor empty(c10::IntArrayRef size, at::ScalarType type, int device) {
  return at::detail::empty_cuda(size, type, c10::Device(c10::kCUDA, (c10::DeviceIndex)device), std::nullopt);
}

// Tickets (int32, zero between launches) for a call on this stream.  They are kept for each stream,
// whose calls run one after another.  A captured call gets some of its own for good, so that graphs
// may be replayed side by side: from an arena that is zeroed once, at the device's first call outside a
// capture; without one (or when it is used up) they are zeroed by the graph itself, a node
// that costs each replay about 3 us.
at::Tensor tickets_of(long n, int device, cudaStream_t stream) {
  constexpr long ARENA = 1 << 20;
  struct Arena {
    at::Tensor memory;
    long used = 0;
  };
  static auto* kept = new std::map<std::pair<int, cudaStream_t>, at::Tensor>();      // (these outlive the interpreter)
  static auto* arenas = new std::map<int, Arena>();
  auto zeroed = [&](long count) {
    at::Tensor t = empty({count}, at::kInt, device);
    if (cudaMemsetAsync(t.data_ptr(), 0, (size_t)count * 4, stream) != cudaSuccess) refuse("tickets cannot be zeroed");
    return t;
  };
  cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
  if (cudaStreamIsCapturing(stream, &capture) != cudaSuccess) refuse("the stream's state cannot be read");
  Arena& arena = (*arenas)[device];
  if (capture != cudaStreamCaptureStatusNone) {
    const long wanted = (n + 31) / 32 * 32;
    if (!arena.memory.defined() || arena.used + wanted > ARENA) return zeroed(n);
    at::Tensor t = arena.memory.narrow(0, arena.used, n);
    arena.used += wanted;
    return t;
  }
  if (!arena.memory.defined()) {
    arena.memory = zeroed(ARENA);
    // (a graph that is captured later may be replayed on a stream that knows nothing of this one)
    if (cudaStreamSynchronize(stream) != cudaSuccess) refuse("the tickets' arena cannot be set up");
  }
  at::Tensor& t = (*kept)[{device, stream}];
  if (!t.defined() || t.numel() < n) t = zeroed(std::max(n, 4096L));
  return t;
}

// attention(q, n_heads, n_kv_heads, head_dim, k_pages, v_pages, page_table, cu_seqlens, ctx_lens,
//           seq_of_token, positions, scale, window, max_new_tokens, max_ctx_len, mma_only, sinks,
//           weight_sums, stored_positions, token_positions, cluster, groups, n_ctas, n_sms, status)
// window 0: none.  weight_sums None: a window and sinks, else no window.  cluster, groups, n_ctas: the
// plan of a step in which every sequence brings one token.
at::Tensor attention(const Args& a) {
  const at::Tensor &q = a.tensor(0, "q"), &k = a.tensor(4, "k_pages"), &v = a.tensor(5, "v_pages"),
                   &table = a.tensor(6, "page_table"), &cu = a.tensor(7, "cu_seqlens"), &ctx = a.tensor(8, "ctx_lens"),
                   &seq = a.tensor(9, "seq_of_token"), &pos = a.tensor(10, "positions");
  const int nh = a.integer(1, "n_heads"), nkv = a.integer(2, "n_kv_heads"), hd = a.integer(3, "head_dim");
  const float scale = (float)a.real(11, "scale");
  const int window = a.integer(12, "window", 1L << 30);
  const int max_new = a.integer(13, "max_new_tokens"), max_ctx = a.integer(14, "max_ctx_len");
  const bool mma_only = a.number(15, "mma_only") != 0, sums = !a.none(17);
  const int sinks = a.integer(16, "sinks", 1L << 30);
  // (masked scores are -inf ahead of the scale in some kernels)
  if (!(scale > 0.f) || scale > 1e30f) refuse("scale must be positive and finite");
  const int device = current_device_of(q, "q");
  const at::ScalarType type = q.scalar_type();
  if (type != at::kBFloat16 && type != at::kFloat) refuse("unsupported element type");
  if (q.dim() != 2 || q.stride(1) != 1 || nkv < 1 || nh % nkv || nh < 1 || hd < 1 || q.size(1) < (long)nh * hd)
    refuse("q must be a matrix with unit column stride, at least n_heads * head_dim wide, and n_heads a multiple of n_kv_heads");
  if (k.dim() != 4 || k.size(1) != nkv || k.size(2) != PAGE || k.size(3) != hd || !is(k, type, k.numel(), device) ||
      v.sizes() != k.sizes() || !is(v, type, k.numel(), device) || ((address(k) | address(v)) & 15))
    refuse("pages must be contiguous [n_pages, n_kv_heads, PAGE, head_dim] of q's type, on its device, "
           "and begin at a multiple of 16 bytes");
  const int T = as_int(q.size(0), "the number of tokens"), B = as_int(ctx.numel(), "the number of sequences");
  const int n_pages = as_int(k.size(0), "n_pages");
  const int q_stride = T == 1 ? nh * hd : as_int(q.stride(0), "q's row stride");     // (a single row's stride may be anything)
  if (table.dim() != 2 || table.size(0) != B) refuse("page_table must have a row for every sequence");
  need_ints(table, "page_table", table.numel(), device);
  need_ints(cu, "cu_seqlens", B + 1L, device);
  need_ints(ctx, "ctx_lens", B, device);
  need_ints(seq, "seq_of_token", T, device);
  need_ints(pos, "positions", T, device);
  if (max_new < 1 || max_ctx < 1) refuse("max_ctx_len and max_new_tokens must be at least 1");
  const int width = as_int(table.size(1), "page_table's width");
  if ((max_ctx + PAGE - 1) / PAGE > width || n_pages < 1) refuse("page_table must have an entry for every block of max_ctx_len positions");
  float* weight_sums = nullptr;
  int *stored = nullptr, *told = nullptr;
  if (sums) {
    const at::Tensor &ws = a.tensor(17, "weight_sums"), &sp = a.tensor(18, "stored_positions"), &tp = a.tensor(19, "token_positions");
    const long n = (long)n_pages * nkv * PAGE;
    const bool shaped = ws.dim() == 3 && ws.size(0) == n_pages && ws.size(1) == nkv;
    if (!shaped || !is(ws, at::kFloat, n, device)) refuse("weight_sums must be contiguous float32 [n_pages, n_kv_heads, PAGE]");
    if (sp.sizes() != ws.sizes() || !is(sp, at::kInt, n, device))
      refuse("stored_positions must be contiguous int32 [n_pages, n_kv_heads, PAGE]");
    if (!is(tp, at::kInt, T, device)) refuse("token_positions must be contiguous int32 [T]");
    weight_sums = ws.data_ptr<float>();
    stored = sp.data_ptr<int>();
    told = tp.data_ptr<int>();
  }
  at::Tensor out = empty({T, (long)nh * hd}, type, device);
  if (T == 0) return out;
  if (B < 1) refuse("q has tokens, but there are no sequences");
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(device).stream();
  const int n_sms = a.integer(23, "n_sms");
  int* const status = (int*)a.tensor(24, "status").data_ptr();
  const int out_stride = nh * hd;
  const int *table_p = table.data_ptr<int>(), *cu_p = cu.data_ptr<int>(), *ctx_p = ctx.data_ptr<int>();
  const bool fast = type == at::kBFloat16 && wpc_attention_mma_supports(nh, nkv, hd) && q_stride % 2 == 0 && address(q) % 4 == 0;

  if (fast && max_new == 1 && B <= MAX_DECODE_SEQS) {
    // every sequence brings one token; with sums the scores stay in scratch memory until the rows'
    // maxima and sums are known
    if (T != B) refuse("one token per sequence expected");
    const int cluster = a.integer(20, "cluster"), groups = a.integer(21, "groups"), n_ctas = a.integer(22, "n_ctas");
    const long pairs = (long)B * nkv;
    at::Tensor part, tickets, scores;
    float *part_o = nullptr, *part_ml = nullptr;
    int* counters = nullptr;
    if (!cluster || groups > 1) {
      const long n_o = cluster ? pairs * groups * (nh / nkv) * hd : (n_ctas + pairs) * 16 * hd;
      const long n_ml = cluster ? pairs * groups * 32 : (n_ctas + pairs) * 32;
      part = empty({n_o + n_ml}, at::kFloat, device);
      part_o = part.data_ptr<float>();
      part_ml = part_o + n_o;
      tickets = tickets_of(pairs, device, stream);
      counters = tickets.data_ptr<int>();
    }
    const long score_stride = (max_ctx + PAGE - 1) / PAGE * PAGE;
    float *score_p = nullptr, *row_ml = nullptr;
    if (sums) {
      scores = empty({(long)B * nh * (score_stride + 2)}, at::kFloat, device);
      score_p = scores.data_ptr<float>();
      row_ml = score_p + (long)B * nh * score_stride;
    }
    launched("attention_decode_bounded", wpc_attention_decode_bounded(
        q.data_ptr(), q_stride, out.data_ptr(), out_stride, k.data_ptr(), v.data_ptr(), table_p, width, ctx_p, B, nh, nkv, hd,
        scale, window, sinks, n_ctas, cluster, groups, part_o, part_ml, counters, (int)pairs, score_p, (int)score_stride,
        row_ml, told, max_ctx, n_pages, weight_sums, stored, status, stream));
    return out;
  }
  const int longest = std::min(max_new, T);              // (a larger bound would only start blocks without work)
  at::Tensor lse;
  float* lse_p = nullptr;
  if (sums) {
    lse = empty({T, nh}, at::kFloat, device);
    lse_p = lse.data_ptr<float>();
  }
  const bool aligned = fast && q_stride % 8 == 0 && address(q) % 16 == 0;      // q rows can be copied 16 bytes at a time
  // (rows that overlap, an expanded one for instance, cannot be described to the copy engine)
  const bool on_tc = aligned && !mma_only && q_stride >= nh * hd && wpc_attention_prefill_tc_supports(nh, nkv, hd);
  if (!fast) {
    const int keys = window ? (int)std::min<long>(max_ctx, (long)window + sinks) : max_ctx;
    // Blocks that share a query's keys: about 64 keys each, at most 16, and no more blocks than eight to an SM.
    // Four sequences of up to 1,000 positions, window 257, 14 heads of 64: 1 block 15.4 us, 4 (the rule) 9.5,
    // 12 11.2; one sequence, window 2,048: 1 block 92.5, 16 (the rule) 16.5, 32 18.2.
    const long rows = std::max<long>((long)T * nh, 1);
    // Without a window the split is that of the ordinary attention, so that keeping sums changes no bit of it.
    const int splits = (int)std::max<long>(1, window ? std::min<long>(std::min(keys / 64, 16), 8L * n_sms / rows)
                                                     : std::min<long>(keys / 256, 2L * n_sms / rows));
    at::Tensor part;
    if (splits > 1) part = empty({(long)T * nh * splits * (hd + 2)}, at::kFloat, device);
    launched("attention_plain", wpc_attention_plain_bounded(
        q.data_ptr(), q_stride, out.data_ptr(), out_stride, type == at::kFloat ? 0 : 1, k.data_ptr(), v.data_ptr(), table_p,
        width, seq.data_ptr<int>(), pos.data_ptr<int>(), T, nh, nkv, hd, scale, window, sinks, splits,
        splits > 1 ? part.data_ptr<float>() : nullptr, lse_p, n_pages, stream));
  } else if (on_tc) {
    // A chunk of few tokens over a long cache has fewer row tiles than the SMs have places (two each): then as
    // many CTAs as there are places for share a tile's pages, four pages each at least.  7B shape:
    // 64 tokens of 2,048 positions, window 1,024: alone 23.0 us, 4 pages each 14.4, 8 pages 18.0; of 8,192, window
    // 4,096: 64.0, 23.0, 19.1 (two tokens: 68.8, 16.5, 18.0); 512 tokens (two CTAs to a tile) 63.8 -> 48.1, and with
    // the shorter window 24.2 -> 24.6.
    const long tiles = ((long)longest * (nh / nkv) + 127) / 128 * nkv * B;
    const long seen = window ? std::min<long>(max_ctx, (long)window + longest + sinks + PAGE) : max_ctx;
    const int splits = (int)std::max<long>(1, std::min<long>(std::min<long>(16, 2L * n_sms / tiles), seen / PAGE / 4));
    at::Tensor part;
    if (splits > 1) part = empty({splits * tiles * 128 * (hd + 2)}, at::kFloat, device);
    launched("attention_prefill_tc_bounded", wpc_attention_prefill_tc_bounded(
        q.data_ptr(), q_stride, out.data_ptr(), out_stride, k.data_ptr(), v.data_ptr(), table_p, width, cu_p, ctx_p, B, longest,
        nh, nkv, hd, scale, window, sinks, lse_p, status, n_pages, splits, splits > 1 ? part.data_ptr<float>() : nullptr, stream));
  } else {
    launched("attention_prefill_bounded", wpc_attention_prefill_bounded(
        q.data_ptr(), q_stride, out.data_ptr(), out_stride, k.data_ptr(), v.data_ptr(), table_p, width, cu_p, ctx_p, B, longest,
        nh, nkv, hd, scale, window, sinks, lse_p, n_pages, stream));
  }
  if (!sums) return out;
  if (on_tc) {
    at::Tensor part = empty({2L * n_sms * SUMS_KEYS}, at::kFloat, device);
    const long n_tickets = (long)B * nkv * ((max_ctx + SUMS_KEYS - 1) / SUMS_KEYS);
    at::Tensor tickets = tickets_of(n_tickets, device, stream);
    launched("weight_sums_tc", wpc_weight_sums_tc(
        q.data_ptr(), q_stride, T, k.data_ptr(), table_p, width, cu_p, ctx_p, told, lse_p, B, nh, nkv, hd, scale, longest,
        max_ctx, n_pages, weight_sums, stored, status, part.data_ptr<float>(), tickets.data_ptr<int>(), (int)tickets.numel(),
        stream));
  } else if (aligned) {
    launched("weight_sums_mma", wpc_weight_sums_mma(
        q.data_ptr(), q_stride, k.data_ptr(), table_p, width, cu_p, ctx_p, told, lse_p, B, nh, nkv, hd, scale, longest, max_ctx,
        n_pages, weight_sums, stored, status, stream));
  } else {
    launched("weight_sums_plain", wpc_weight_sums_plain(
        q.data_ptr(), q_stride, type == at::kFloat ? 0 : 1, k.data_ptr(), table_p, width, cu_p, ctx_p, told, lse_p, B, nh, nkv,
        hd, scale, longest, max_ctx, n_pages, weight_sums, stored, status, stream));
  }
  return out;
}

// The two records of one layer or of several, and a page table.
struct Record {
  int device, layers, n_pages, nkv, B, width;
  float* sums;
  int *stored, *table;
  Record(const at::Tensor& ws, const at::Tensor& sp, const at::Tensor& pt) {
    device = current_device_of(ws, "weight_sums");
    const long d = ws.dim();
    if ((d != 3 && d != 4) || ws.size(d - 1) != PAGE || !is(ws, at::kFloat, ws.numel(), device))
      refuse("weight_sums must be contiguous float32 [layers, n_pages, n_kv_heads, PAGE] (or of one layer)");
    if (sp.sizes() != ws.sizes() || !is(sp, at::kInt, ws.numel(), device))
      refuse("stored_positions must be contiguous int32 of weight_sums' shape");
    if (pt.dim() != 2 || !is(pt, at::kInt, pt.numel(), device)) refuse("page_table must be contiguous int32 [B, width]");
    layers = d == 3 ? 1 : as_int(ws.size(0), "the number of layers");
    n_pages = as_int(ws.size(d - 3), "n_pages");
    nkv = as_int(ws.size(d - 2), "n_kv_heads");
    B = as_int(pt.size(0), "the number of sequences");
    width = as_int(pt.size(1), "page_table's width");
    sums = ws.data_ptr<float>();
    stored = sp.data_ptr<int>();
    table = pt.data_ptr<int>();
  }
};

// select_kept(weight_sums, stored_positions, page_table, stored_lens, next_positions, keep, sinks, recent, status)
at::Tensor select_kept(const Args& a) {
  const int keep = a.integer(5, "keep"), sinks = a.integer(6, "sinks"), recent = a.integer(7, "recent");
  const at::Tensor &ws = a.tensor(0, "weight_sums"), &lens = a.tensor(3, "stored_lens"), &next = a.tensor(4, "next_positions");
  const Record r(ws, a.tensor(1, "stored_positions"), a.tensor(2, "page_table"));
  if (!is(lens, at::kInt, r.B, r.device)) refuse("stored_lens must be contiguous int32 [B]");
  if (!is(next, at::kInt, r.B, r.device)) refuse("next_positions must be contiguous int32 [B]");
  at::Tensor kept = ws.dim() == 3 ? empty({r.B, r.nkv, keep}, at::kInt, r.device)
                                  : empty({r.layers, r.B, r.nkv, keep}, at::kInt, r.device);
  if (!kept.numel()) return kept;
  at::Tensor scratch;
  if (const long places = wpc_select_kept_scratch(keep, r.width))
    scratch = empty({(long)r.layers * r.B * r.nkv * places}, at::kInt, r.device);
  launched("select_kept", wpc_select_kept(r.sums, r.stored, r.table, r.width, lens.data_ptr<int>(), next.data_ptr<int>(),
                                          r.layers, r.B, r.nkv, r.n_pages, keep, sinks, recent, kept.data_ptr<int>(),
                                          scratch.defined() ? scratch.data_ptr<int>() : nullptr,
                                          (int*)a.tensor(8, "status").data_ptr(),
                                          c10::cuda::getCurrentCUDAStream(r.device).stream()));
  return kept;
}

// move_kept(k_pages, v_pages, weight_sums, stored_positions, page_table, kept, status)
void move_kept(const Args& a) {
  const at::Tensor &k = a.tensor(0, "k_pages"), &v = a.tensor(1, "v_pages"), &ws = a.tensor(2, "weight_sums"),
                   &kept = a.tensor(5, "kept");
  const Record r(ws, a.tensor(3, "stored_positions"), a.tensor(4, "page_table"));
  const long d = ws.dim();
  for (const at::Tensor* t : {&k, &v}) {
    const auto type = t->scalar_type();
    if (t->dim() != d + 1 || t->sizes().slice(0, d) != ws.sizes() || (type != at::kFloat && type != at::kBFloat16) ||
        !is(*t, type, t->numel(), r.device))
      refuse(std::string(t == &k ? "k_pages" : "v_pages") + " must be contiguous [.., n_pages, n_kv_heads, PAGE, head_dim] like weight_sums");
  }
  if (kept.dim() != d || (d == 4 && kept.size(0) != r.layers) || kept.size(d - 3) != r.B || kept.size(d - 2) != r.nkv ||
      !is(kept, at::kInt, kept.numel(), r.device))
    refuse("kept must be contiguous int32 [.., B, n_kv_heads, keep]");
  if (kept.numel())
    launched("move_kept", wpc_move_kept(k.data_ptr(), v.data_ptr(), as_int(k.size(d) * k.element_size(), "an entry's key"),
                                        as_int(v.size(d) * v.element_size(), "an entry's value"), r.sums, r.stored, r.table,
                                        r.width, kept.data_ptr<int>(), r.layers, r.B, r.nkv, r.n_pages,
                                        as_int(kept.size(d - 1), "keep"), (int*)a.tensor(6, "status").data_ptr(),
                                        c10::cuda::getCurrentCUDAStream(r.device).stream()));
}

template <typename F>
PyObject* guarded(PyObject* const* args, Py_ssize_t n, Py_ssize_t want, F&& f) {
  HANDLE_TH_ERRORS
  if (n != want) {
    PyErr_Format(PyExc_TypeError, "%zd arguments expected, got %zd", want, n);
    return nullptr;
  }
  try {
    return f(Args{args});
  } catch (const Refused&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}
PyObject* py_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(args, n, 25, [](const Args& a) { return THPVariable_Wrap(attention(a)); });
}
PyObject* py_select_kept(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(args, n, 9, [](const Args& a) { return THPVariable_Wrap(select_kept(a)); });
}
PyObject* py_move_kept(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(args, n, 7, [](const Args& a) {
    move_kept(a);
    return Py_NewRef(Py_None);
  });
}
PyObject* py_init(PyObject*, PyObject* error) {
  Py_XDECREF(kernel_error);
  kernel_error = Py_NewRef(error);
  return Py_NewRef(Py_None);
}

PyMethodDef methods[] = {
    {"attention", (PyCFunction)(void (*)(void))py_attention, METH_FASTCALL, nullptr},
    {"select_kept", (PyCFunction)(void (*)(void))py_select_kept, METH_FASTCALL, nullptr},
    {"move_kept", (PyCFunction)(void (*)(void))py_move_kept, METH_FASTCALL, nullptr},
    {"init", py_init, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "wpc_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_wpc_host(void) { return PyModule_Create(&module); }
