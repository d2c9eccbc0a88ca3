// The Python boundary in native code: what stk_amd/backend/hip_kernels.py checks, allocates and launches, as one call
// per operation on torch tensors.  The checks, the errors they raise and the launches are those of the C ABI
// (include/stk_amd.h); what this saves is the host time of a launch.  Through ctypes, with the checks in Python, a call
// took 10 - 14 us on the host, more than most kernels of a small problem take on the GPU; here it takes 3 - 5 us.
//
// Everything - copies of operands, allocations, launches - happens on torch's current stream of the tensors' device.  No
// state is kept between calls but one pinned word per host thread and device (Mailbox).
#include <torch/extension.h>

#include <torch/csrc/autograd/functions/basic_ops.h>

#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>

#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "../../include/stk_amd.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

// ------------------------------------------------------------------------------------------------ errors
// (the functions run without the interpreter's lock)
[[noreturn]] void raise(PyObject* type, const std::string& text) {
  py::gil_scoped_acquire gil;
  PyErr_SetString(type, text.c_str());
  throw py::error_already_set();
}
void require(bool ok, const char* text) {
  if (!ok) raise(PyExc_AssertionError, text);
}
// The exception that the reference raises in the same situation.
void check(int status) {
  if (status == STK_OK) return;
  raise(status == STK_ERR_DIMS ? PyExc_AssertionError : status == STK_ERR_UNSUPPORTED ? PyExc_NotImplementedError : PyExc_RuntimeError,
        stk_last_error());
}
void need_gpu(const Tensor& t) {
  if (!t.is_cuda()) raise(PyExc_RuntimeError, "stk_amd: this operation runs on a ROCm GPU only; got a tensor on " + t.device().str());
}

// ------------------------------------------------------------------------------------------------ operands
int value_dtype(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kHalf: return STK_F16;
    case at::kBFloat16: return STK_BF16;
    case at::kFloat: return STK_F32;
    default:
      raise(PyExc_NotImplementedError, std::string("stk_amd: products need float16, bfloat16 or float32 values, got ") + c10::toString(t.scalar_type()));
  }
}
int index_dtype(at::ScalarType t) {
  if (t == at::kShort) return STK_I16;
  if (t == at::kInt) return STK_I32;
  raise(PyExc_NotImplementedError, std::string("stk_amd: indices must be int16 or int32, got ") + c10::toString(t));
}
// Index tensors may arrive as strided views (stk/ops/matrix_ops.py:73-75).
Tensor index(const Tensor& t) {
  index_dtype(t.scalar_type());
  return t.contiguous();
}
Tensor offsets32(const Tensor& t) {
  if (t.scalar_type() != at::kInt) raise(PyExc_NotImplementedError, std::string("stk_amd: offsets must be int32, got ") + c10::toString(t.scalar_type()));
  return t.contiguous();
}
bool aligned(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15u) == 0; }
// A 2-D operand the kernels can read in place: unit stride in one dimension, the other stride a multiple of 8
// elements, 16-byte aligned base.  Anything else is copied to row-major first.
Tensor dense_operand(const Tensor& x) {
  require(x.dim() == 2, "dense operands have two dimensions");
  const int64_t s0 = x.stride(0), s1 = x.stride(1);
  if (((s1 == 1 && s0 % 8 == 0) || (s0 == 1 && s1 % 8 == 0 && x.size(0) > 1)) && aligned(x)) return x;
  Tensor c = x.contiguous();
  if (!aligned(c) || c.stride(0) % 8) raise(PyExc_NotImplementedError, "stk_amd: dense operands need a row length divisible by 8");
  return c;
}
void matmul_dims(int64_t m, int64_t k, int64_t n, int64_t b) {
  // stk/backend/triton_kernels.py:15-19 with BLOCK_M = BLOCK_N = blocking, BLOCK_K = 32
  const auto test = [](int64_t v, int64_t by) {
    if (by == 0 || v % by)
      raise(PyExc_AssertionError, "incompatible dimensions: tensor has dim with length: " + std::to_string(v) + ", which must be divisible by " + std::to_string(by));
  };
  test(m, b);
  test(k, 32);
  test(n, b);
}
template <class T>
T* ptr(const Tensor& t) { return static_cast<T*>(const_cast<void*>(t.const_data_ptr())); }
template <class T>
T* ptr(const OptTensor& t) { return t ? ptr<T>(*t) : nullptr; }

// The stream a call launches on.
hipStream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

// ------------------------------------------------------------------------------------------------ products
// The sparse operand's arrays as the launches take them.
struct Meta {
  Tensor offsets, ci, offsets_t, cit, bot;
  int idx;
  Meta(const Tensor& offsets_, const Tensor& ci_, const Tensor& offsets_t_, const Tensor& cit_, const Tensor& bot_)
      : offsets(offsets32(offsets_)), ci(index(ci_)), offsets_t(offsets32(offsets_t_)), cit(index(cit_)), bot(offsets32(bot_)),
        idx(index_dtype(ci.scalar_type())) {}
};
#define META_ARGS const Tensor &offsets, const Tensor &column_indices, const Tensor &offsets_t, const Tensor &column_indices_t, const Tensor &block_offsets_t
#define META_PTRS(m) ptr<int32_t>(m.offsets), ptr<void>(m.ci), ptr<int32_t>(m.offsets_t), ptr<void>(m.cit), ptr<int32_t>(m.bot)

void sdd(const Tensor& lhs_, const Tensor& rhs_, const Tensor& out, const OptTensor& offsets, const Tensor& row_indices, const Tensor& column_indices,
         const OptTensor& plan, int activation, const OptTensor& multiplier, const OptTensor& block_order, const OptTensor& sums) {
  need_gpu(lhs_), need_gpu(rhs_), need_gpu(out);
  require(lhs_.dim() == 2 && rhs_.dim() == 2 && lhs_.size(1) == rhs_.size(0), "incompatible dimensions");
  const int64_t m = lhs_.size(0), k = lhs_.size(1), n = rhs_.size(1), b = out.size(-1), nnz = row_indices.numel();
  matmul_dims(m, k, n, b);
  require(out.is_contiguous(), "out must be contiguous");
  const auto like_out = [&](const OptTensor& t, const char* text) {
    if (!t) return;
    need_gpu(*t);
    require(t->sizes() == out.sizes() && t->scalar_type() == out.scalar_type() && t->is_contiguous(), text);
  };
  like_out(multiplier, "the multiplier's values must be laid out like out");
  like_out(sums, "sums must be laid out like out");
  require(!sums || sums->const_data_ptr() != out.const_data_ptr(), "sums need an array of their own");
  if (nnz == 0) return;
  const c10::DeviceGuard guard(out.device());
  const Tensor lhs = dense_operand(lhs_), rhs = dense_operand(rhs_);
  require(lhs.scalar_type() == rhs.scalar_type() && lhs.scalar_type() == out.scalar_type(), "operands and out must have one dtype");
  const Tensor ri = index(row_indices), ci = index(column_indices);
  require(ri.scalar_type() == ci.scalar_type(), "row and column indices must have one dtype");
  OptTensor order;
  if (block_order) {
    require(block_order->scalar_type() == at::kInt && block_order->numel() == nnz, "block_order must be an int32 permutation of the blocks");
    order = block_order->contiguous();
  }
  OptTensor offs;
  if (plan) offs = offsets32(*offsets);
  check(stk_sdd_fused_sums(ptr<void>(lhs), lhs.stride(0), lhs.stride(1), ptr<void>(rhs), rhs.stride(0), rhs.stride(1), m, k, n, ptr<void>(out),
                           ptr<int32_t>(offs), ptr<void>(ri), ptr<void>(ci), ptr<int32_t>(order), nnz, (int)b, value_dtype(out),
                           index_dtype(ri.scalar_type()), ptr<uint8_t>(plan), activation, ptr<void>(multiplier), ptr<void>(sums), stream_of(out)));
}

// The status of the launch: the caller owns the workspace, whose state depends on it.  (Operands that are refused raise.)
int dsd(int64_t m, int64_t k, const Tensor& data, META_ARGS, bool transpose_a, const Tensor& rhs_, const Tensor& out, const OptTensor& plan,
        const OptTensor& workspace) {
  need_gpu(data), need_gpu(rhs_), need_gpu(out);
  require(rhs_.dim() == 2 && k == rhs_.size(0), "incompatible dimensions");
  const int64_t n = rhs_.size(1), b = data.size(-1);
  matmul_dims(m, k, n, b);
  const c10::DeviceGuard guard(out.device());
  const Tensor rhs = dense_operand(rhs_);
  require(data.is_contiguous() && out.stride(1) == 1, "the sparse values must be contiguous and out row-major");
  require(data.scalar_type() == rhs.scalar_type() && data.scalar_type() == out.scalar_type(), "operands and out must have one dtype");
  const Meta s(offsets, column_indices, offsets_t, column_indices_t, block_offsets_t);
  return stk_dsd(m, k, n, ptr<void>(data), META_PTRS(s), transpose_a, ptr<void>(rhs), rhs.stride(0), rhs.stride(1), ptr<void>(out), out.stride(0),
                 data.size(0), (int)b, value_dtype(out), s.idx, ptr<uint8_t>(plan), ptr<void>(workspace), workspace ? workspace->numel() : 0,
                 stream_of(out));
}

void dds(const Tensor& lhs_, int64_t k, int64_t n, const Tensor& data, META_ARGS, bool transpose_b, const Tensor& out, const OptTensor& plan) {
  need_gpu(data), need_gpu(lhs_), need_gpu(out);
  require(lhs_.dim() == 2 && lhs_.size(1) == k, "incompatible dimensions");
  const int64_t m = lhs_.size(0), b = data.size(-1);
  matmul_dims(m, k, n, b);
  const c10::DeviceGuard guard(out.device());
  const Tensor lhs = dense_operand(lhs_);
  require(data.is_contiguous() && out.stride(1) == 1, "the sparse values must be contiguous and out row-major");
  require(data.scalar_type() == lhs.scalar_type() && data.scalar_type() == out.scalar_type(), "operands and out must have one dtype");
  const Meta s(offsets, column_indices, offsets_t, column_indices_t, block_offsets_t);
  check(stk_dds(m, k, n, ptr<void>(lhs), lhs.stride(0), lhs.stride(1), ptr<void>(data), META_PTRS(s), transpose_b, ptr<void>(out), out.stride(0),
                data.size(0), (int)b, value_dtype(out), s.idx, ptr<uint8_t>(plan), stream_of(out)));
}

void dsd_dds(int64_t m, int64_t k, const Tensor& data, META_ARGS, const Tensor& rhs_, const Tensor& out_dsd, const Tensor& lhs_, const Tensor& out_dds,
             const OptTensor& plan) {
  need_gpu(data), need_gpu(rhs_), need_gpu(lhs_), need_gpu(out_dsd), need_gpu(out_dds);
  require(rhs_.dim() == 2 && lhs_.dim() == 2 && rhs_.size(0) == k && lhs_.size(1) == m, "incompatible dimensions");
  const int64_t b = data.size(-1);
  matmul_dims(m, k, rhs_.size(1), b);
  matmul_dims(lhs_.size(0), m, k, b);
  const c10::DeviceGuard guard(data.device());
  const Tensor rhs = dense_operand(rhs_), lhs = dense_operand(lhs_);
  require(data.is_contiguous() && out_dsd.stride(1) == 1 && out_dds.stride(1) == 1, "the sparse values must be contiguous and the results row-major");
  const auto t = data.scalar_type();
  require(rhs.scalar_type() == t && lhs.scalar_type() == t && out_dsd.scalar_type() == t && out_dds.scalar_type() == t, "operands and results must have one dtype");
  const Meta s(offsets, column_indices, offsets_t, column_indices_t, block_offsets_t);
  check(stk_dsd_dds(m, k, ptr<void>(data), META_PTRS(s), rhs.size(1), ptr<void>(rhs), rhs.stride(0), rhs.stride(1), ptr<void>(out_dsd), out_dsd.stride(0),
                    lhs.size(0), ptr<void>(lhs), lhs.stride(0), lhs.stride(1), ptr<void>(out_dds), out_dds.stride(0), data.size(0), (int)b,
                    value_dtype(data), s.idx, ptr<uint8_t>(plan), stream_of(data)));
}

void dsd_dsd(int64_t m, int64_t k, const Tensor& data, META_ARGS, const Tensor& rhs_, const Tensor& out, const Tensor& rhs_t_, const Tensor& out_t,
             const OptTensor& plan) {
  need_gpu(data), need_gpu(rhs_), need_gpu(rhs_t_), need_gpu(out), need_gpu(out_t);
  require(rhs_.dim() == 2 && rhs_t_.dim() == 2 && rhs_.size(0) == k && rhs_t_.size(0) == m, "incompatible dimensions");
  const int64_t b = data.size(-1);
  matmul_dims(m, k, rhs_.size(1), b);
  matmul_dims(k, m, rhs_t_.size(1), b);
  const c10::DeviceGuard guard(data.device());
  const Tensor rhs = dense_operand(rhs_), rhs_t = dense_operand(rhs_t_);
  require(data.is_contiguous() && out.stride(1) == 1 && out_t.stride(1) == 1, "the sparse values must be contiguous and the results row-major");
  const auto t = data.scalar_type();
  require(rhs.scalar_type() == t && rhs_t.scalar_type() == t && out.scalar_type() == t && out_t.scalar_type() == t, "operands and results must have one dtype");
  const Meta s(offsets, column_indices, offsets_t, column_indices_t, block_offsets_t);
  check(stk_dsd_dsd(m, k, ptr<void>(data), META_PTRS(s), rhs.size(1), ptr<void>(rhs), rhs.stride(0), rhs.stride(1), ptr<void>(out), out.stride(0),
                    rhs_t.size(1), ptr<void>(rhs_t), rhs_t.stride(0), rhs_t.stride(1), ptr<void>(out_t), out_t.stride(0), data.size(0), (int)b,
                    value_dtype(data), s.idx, ptr<uint8_t>(plan), stream_of(data)));
}

void sdd_dsd(int64_t m, int64_t n, const Tensor& lhs_, const Tensor& rhs_sdd_, const Tensor& out_sdd, const Tensor& data, const Tensor& row_indices,
             META_ARGS, bool transpose_a, const Tensor& rhs_dsd_, const Tensor& out_dsd, const OptTensor& plan) {
  need_gpu(data), need_gpu(lhs_), need_gpu(rhs_sdd_), need_gpu(rhs_dsd_), need_gpu(out_sdd), need_gpu(out_dsd);
  const int64_t b = data.size(-1);
  require(lhs_.dim() == 2 && rhs_sdd_.dim() == 2 && rhs_dsd_.dim() == 2 && lhs_.size(0) == m && rhs_sdd_.size(1) == n && lhs_.size(1) == rhs_sdd_.size(0) &&
              rhs_dsd_.size(0) == (transpose_a ? m : n), "incompatible dimensions");
  matmul_dims(m, lhs_.size(1), n, b);
  matmul_dims(transpose_a ? n : m, rhs_dsd_.size(0), rhs_dsd_.size(1), b);
  const c10::DeviceGuard guard(data.device());
  const Tensor lhs = dense_operand(lhs_), rhs_sdd = dense_operand(rhs_sdd_), rhs_dsd = dense_operand(rhs_dsd_);
  require(data.is_contiguous() && out_sdd.is_contiguous() && out_sdd.sizes() == data.sizes() && out_dsd.stride(1) == 1,
          "the sparse values must be contiguous and the results laid out like them and row-major");
  const auto t = data.scalar_type();
  require(lhs.scalar_type() == t && rhs_sdd.scalar_type() == t && rhs_dsd.scalar_type() == t && out_sdd.scalar_type() == t && out_dsd.scalar_type() == t,
          "operands and results must have one dtype");
  const Tensor ri = index(row_indices);
  const Meta s(offsets, column_indices, offsets_t, column_indices_t, block_offsets_t);
  require(ri.scalar_type() == s.ci.scalar_type() && ri.scalar_type() == s.cit.scalar_type(), "the indices must have one dtype");
  check(stk_sdd_dsd(m, n, ptr<int32_t>(s.offsets), ptr<void>(ri), ptr<void>(s.ci), ptr<int32_t>(s.offsets_t), ptr<void>(s.cit), ptr<int32_t>(s.bot),
                    ptr<void>(lhs), lhs.stride(0), lhs.stride(1), ptr<void>(rhs_sdd), rhs_sdd.stride(0), rhs_sdd.stride(1), lhs.size(1), ptr<void>(out_sdd),
                    ptr<void>(data), transpose_a, rhs_dsd.size(1), ptr<void>(rhs_dsd), rhs_dsd.stride(0), rhs_dsd.stride(1), ptr<void>(out_dsd),
                    out_dsd.stride(0), data.size(0), (int)b, value_dtype(data), s.idx, ptr<uint8_t>(plan), stream_of(data)));
}

// ------------------------------------------------------------------------------------------------ plan, streams, workspaces
Tensor build_plan(const Tensor& offsets_, const Tensor& column_indices, const OptTensor& offsets_t_, const OptTensor& column_indices_t, int blocking) {
  need_gpu(offsets_), need_gpu(column_indices);
  const c10::DeviceGuard guard(offsets_.device());
  const Tensor offsets = offsets32(offsets_), ci = index(column_indices);
  OptTensor offsets_t, cit;
  if (offsets_t_ && column_indices_t) offsets_t = offsets32(*offsets_t_), cit = index(*column_indices_t);
  const int64_t rows = offsets.numel() - 1, cols = offsets_t ? offsets_t->numel() - 1 : 0, nnz = ci.numel();
  const int64_t bytes = (int64_t)stk_plan_bytes(rows, cols, nnz);
  Tensor plan = at::empty({bytes > 0 ? bytes : 1}, offsets.options().dtype(at::kByte));
  check(stk_build_plan(ptr<int32_t>(offsets), ptr<void>(ci), rows, ptr<int32_t>(offsets_t), ptr<void>(cit), cols, nnz, blocking,
                       index_dtype(ci.scalar_type()), ptr<uint8_t>(plan), (size_t)bytes, stream_of(offsets)));
  return plan;
}

uint64_t capture_id(int64_t stream) {
  uint64_t id = 0;
  check(stk_stream_capture_id(reinterpret_cast<stk_stream_t>(stream), &id));
  return id;
}

// What is launched on the stream `waiting` from now on starts after what has been launched on `first`.
void follow(int64_t waiting, int64_t first) {
  const auto test = [](hipError_t e) {
    if (e != hipSuccess) raise(PyExc_RuntimeError, std::string("stk_amd: ordering two streams: ") + hipGetErrorString(e));
  };
  hipEvent_t event;
  test(hipEventCreateWithFlags(&event, hipEventDisableTiming));
  hipError_t e = hipEventRecord(event, reinterpret_cast<hipStream_t>(first));
  if (e == hipSuccess) e = hipStreamWaitEvent(reinterpret_cast<hipStream_t>(waiting), event, 0);
  (void)hipEventDestroy(event);   // (released once it has been reached)
  test(e);
}

// A word of pinned host memory that a kernel writes a count into and the host polls: one per host thread and device,
// in use only until the call that took it returns.
struct Mailbox {
  volatile int32_t* word;
  explicit Mailbox(const at::Device& device) {
    static thread_local std::vector<Tensor> words;
    const size_t at = (size_t)device.index();
    if (words.size() <= at) words.resize(at + 1);
    if (!words[at].defined()) words[at] = at::empty({1}, at::TensorOptions().dtype(at::kInt).pinned_memory(true));
    word = ptr<int32_t>(words[at]);
    *word = -1;
  }
  // The count.  Polled for a while - a stream wait costs more than the kernels of a small problem - then waited for, which
  // also reports a launch that failed.
  int32_t receive(hipStream_t stream) const {
    for (int i = 0; i < 200000 && *word < 0; i++) __builtin_ia32_pause();
    if (*word < 0) {
      const hipError_t e = hipStreamSynchronize(stream);
      if (e != hipSuccess || *word < 0)
        raise(PyExc_RuntimeError, e != hipSuccess ? std::string("stk_amd: ") + hipGetErrorString(e) : "stk_amd: the count was not delivered");
    }
    return *word;
  }
};

// ------------------------------------------------------------------------------------------------ topology and formats
void row_indices(const Tensor& offsets_, const Tensor& out) {
  need_gpu(offsets_), need_gpu(out);
  require(out.is_contiguous(), "out must be contiguous");
  const c10::DeviceGuard guard(out.device());
  const Tensor offsets = offsets32(offsets_);
  check(stk_row_indices(ptr<int32_t>(offsets), offsets.numel() - 1, out.numel(), ptr<void>(out), index_dtype(out.scalar_type()), stream_of(out)));
}

std::tuple<Tensor, Tensor, Tensor> transpose_meta(int64_t block_cols, const Tensor& row_indices, const Tensor& column_indices) {
  need_gpu(row_indices), need_gpu(column_indices);
  const c10::DeviceGuard guard(column_indices.device());
  const Tensor ri = index(row_indices), ci = index(column_indices);
  require(ri.scalar_type() == ci.scalar_type(), "row and column indices must have one dtype");
  const int64_t nnz = ci.numel();
  Tensor cit = at::empty({nnz}, ri.options()), offsets_t = at::empty({block_cols + 1}, ri.options().dtype(at::kInt));
  Tensor bot = at::empty({nnz}, offsets_t.options());
  const size_t bytes = stk_transpose_meta_workspace_bytes(nnz);
  Tensor ws = at::empty({(int64_t)bytes}, ri.options().dtype(at::kByte));
  check(stk_transpose_meta(ptr<void>(ri), ptr<void>(ci), nnz, block_cols, index_dtype(ci.scalar_type()), ptr<void>(cit), ptr<int32_t>(offsets_t),
                           ptr<int32_t>(bot), ptr<void>(ws), bytes, stream_of(ci)));
  return {cit, offsets_t, bot};
}

// offsets, row_indices, column_indices, offsets_t, column_indices_t, block_offsets_t and, with_plan, the fusion plan
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, OptTensor> dmoe_topology(const Tensor& padded_bins, int blocking, int64_t block_rows,
                                                                                    int64_t width, bool int32_indices, bool with_plan) {
  need_gpu(padded_bins);
  require(padded_bins.dim() == 1 && padded_bins.numel() > 0, "padded_bins holds one number per expert");
  const c10::DeviceGuard guard(padded_bins.device());
  const Tensor bins = offsets32(padded_bins);
  const int64_t experts = bins.numel(), nnz = block_rows * width;
  const auto ints = bins.options(), idx = ints.dtype(int32_indices ? at::kInt : at::kShort);
  Tensor offsets = at::empty({block_rows + 1}, ints), offsets_t = at::empty({experts * width + 1}, ints), ri = at::empty({nnz}, idx),
         ci = at::empty({nnz}, idx), cit = at::empty({nnz}, idx), bot = at::empty({nnz}, ints);
  OptTensor plan;
  size_t bytes = 0;
  if (with_plan) {
    bytes = stk_plan_bytes(block_rows, experts * width, nnz);
    plan = at::empty({(int64_t)bytes}, ints.dtype(at::kByte));
  }
  check(stk_dmoe_topology_plan(ptr<int32_t>(bins), experts, blocking, block_rows, width, int32_indices ? STK_I32 : STK_I16, ptr<int32_t>(offsets), ptr<void>(ri),
                               ptr<void>(ci), ptr<int32_t>(offsets_t), ptr<void>(cit), ptr<int32_t>(bot), ptr<uint8_t>(plan), bytes, stream_of(bins)));
  return {offsets, ri, ci, offsets_t, cit, bot, plan};
}

int elem_bytes(const Tensor& t) {
  if (t.element_size() != 2 && t.element_size() != 4)
    raise(PyExc_NotImplementedError, std::string("stk_amd: format conversion handles 2- and 4-byte elements, got ") + c10::toString(t.scalar_type()));
  return (int)t.element_size();
}

Tensor to_dense(const Tensor& data_, const Tensor& row_indices, const Tensor& column_indices, int64_t rows, int64_t cols, const OptTensor& offsets) {
  need_gpu(data_);
  const c10::DeviceGuard guard(data_.device());
  const Tensor data = data_.detach().contiguous(), ri = index(row_indices), ci = index(column_indices);
  Tensor out = at::empty({rows, cols}, data.options());
  const int64_t blocking = data.size(-1);
  const bool by_rows = offsets && offsets->scalar_type() == at::kInt && offsets->is_contiguous() && offsets->device() == data.device() && blocking > 0 &&
                       ci.numel() == data.size(0) && rows % blocking == 0 && offsets->numel() == rows / blocking + 1;
  check(stk_to_dense_rows(ptr<void>(data), by_rows ? ptr<int32_t>(*offsets) : nullptr, ptr<void>(ri), ptr<void>(ci), data.size(0), (int)blocking, rows, cols,
                          elem_bytes(data), index_dtype(ci.scalar_type()), ptr<void>(out), stream_of(data)));
  return out;
}

// Scratch allocations of this size or more are not left alive behind the small views returned.
constexpr int64_t kKeepBytes = 1 << 16;

// data, row_indices, column_indices and offsets of the nonzero blocks of x, and for matrices of few blocks, where they come
// with the rest, column_indices_t, offsets_t and block_offsets_t
std::tuple<Tensor, Tensor, Tensor, Tensor, OptTensor, OptTensor, OptTensor> to_sparse(const Tensor& x_, int64_t blocking, bool int32_indices) {
  need_gpu(x_);
  require(x_.dim() == 2, "to_sparse takes a matrix");
  const int64_t rows = x_.size(0), cols = x_.size(1);
  require(blocking > 0 && rows % blocking == 0 && cols % blocking == 0, "the matrix must be made of whole blocks");
  const c10::DeviceGuard guard(x_.device());
  const Tensor x = (x_.stride(1) != 1 && cols > 1 ? x_.contiguous() : x_).detach();
  const int64_t br = rows / blocking, bc = cols / blocking, blocks = br * bc;
  const hipStream_t stream = stream_of(x);
  if (capture_id(reinterpret_cast<int64_t>(stream)))
    raise(PyExc_RuntimeError, "to_sparse sizes its result by the number of nonzero blocks, which the host reads back: it cannot be captured into a graph");
  const int bytes = elem_bytes(x), idx = int32_indices ? STK_I32 : STK_I16;
  const bool small = blocks > 0 && blocks <= STK_TO_SPARSE_INDEX_BLOCKS && br <= 1024 && bc <= 1024;
  // one allocation for offsets (int32) and the block mask (bytes) behind it
  Tensor scratch = at::empty({4 * (br + 1) + std::max<int64_t>(blocks, 1)}, x.options().dtype(at::kByte));
  Tensor offsets = scratch.narrow(0, 0, 4 * (br + 1)).view(at::kInt);
  uint8_t* mask = ptr<uint8_t>(scratch) + 4 * (br + 1);
  // the index arrays need no nnz: launched before the host knows it, into room for every block (the first nnz entries are
  // written; the index tensors returned are views of that room, at multiples of 256 bytes like allocations of their own)
  const int64_t half = std::max<int64_t>((blocks + 127) / 128 * 128, 128), columns = (bc + 1 + 63) / 64 * 64;
  Tensor room = at::empty({(small ? 3 : 2) * half}, x.options().dtype(int32_indices ? at::kInt : at::kShort)), room_t;
  const auto third = [&](int i) { return ptr<char>(room) + i * half * room.element_size(); };
  const Mailbox box(x.device());
  int coordinates = STK_OK;
  if (small) {
    room_t = at::empty({columns + half}, x.options().dtype(at::kInt));
    check(stk_to_sparse_index(ptr<void>(x), rows, cols, x.stride(0), (int)blocking, bytes, mask, ptr<int32_t>(offsets), third(0), third(1),
                              ptr<int32_t>(room_t), third(2), ptr<int32_t>(room_t) + columns, idx, const_cast<int32_t*>(box.word), stream));
  } else {
    check(stk_to_sparse_count_nnz(ptr<void>(x), rows, cols, x.stride(0), (int)blocking, bytes, mask, ptr<int32_t>(offsets), const_cast<int32_t*>(box.word), stream));
    coordinates = stk_to_sparse_coordinates(rows, cols, (int)blocking, mask, ptr<int32_t>(offsets), third(0), third(1), idx, stream);
  }
  const int64_t nnz = box.receive(stream);   // (also where a launch behind the count's failed: the word is free only once it is delivered)
  check(coordinates);
  Tensor data = at::empty({nnz, blocking, blocking}, x.options());
  check(stk_to_sparse_gather(ptr<void>(x), rows, cols, x.stride(0), (int)blocking, bytes, third(0), third(1), nnz, idx, ptr<void>(data), stream));
  Tensor ri = room.narrow(0, 0, nnz), ci = room.narrow(0, half, nnz);
  OptTensor ci_t, offsets_t, bo_t;
  if (small) ci_t = room.narrow(0, 2 * half, nnz), offsets_t = room_t.narrow(0, 0, bc + 1), bo_t = room_t.narrow(0, columns, nnz);
  // A Matrix keeps these tensors for as long as it lives.  Where the room for every block is much more than the
  // nonzero blocks need (a large, very sparse matrix), they are copied out of it, and the offsets out of the
  // allocation they share with the block mask, so that the O(rows x columns / blocking^2) buffers can go.
  if (room.numel() * room.element_size() >= kKeepBytes && 4 * nnz <= blocks) {
    ri = ri.clone(), ci = ci.clone();
    if (small) ci_t = ci_t->clone(), offsets_t = offsets_t->clone(), bo_t = bo_t->clone();
  }
  if (scratch.numel() >= kKeepBytes && 16 * (br + 1) <= scratch.numel()) offsets = offsets.clone();
  return {data, ri, ci, offsets, ci_t, offsets_t, bo_t};
}

// ------------------------------------------------------------------------------------------------ values and routing
Tensor activation_product(const Tensor& sums_, const OptTensor& factor_, int activation) {
  need_gpu(sums_);
  const c10::DeviceGuard guard(sums_.device());
  const Tensor sums = sums_.detach().contiguous();
  Tensor out = at::empty_like(sums);
  OptTensor factor;
  if (factor_) {
    need_gpu(*factor_);
    factor = factor_->detach().contiguous();
    require(factor->sizes() == sums.sizes() && factor->scalar_type() == sums.scalar_type(), "sums and factor must have one shape and dtype");
  }
  if (sums.numel() == 0) return out;
  check(stk_activation_product(ptr<void>(sums), ptr<void>(factor), ptr<void>(out), sums.numel(), activation, value_dtype(sums), stream_of(sums)));
  return out;
}

// indices, bin_ids, bins, padded_bins, slot_rows, row_slots.  padded_rows < 0: row_slots gets exactly the rows of the
// padded layout, whose number the host waits for.
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> route(const Tensor& top_experts, int64_t experts, int64_t blocking, int64_t padded_rows) {
  need_gpu(top_experts);
  const c10::DeviceGuard guard(top_experts.device());
  const Tensor e = top_experts.reshape({-1}).to(at::kInt).contiguous();
  const int64_t slots = e.numel();
  const bool exact = padded_rows < 0;
  const int64_t rows = exact ? (slots + experts * (blocking - 1)) / std::max<int64_t>(blocking, 1) * blocking : padded_rows;
  const int64_t ws = ((int64_t)stk_route_workspace_bytes(slots, experts) + 3) / 4;
  // one allocation for the six outputs and the workspace
  Tensor all = at::empty({3 * slots + 2 * experts + rows + ws}, e.options());
  int64_t used = 0;
  const auto part = [&](int64_t n) {
    Tensor t = all.narrow(0, used, n);
    used += n;
    return t;
  };
  Tensor indices = part(slots), bin_ids = part(slots), slot_rows = part(slots), bins = part(experts), padded_bins = part(experts), row_slots = part(rows);
  const hipStream_t stream = stream_of(e);
  if (exact && capture_id(reinterpret_cast<int64_t>(stream)))
    raise(PyExc_RuntimeError, "route sizes the padded layout by the expert choices, which the host reads back: under a graph capture give it padded_rows");
  std::optional<Mailbox> box;
  if (exact) box.emplace(e.device());
  check(stk_route_total(ptr<int32_t>(e), slots, experts, (int)blocking, rows, ptr<int32_t>(indices), ptr<int32_t>(bin_ids), ptr<int32_t>(bins),
                        ptr<int32_t>(padded_bins), ptr<int32_t>(slot_rows), ptr<int32_t>(row_slots), ptr<int32_t>(all) + used, (size_t)ws * 4,
                        box ? const_cast<int32_t*>(box->word) : nullptr, stream));
  if (exact) row_slots = row_slots.narrow(0, 0, box->receive(stream));
  return {indices, bin_ids, bins, padded_bins, slot_rows, row_slots};
}

// 2-D 16-bit tensor whose rows the copy kernels can read in place (unit column stride, rows at multiples of 16 bytes);
// anything else is copied to row-major first.
Tensor rows16(const Tensor& x_) {
  const Tensor x = x_.detach();
  require(x.dim() == 2, "token rows are a matrix");
  if (x.numel() && !(x.stride(1) == 1 && x.stride(0) % 8 == 0 && x.stride(0) >= x.size(1) && aligned(x))) return x.contiguous();
  return x;
}
int64_t row_stride(const Tensor& x) { return x.numel() && x.size(0) > 1 ? x.stride(0) : std::max<int64_t>(x.size(1), 1); }
OptTensor weights32(const OptTensor& weights, int64_t slots) {
  if (!weights) return {};
  if (weights->numel() > 0) need_gpu(*weights);   // (a kernel reads them: an address in host memory would be a fault)
  Tensor w = weights->detach().reshape({-1}).to(at::kFloat).contiguous();
  if (w.numel() != slots)
    raise(PyExc_AssertionError, "one weight per slot: " + std::to_string(w.numel()) + " weights for " + std::to_string(slots) + " slots");
  return w;
}

// out[r] = (weights[s]) * x[s / top_k], s = row_slots[r]; zeros where s < 0
Tensor padded_gather(const Tensor& x_, const Tensor& row_slots, int top_k, const OptTensor& weights) {
  need_gpu(x_), need_gpu(row_slots);
  const c10::DeviceGuard guard(x_.device());
  const Tensor x = rows16(x_);
  const int64_t tokens = x.size(0), cols = x.size(1), rows = row_slots.numel();
  const OptTensor w = weights32(weights, tokens * top_k);
  Tensor out = at::empty({rows, cols}, x.options());
  check(stk_padded_gather(ptr<void>(x), tokens, cols, row_stride(x), ptr<int32_t>(row_slots), ptr<float>(w), top_k, rows, ptr<void>(out),
                          std::max<int64_t>(cols, 1), value_dtype(x), stream_of(x)));
  return out;
}

// out[t] = sum_k (weights[s]) * x[slot_rows[s]], s = t * top_k + k
Tensor padded_scatter(const Tensor& x_, const Tensor& slot_rows, int top_k, const OptTensor& weights) {
  need_gpu(x_), need_gpu(slot_rows);
  const c10::DeviceGuard guard(x_.device());
  const Tensor x = rows16(x_);
  const int64_t rows = x.size(0), cols = x.size(1), slots = slot_rows.numel();
  if (top_k < 1 || slots % top_k)
    raise(PyExc_AssertionError, std::to_string(slots) + " slots are not a multiple of top_k = " + std::to_string(top_k));
  const OptTensor w = weights32(weights, slots);
  Tensor out = at::empty({slots / top_k, cols}, x.options());
  check(stk_padded_scatter(ptr<void>(x), rows, cols, row_stride(x), ptr<int32_t>(slot_rows), ptr<float>(w), top_k, slots / top_k, ptr<void>(out),
                           std::max<int64_t>(cols, 1), value_dtype(x), stream_of(x)));
  return out;
}

// fp32 [slots]: <x[slot_rows[s]], grad[s / top_k]>
Tensor padded_scatter_weight_gradient(const Tensor& x_, const Tensor& grad_, const Tensor& slot_rows, int top_k) {
  need_gpu(x_), need_gpu(grad_), need_gpu(slot_rows);
  const c10::DeviceGuard guard(x_.device());
  const Tensor x = rows16(x_), grad = rows16(grad_);
  require(x.scalar_type() == grad.scalar_type() && x.size(1) == grad.size(1), "x and grad must have one dtype and row length");
  const int64_t slots = slot_rows.numel();
  require(grad.size(0) * top_k == slots, "one gradient row per token");
  Tensor out = at::empty({slots}, x.options().dtype(at::kFloat));
  check(stk_padded_scatter_weight_gradient(ptr<void>(x), x.size(0), x.size(1), row_stride(x), ptr<void>(grad), row_stride(grad), ptr<int32_t>(slot_rows),
                                           top_k, grad.size(0), ptr<float>(out), value_dtype(x), stream_of(x)));
  return out;
}

// out = act(sdd(padded_gather(x), rhs)); false, with nothing launched, when the library has no such kernel for this case
bool sdd_gather(const Tensor& x_, const Tensor& row_slots, int top_k, const Tensor& rhs_, int64_t m, int64_t n, const Tensor& out, const Tensor& offsets,
                const Tensor& row_indices, const Tensor& column_indices, const OptTensor& plan, int activation) {
  need_gpu(x_), need_gpu(row_slots), need_gpu(rhs_), need_gpu(out);
  const int64_t b = out.size(-1), nnz = row_indices.numel();
  const c10::DeviceGuard guard(out.device());
  const Tensor x = rows16(x_);
  const int64_t tokens = x.size(0), k = x.size(1);
  require(rhs_.dim() == 2 && k == rhs_.size(0) && n == rhs_.size(1), "incompatible dimensions");
  require(row_slots.scalar_type() == at::kInt && row_slots.is_contiguous() && row_slots.numel() >= m, "row_slots must name the rows of the padded layout");
  matmul_dims(m, k, n, b);
  if (tokens == 0 || tokens * row_stride(x) * 2 >= (int64_t(1) << 32)) return false;
  if (nnz == 0) return true;
  const Tensor rhs = dense_operand(rhs_);
  require(out.is_contiguous() && x.scalar_type() == rhs.scalar_type() && x.scalar_type() == out.scalar_type(), "operands and out must have one dtype");
  const Tensor ri = index(row_indices), ci = index(column_indices), offs = offsets32(offsets);
  const int status = stk_sdd_gather(ptr<void>(x), tokens, row_stride(x), ptr<int32_t>(row_slots), top_k, ptr<void>(rhs), rhs.stride(0), rhs.stride(1), m, k, n,
                                    ptr<void>(out), plan ? ptr<int32_t>(offs) : nullptr, ptr<void>(ri), ptr<void>(ci), nnz, (int)b, value_dtype(out),
                                    index_dtype(ri.scalar_type()), ptr<uint8_t>(plan), activation, stream_of(out));
  if (status == STK_ERR_UNSUPPORTED) return false;
  check(status);
  return true;
}

// out = padded_scatter(sparse @ rhs, top_k = 1, weights); the status, STK_ERR_UNSUPPORTED, with nothing launched, when the
// library has no such kernel
int dsd_scatter(int64_t m, int64_t k, const Tensor& data, const Tensor& offsets, const Tensor& column_indices, const Tensor& rhs_, const Tensor& row_slots,
                 const OptTensor& weights, const Tensor& out, const Tensor& plan, const OptTensor& workspace) {
  need_gpu(data), need_gpu(rhs_), need_gpu(row_slots), need_gpu(out);
  require(rhs_.dim() == 2 && k == rhs_.size(0), "incompatible dimensions");
  const int64_t n = rhs_.size(1), b = data.size(-1);
  matmul_dims(m, k, n, b);
  const c10::DeviceGuard guard(out.device());
  const Tensor rhs = dense_operand(rhs_);
  require(data.is_contiguous() && out.stride(1) == 1 && out.size(1) == n, "the sparse values must be contiguous and out row-major");
  require(data.scalar_type() == rhs.scalar_type() && data.scalar_type() == out.scalar_type(), "operands and out must have one dtype");
  require(row_slots.scalar_type() == at::kInt && row_slots.is_contiguous() && row_slots.numel() >= m, "row_slots must name the rows of the padded layout");
  const OptTensor w = weights32(weights, out.size(0));
  const Tensor ci = index(column_indices), offs = offsets32(offsets);
  return stk_dsd_scatter(m, k, n, ptr<void>(data), ptr<int32_t>(offs), ptr<void>(ci), ptr<void>(rhs), rhs.stride(0), rhs.stride(1),
                         ptr<int32_t>(row_slots), ptr<float>(w), out.size(0), ptr<void>(out), out.stride(0), data.size(0), (int)b, value_dtype(out),
                         index_dtype(ci.scalar_type()), ptr<uint8_t>(plan), ptr<void>(workspace), workspace ? workspace->numel() : 0,
                         stream_of(out));
}

// Whether dsd_scatter_few is for these sizes (-1: no), and the size of the workspace, with room for `partial_tiles`, of the
// stk_dsd whose bits it gives, 0 if that one cuts no tile.
int64_t dsd_scatter_few_case(int64_t m, int64_t n, int64_t nnz, int64_t slots, int64_t partial_tiles) {
  if (stk_dsd_scatter_few_bytes(m, n, nnz, slots) == 0) return -1;
  const int64_t bytes = partial_tiles > 0 ? stk_dsd_workspace_counter_bytes() + partial_tiles * stk_dsd_workspace_slot_bytes() : 0;
  return stk_dsd_cuts(m, n, nnz, bytes) ? bytes : 0;
}

// padded_scatter(sparse @ rhs, top_k, weights) where the block rows hold few slots each; nothing, with nothing launched, when the
// library has no kernel for this case
OptTensor dsd_scatter_few(int64_t m, int64_t k, const Tensor& data, const Tensor& offsets, const Tensor& column_indices, const Tensor& rhs_,
                          const Tensor& row_slots, const Tensor& slot_rows, int top_k, const OptTensor& weights, const OptTensor& plan,
                          int64_t dsd_workspace_bytes) {
  // (what the two calls refuse is left to them)
  if (rhs_.dim() != 2 || k != rhs_.size(0) || top_k < 1) return {};
  const int64_t n = rhs_.size(1), b = data.size(-1), slots = slot_rows.numel(), nnz = data.size(0);
  for (const Tensor* t : {&rhs_, &row_slots, &slot_rows, &offsets, &column_indices})
    if (t->device() != data.device()) return {};
  for (const Tensor* t : {&row_slots, &slot_rows})
    if (t->scalar_type() != at::kInt || !t->is_contiguous()) return {};
  if (b != 128 || n % b || slots % top_k || data.scalar_type() != rhs_.scalar_type() || !data.is_contiguous() || !aligned(data) || row_slots.numel() < m ||
      (data.scalar_type() != at::kHalf && data.scalar_type() != at::kBFloat16))
    return {};
  const int64_t bytes = stk_dsd_scatter_few_bytes(m, n, nnz, slots);
  if (bytes == 0) return {};
  const c10::DeviceGuard guard(rhs_.device());
  const Tensor rhs = dense_operand(rhs_);
  const OptTensor w = weights32(weights, slots);
  const Tensor ci = index(column_indices), offs = offsets32(offsets);
  Tensor out = at::empty({slots / top_k, n}, rhs.options());
  const Tensor sums = at::empty({bytes / 4}, rhs.options().dtype(at::kFloat));
  const int status = stk_dsd_scatter_few_as_cut(m, k, n, ptr<void>(data), ptr<int32_t>(offs), ptr<void>(ci), ptr<void>(rhs), rhs.stride(0), rhs.stride(1),
                                         ptr<int32_t>(row_slots), ptr<int32_t>(slot_rows), ptr<float>(w), top_k, slots / top_k, ptr<void>(out), n, nnz,
                                         (int)b, value_dtype(rhs), index_dtype(ci.scalar_type()), ptr<void>(sums), bytes,
                                                ptr<uint8_t>(plan), dsd_workspace_bytes, stream_of(rhs));
  if (status == STK_ERR_UNSUPPORTED) return {};
  check(status);
  return out;
}

// ------------------------------------------------------------------------------------------------ layer norm
// x [..., size] as rows of `size` values at one distance from each other: in place where the leading dimensions allow that,
// copied to row-major otherwise.
struct Rows {
  Tensor t;
  int64_t rows, size, stride;
  explicit Rows(const Tensor& x) : t(x.detach()), rows(1), size(x.size(-1)), stride(0) {
    for (int64_t d = 0; d < t.dim() - 1; d++) rows *= t.size(d);
    bool in_place = size <= 1 || t.stride(-1) == 1;
    stride = size;
    int64_t step = -1, inside = 1;   // the distance between rows, and the rows spanned by the dimensions behind d
    for (int64_t d = t.dim() - 2; d >= 0 && in_place; d--) {
      if (t.size(d) == 1) continue;
      if (step < 0) step = t.stride(d);
      else in_place = t.stride(d) == step * inside;
      inside *= t.size(d);
    }
    if (step >= 0) stride = step;
    if (rows > 0 && !in_place) t = t.contiguous(), stride = size;
  }
};
// A parameter of a layer norm: one value per feature, of the rows' type or float32.
OptTensor norm_parameter(const OptTensor& p_, const Tensor& x, const char* what) {
  if (!p_) return {};
  need_gpu(*p_);
  const OptTensor p = p_->detach().contiguous();
  require(p->dim() == 1 && p->numel() == x.size(-1), "layer_norm: weight and bias have one value per feature");
  require(p->device() == x.device(), "layer_norm: the rows and their parameters are on one device");
  if (p->scalar_type() != x.scalar_type() && p->scalar_type() != at::kFloat)
    raise(PyExc_NotImplementedError, std::string("stk_amd: layer_norm's ") + what + " has the rows' type or float32, got " + c10::toString(p->scalar_type()));
  return p;
}
int norm_parameter_dtype(const OptTensor& weight, const OptTensor& bias, const Tensor& x) {
  require(!weight || !bias || weight->scalar_type() == bias->scalar_type(), "layer_norm: weight and bias have one type");
  return weight ? value_dtype(*weight) : bias ? value_dtype(*bias) : value_dtype(x);
}
// The result and, with_statistics, mean and 1 / deviation of the rows.
std::tuple<Tensor, OptTensor> layer_norm(const Tensor& x_, const OptTensor& weight_, const OptTensor& bias_, double eps, bool with_statistics) {
  need_gpu(x_);
  require(x_.dim() >= 1 && x_.size(-1) >= 1, "layer_norm: rows of at least one value");
  value_dtype(x_);
  const c10::DeviceGuard guard(x_.device());
  const OptTensor weight = norm_parameter(weight_, x_, "weight"), bias = norm_parameter(bias_, x_, "bias");
  const int param = norm_parameter_dtype(weight, bias, x_);
  const Rows x(x_);
  Tensor out = at::empty(x_.sizes(), x_.options());
  OptTensor statistics;
  if (with_statistics) statistics = at::empty({2, x.rows}, x_.options().dtype(at::kFloat));
  float* mean = ptr<float>(statistics);
  check(stk_layer_norm(ptr<void>(x.t), x.rows, x.size, x.stride, ptr<void>(weight), ptr<void>(bias), (float)eps, ptr<void>(out), x.size, mean,
                       mean ? mean + x.rows : nullptr, value_dtype(x_), param, stream_of(x_)));
  return {out, statistics};
}
// The gradients that are asked for.
std::tuple<OptTensor, OptTensor, OptTensor> layer_norm_backward(const Tensor& grad_, const Tensor& x_, const Tensor& statistics, const OptTensor& weight_,
                                                                const OptTensor& bias_, bool want_x, bool want_weight, bool want_bias) {
  need_gpu(grad_), need_gpu(x_);
  require(grad_.sizes() == x_.sizes() && grad_.scalar_type() == x_.scalar_type(), "layer_norm: the gradient is laid out like the result");
  const c10::DeviceGuard guard(x_.device());
  const OptTensor weight = norm_parameter(weight_, x_, "weight"), bias = norm_parameter(bias_, x_, "bias");
  const int param = norm_parameter_dtype(weight, bias, x_);
  const Rows x(x_), grad(grad_);
  OptTensor dx, dweight, dbias, workspace;
  if (want_x) dx = at::empty(x_.sizes(), x_.options());
  if (want_weight && weight) dweight = at::empty_like(*weight);
  if (want_bias && bias) dbias = at::empty_like(*bias);
  size_t bytes = 0;
  if (dweight || dbias) {
    bytes = stk_layer_norm_backward_workspace_bytes(x.rows, x.size);
    workspace = at::empty({(int64_t)bytes}, x_.options().dtype(at::kByte));
  }
  check(stk_layer_norm_backward(ptr<void>(grad.t), grad.stride, ptr<void>(x.t), x.stride, ptr<float>(statistics), ptr<float>(statistics) + x.rows, ptr<void>(weight),
                                x.rows, x.size, ptr<void>(dx), x.size, ptr<void>(dweight), ptr<void>(dbias), value_dtype(x_), param, ptr<void>(workspace), bytes,
                                stream_of(x_)));
  return {dx, dweight, dbias};
}

// Outputs of a backward pass that has no gradient of its own: asked for with create_graph they say so when they are differentiated.
torch::autograd::variable_list once_differentiable(torch::autograd::variable_list grads, const char* what) {
  if (!at::GradMode::is_enabled()) return grads;
  torch::autograd::variable_list inputs;
  for (const Tensor& t : grads) inputs.push_back(t.defined() ? t.detach().requires_grad_(true) : t);
  const auto error = std::make_shared<torch::autograd::DelayedError>(std::string("stk_amd: ") + what + " can be differentiated once", (int64_t)inputs.size());
  return error->apply(std::move(inputs));
}

// Autograd in native code: through a Python function a forward and backward pass cost 30 us more on the host than these, longer than
// the kernels of a layer norm of 16384 x 1024 values take.
struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
    auto [out, statistics] = layer_norm(x, weight, bias, eps, true);
    ctx->save_for_backward({x, weight ? *weight : Tensor(), bias ? *bias : Tensor(), *statistics});
    return out;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const auto given = [&](size_t i) { return saved[i].defined() ? OptTensor(saved[i]) : OptTensor(); };
    // (parameters that are not there have no edge)
    size_t edge = 0;
    const bool want_x = ctx->needs_input_grad(edge++), want_weight = saved[1].defined() && ctx->needs_input_grad(edge++);
    const bool want_bias = saved[2].defined() && ctx->needs_input_grad(edge++);
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    const auto [dx, dweight, dbias] = layer_norm_backward(grads[0], saved[0], saved[3], given(1), given(2), want_x, want_weight, want_bias);
    return once_differentiable({dx.value_or(Tensor()), dweight.value_or(Tensor()), dbias.value_or(Tensor()), Tensor()}, "layer_norm");
  }
};
bool wants_gradient(const OptTensor& t) { return t && t->requires_grad(); }
// layer_norm with its place in the graph where a gradient is wanted.
Tensor layer_norm_graph(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
  if (at::GradMode::is_enabled() && (x.requires_grad() || wants_gradient(weight) || wants_gradient(bias))) return LayerNorm::apply(x, weight, bias, eps);
  return std::get<0>(layer_norm(x, weight, bias, eps, false));
}

// ------------------------------------------------------------------------------------------------ router
// Scores as rows: one dimension of tokens in front of that of the experts.
Tensor score_rows(const Tensor& scores) {
  require(scores.dim() == 2, "top_experts: scores are [tokens, experts]");
  const Tensor s = scores.detach();
  return s.size(1) <= 1 || s.stride(1) == 1 ? s : s.contiguous();
}
// chosen and weights
std::tuple<Tensor, Tensor> top_experts(const Tensor& scores_, int64_t top_k, bool normalize) {
  need_gpu(scores_);
  const int dtype = value_dtype(scores_);
  const c10::DeviceGuard guard(scores_.device());
  const Tensor scores = score_rows(scores_);
  const int64_t tokens = scores.size(0), experts = scores.size(1);
  require(top_k >= 1 && top_k <= experts, "top_experts: top_k of 1 up to the number of experts");
  Tensor chosen = at::empty({tokens, top_k}, scores.options().dtype(at::kInt)), weights = at::empty({tokens, top_k}, scores.options().dtype(at::kFloat));
  check(stk_top_experts(ptr<void>(scores), tokens, experts, scores.stride(0), (int)std::min<int64_t>(top_k, INT32_MAX), normalize, ptr<int32_t>(chosen),
                        ptr<float>(weights), dtype, stream_of(scores)));
  return {chosen, weights};
}
Tensor top_experts_backward(const Tensor& scores_, const Tensor& chosen, const Tensor& weights, const Tensor& grad_, bool normalize) {
  need_gpu(grad_);
  const c10::DeviceGuard guard(scores_.device());
  const Tensor scores = score_rows(scores_), grad = grad_.detach().to(at::kFloat).contiguous();
  require(grad.sizes() == weights.sizes(), "top_experts: one gradient per weight");
  Tensor out = at::empty(scores.sizes(), scores.options());
  check(stk_top_experts_backward(ptr<void>(scores), scores.stride(0), ptr<int32_t>(chosen), ptr<float>(weights), ptr<float>(grad), scores.size(0),
                                 scores.size(1), (int)weights.size(1), normalize, ptr<void>(out), out.size(1), value_dtype(scores), stream_of(scores)));
  return out;
}

struct TopExperts : torch::autograd::Function<TopExperts> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& scores, int64_t top_k, bool normalize) {
    auto [chosen, weights] = top_experts(scores, top_k, normalize);
    ctx->save_for_backward({scores, chosen, weights});
    ctx->saved_data["normalize"] = normalize;
    ctx->mark_non_differentiable({chosen});
    return {chosen, weights};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    if (!grads[1].defined()) return {Tensor(), Tensor(), Tensor()};
    return once_differentiable({top_experts_backward(saved[0], saved[1], saved[2], grads[1], ctx->saved_data["normalize"].toBool()), Tensor(), Tensor()}, "top_experts");
  }
};
std::tuple<Tensor, Tensor> top_experts_graph(const Tensor& scores, int64_t top_k, bool normalize) {
  if (!at::GradMode::is_enabled() || !scores.requires_grad()) return top_experts(scores, top_k, normalize);
  const auto out = TopExperts::apply(scores, top_k, normalize);
  return {out[0], out[1]};
}

// ------------------------------------------------------------------------------------------------ 4-bit weights
// codes [experts, inputs, outputs] and scales, offsets [experts, groups, outputs] of weights [experts, inputs, outputs]
std::tuple<Tensor, Tensor, OptTensor> quantize_4bit(const Tensor& w_, int64_t group, bool with_offsets, at::ScalarType dtype) {
  need_gpu(w_);
  const Tensor w = w_.detach();
  require(w.dim() == 3 && group >= 1, "quantize_4bit: weights are [inputs, outputs] or [experts, inputs, outputs], in groups of inputs");
  const c10::DeviceGuard guard(w.device());
  const int64_t experts = w.size(0), inputs = w.size(1), outputs = w.size(2), groups = inputs / group + (inputs % group != 0);
  Tensor codes = at::empty({experts, inputs, outputs}, w.options().dtype(at::kByte)), scales = at::empty({experts, groups, outputs}, w.options().dtype(dtype));
  OptTensor offsets;
  if (with_offsets) offsets = at::empty_like(scales);
  check(stk_quantize_4bit(ptr<void>(w), w.stride(0), w.stride(1), w.stride(2), experts, inputs, outputs, group, ptr<uint8_t>(codes), ptr<void>(scales),
                          ptr<void>(offsets), value_dtype(w), value_dtype(scales), stream_of(w)));
  return {codes, scales, offsets};
}
// The packed codes, scales and offsets; codes [experts, inputs, outputs], scales and offsets [experts, groups, outputs].
std::tuple<Tensor, Tensor, OptTensor> pack_4bit(const Tensor& codes_, const Tensor& scales_, int64_t group, const OptTensor& offsets_) {
  need_gpu(codes_), need_gpu(scales_);
  require(codes_.dim() == 3 && scales_.dim() == 3 && group >= 1, "pack_4bit: codes [experts, inputs, outputs], scales [experts, groups, outputs]");
  if (codes_.scalar_type() != at::kByte) raise(PyExc_NotImplementedError, std::string("stk_amd: 4-bit codes are uint8, one a byte, got ") + c10::toString(codes_.scalar_type()));
  const c10::DeviceGuard guard(codes_.device());
  const int64_t experts = codes_.size(0), inputs = codes_.size(1), outputs = codes_.size(2), groups = inputs / group + (inputs % group != 0);
  require(scales_.size(0) == experts && scales_.size(1) == groups && scales_.size(2) == outputs && scales_.device() == codes_.device(),
          "pack_4bit: one scale per group of inputs and output");
  if (scales_.scalar_type() != at::kHalf && scales_.scalar_type() != at::kBFloat16)
    raise(PyExc_NotImplementedError, std::string("stk_amd: 4-bit weights have scales of float16 or bfloat16, got ") + c10::toString(scales_.scalar_type()));
  const Tensor codes = codes_.contiguous(), scales = scales_.detach().contiguous();
  OptTensor offsets, packed_offsets;
  if (offsets_) {
    need_gpu(*offsets_);
    require(offsets_->sizes() == scales.sizes() && offsets_->scalar_type() == scales.scalar_type() && offsets_->device() == scales.device(),
            "pack_4bit: offsets are laid out like the scales");
    offsets = offsets_->detach().contiguous();
  }
  const int64_t along = (inputs + 127) / 128, down = (outputs + 15) / 16;
  Tensor packed = at::empty({experts, down, along, stk_4bit_packed_bytes(1, 1, 1)}, codes.options());
  Tensor packed_scales = at::empty({experts, down, stk_4bit_scales(1, inputs, 1, group)}, scales.options());
  if (offsets) packed_offsets = at::empty_like(packed_scales);
  check(stk_pack_4bit(ptr<uint8_t>(codes), ptr<void>(scales), ptr<void>(offsets), experts, inputs, outputs, group, ptr<void>(packed), ptr<void>(packed_scales),
                      ptr<void>(packed_offsets), stream_of(codes)));
  return {packed, packed_scales, packed_offsets};
}
// Packed weights as the calls take them: what pack_4bit made, in its shapes.
struct Packed {
  int64_t experts, inputs, outputs, group;
  Packed(const Tensor& packed, const Tensor& scales, const OptTensor& offsets, int64_t inputs_, int64_t outputs_, int64_t group_)
      : experts(0), inputs(inputs_), outputs(outputs_), group(group_) {
    need_gpu(packed), need_gpu(scales);
    require(packed.dim() == 4 && packed.scalar_type() == at::kByte && packed.is_contiguous() && scales.is_contiguous() && inputs > 0 && outputs > 0 && group > 0,
            "packed 4-bit weights come from pack_4bit");
    experts = packed.size(0);
    require(packed.numel() == stk_4bit_packed_bytes(experts, inputs, outputs) && scales.numel() == stk_4bit_scales(experts, inputs, outputs, group) &&
                scales.device() == packed.device() &&
                (!offsets || (offsets->numel() == scales.numel() && offsets->is_contiguous() && offsets->scalar_type() == scales.scalar_type() &&
                              offsets->device() == packed.device())),
            "packed 4-bit weights come from pack_4bit");
  }
};
#define PACKED_ARGS const Tensor &packed, const Tensor &scales, const OptTensor &offsets, int64_t inputs, int64_t outputs, int64_t group
Tensor dequantize_4bit(PACKED_ARGS) {
  const Packed w(packed, scales, offsets, inputs, outputs, group);
  const c10::DeviceGuard guard(packed.device());
  Tensor out = at::empty({w.experts, inputs, outputs}, scales.options());
  check(stk_dequantize_4bit(ptr<void>(packed), ptr<void>(scales), ptr<void>(offsets), w.experts, inputs, outputs, group, ptr<void>(out), value_dtype(scales),
                            stream_of(packed)));
  return out;
}
// Rows of the products: `inputs` values of the scales' type, next to each other.
Tensor rows4(const Tensor& x_, const Tensor& scales, int64_t inputs) {
  need_gpu(x_);
  require(x_.dim() == 2 && x_.size(1) == inputs, "incompatible dimensions");
  require(x_.device() == scales.device(), "operands are on one device");
  if (x_.scalar_type() != scales.scalar_type())
    raise(PyExc_NotImplementedError, std::string("stk_amd: rows and scales of 4-bit weights have one type, got ") + c10::toString(x_.scalar_type()) + " and " +
                                         c10::toString(scales.scalar_type()));
  const Tensor x = x_.detach();
  return inputs == 1 || x.stride(1) == 1 ? x : x.contiguous();
}
Tensor matmul_4bit(const Tensor& x_, PACKED_ARGS, int activation) {
  const Packed w(packed, scales, offsets, inputs, outputs, group);
  require(w.experts == 1, "matmul_4bit: the weights of one matrix");
  const c10::DeviceGuard guard(packed.device());
  const Tensor x = rows4(x_, scales, inputs);
  const int64_t rows = x.size(0);
  Tensor out = at::empty({rows, outputs}, x.options());
  check(stk_matmul_4bit(ptr<void>(x), rows, x.stride(0), ptr<void>(packed), ptr<void>(scales), ptr<void>(offsets), inputs, outputs, group, ptr<void>(out), outputs,
                        activation, value_dtype(x), stream_of(x)));
  return out;
}
void check_routing(const Tensor& indices, const Tensor& bins, const Packed& w, const Tensor& scales) {
  need_gpu(indices), need_gpu(bins);
  for (const Tensor* t : {&indices, &bins})
    require(t->scalar_type() == at::kInt && t->is_contiguous() && t->device() == scales.device(), "the routing's arrays come from route");
  require(bins.numel() == w.experts, "one bin for each expert's weights");
}
Tensor gather_matmul_4bit(const Tensor& x_, const Tensor& indices, const Tensor& bins, int top_k, PACKED_ARGS, int activation) {
  const Packed w(packed, scales, offsets, inputs, outputs, group);
  check_routing(indices, bins, w, scales);
  const c10::DeviceGuard guard(packed.device());
  const Tensor x = rows4(x_, scales, inputs);
  const int64_t slots = indices.numel();
  require(top_k >= 1 && x.size(0) * top_k == slots, "one row per token");
  Tensor out = at::empty({slots, outputs}, x.options());
  check(stk_gather_matmul_4bit(ptr<void>(x), x.size(0), x.stride(0), ptr<int32_t>(indices), ptr<int32_t>(bins), top_k, ptr<void>(packed), ptr<void>(scales),
                               ptr<void>(offsets), w.experts, inputs, outputs, group, ptr<void>(out), outputs, activation, value_dtype(x), stream_of(x)));
  return out;
}
Tensor matmul_4bit_scatter(const Tensor& x_, const Tensor& indices, const Tensor& bins, int top_k, PACKED_ARGS, const OptTensor& weights) {
  const Packed w(packed, scales, offsets, inputs, outputs, group);
  check_routing(indices, bins, w, scales);
  const c10::DeviceGuard guard(packed.device());
  const Tensor x = rows4(x_, scales, inputs);
  const int64_t slots = indices.numel();
  require(top_k >= 1 && slots % top_k == 0 && x.size(0) == slots, "one row per slot");
  const OptTensor by_slot = weights32(weights, slots);
  Tensor out = at::empty({slots / top_k, outputs}, x.options());
  const size_t bytes = stk_matmul_4bit_scatter_workspace_bytes(slots, outputs);
  const Tensor ws = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte));
  check(stk_matmul_4bit_scatter(ptr<void>(x), x.stride(0), ptr<int32_t>(indices), ptr<int32_t>(bins), top_k, slots / top_k, ptr<float>(by_slot), ptr<void>(packed),
                                ptr<void>(scales), ptr<void>(offsets), w.experts, inputs, outputs, group, ptr<void>(out), outputs, value_dtype(x), ptr<void>(ws), bytes,
                                stream_of(x)));
  return out;
}

// ------------------------------------------------------------------------------------------------ router with groups
struct GroupChoice {
  int64_t top_k, groups, top_groups, best;
  bool sigmoid, normalize;
  double scale;
};
#define GROUP_CHOICE_ARGS int64_t top_k, int64_t groups, int64_t top_groups, bool sigmoid, int64_t best, bool normalize, double scale
#define GROUP_CHOICE \
  GroupChoice { top_k, groups, top_groups, best, sigmoid, normalize, scale }
int small(int64_t v) { return (int)std::min<int64_t>(std::max<int64_t>(v, INT32_MIN), INT32_MAX); }
std::tuple<Tensor, Tensor> group_choice(const Tensor& scores_, const OptTensor& bias_, const GroupChoice& c) {
  need_gpu(scores_);
  const int dtype = value_dtype(scores_);
  const c10::DeviceGuard guard(scores_.device());
  const Tensor scores = score_rows(scores_);
  const int64_t tokens = scores.size(0), experts = scores.size(1);
  OptTensor bias;
  if (bias_) {
    need_gpu(*bias_);
    require(bias_->dim() == 1 && bias_->numel() == experts && bias_->device() == scores.device(), "group_top_experts: one bias for each expert");
    bias = bias_->detach().to(at::kFloat).contiguous();
  }
  require(c.top_k >= 1 && c.top_k <= experts, "group_top_experts: top_k of 1 up to the number of experts");
  Tensor chosen = at::empty({tokens, c.top_k}, scores.options().dtype(at::kInt)), weights = at::empty({tokens, c.top_k}, scores.options().dtype(at::kFloat));
  check(stk_group_top_experts(ptr<void>(scores), tokens, experts, scores.stride(0), small(c.groups), small(c.top_groups), small(c.best), small(c.top_k), c.sigmoid,
                              ptr<float>(bias), c.normalize, (float)c.scale, ptr<int32_t>(chosen), ptr<float>(weights), dtype, stream_of(scores)));
  return {chosen, weights};
}
std::tuple<Tensor, Tensor> group_top_experts(const Tensor& scores, const OptTensor& bias, GROUP_CHOICE_ARGS) { return group_choice(scores, bias, GROUP_CHOICE); }
Tensor group_top_experts_backward(const Tensor& scores_, const Tensor& chosen, const Tensor& weights, const Tensor& grad_, bool sigmoid, bool normalize, double scale) {
  need_gpu(grad_);
  const c10::DeviceGuard guard(scores_.device());
  const Tensor scores = score_rows(scores_), grad = grad_.detach().to(at::kFloat).contiguous();
  require(grad.sizes() == weights.sizes(), "group_top_experts: one gradient per weight");
  Tensor out = at::empty(scores.sizes(), scores.options());
  check(stk_group_top_experts_backward(ptr<void>(scores), scores.stride(0), ptr<int32_t>(chosen), ptr<float>(weights), ptr<float>(grad), scores.size(0),
                                       scores.size(1), (int)weights.size(1), sigmoid, normalize, (float)scale, ptr<void>(out), out.size(1), value_dtype(scores),
                                       stream_of(scores)));
  return out;
}
struct GroupTopExperts : torch::autograd::Function<GroupTopExperts> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& scores, const OptTensor& bias, const GroupChoice& c) {
    auto [chosen, weights] = group_choice(scores, bias, c);
    ctx->save_for_backward({scores, chosen, weights});
    ctx->set_materialize_grads(false);   // (chosen has none)
    ctx->saved_data["sigmoid"] = c.sigmoid, ctx->saved_data["normalize"] = c.normalize, ctx->saved_data["scale"] = c.scale;
    ctx->mark_non_differentiable({chosen});
    return {chosen, weights};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    if (!grads[1].defined()) return {Tensor(), Tensor(), Tensor()};
    return once_differentiable({group_top_experts_backward(saved[0], saved[1], saved[2], grads[1], ctx->saved_data["sigmoid"].toBool(),
                                                           ctx->saved_data["normalize"].toBool(), ctx->saved_data["scale"].toDouble()),
                                Tensor(), Tensor()},
                               "group_top_experts");
  }
};
std::tuple<Tensor, Tensor> group_top_experts_graph(const Tensor& scores, const OptTensor& bias, GROUP_CHOICE_ARGS) {
  if (!at::GradMode::is_enabled() || !scores.requires_grad()) return group_choice(scores, bias, GROUP_CHOICE);
  const auto out = GroupTopExperts::apply(scores, bias ? OptTensor(bias->detach()) : bias, GROUP_CHOICE);
  return {out[0], out[1]};
}

// ------------------------------------------------------------------------------------------------ 8-bit floating-point weights
// (packed codes, scales) of weights [experts, inputs, outputs], and where wanted those of their transpose.
std::tuple<Tensor, Tensor, OptTensor, OptTensor> quantize_8bit(const Tensor& w_, bool with_transpose) {
  need_gpu(w_);
  const int dtype = value_dtype(w_);
  const Tensor w = w_.detach();
  require(w.dim() == 3 && w.numel() > 0, "quantize_8bit: weights are [inputs, outputs] or [experts, inputs, outputs]");
  const c10::DeviceGuard guard(w.device());
  const int64_t experts = w.size(0), inputs = w.size(1), outputs = w.size(2);
  const auto bytes = w.options().dtype(at::kByte);
  Tensor packed = at::empty({experts, stk_8bit_piece_bytes(1, inputs, outputs)}, bytes), scales = at::empty({experts, stk_8bit_scale_bytes(1, inputs, outputs, 0)}, bytes);
  OptTensor packed_t, scales_t;
  if (with_transpose)
    packed_t = at::empty({experts, stk_8bit_piece_bytes(1, outputs, inputs)}, bytes), scales_t = at::empty({experts, stk_8bit_scale_bytes(1, outputs, inputs, 0)}, bytes);
  check(stk_quantize_8bit(ptr<void>(w), w.stride(0), w.stride(1), w.stride(2), experts, inputs, outputs, dtype, ptr<void>(packed), ptr<void>(scales),
                          ptr<void>(packed_t), ptr<void>(scales_t), stream_of(w)));
  return {packed, scales, packed_t, scales_t};
}
// codes [experts, inputs, outputs] and scales [experts, input blocks, output blocks]
std::tuple<Tensor, Tensor> pack_8bit(const Tensor& codes_, const Tensor& scales_) {
  need_gpu(codes_), need_gpu(scales_);
  require(codes_.dim() == 3 && scales_.dim() == 3 && codes_.numel() > 0, "pack_8bit: codes [experts, inputs, outputs], scales [experts, input blocks, output blocks]");
  if (codes_.scalar_type() != at::kFloat8_e4m3fn)
    raise(PyExc_NotImplementedError, std::string("stk_amd: 8-bit codes are float8_e4m3fn, got ") + c10::toString(codes_.scalar_type()));
  const bool float_scales = scales_.scalar_type() == at::kFloat;
  if (!float_scales && scales_.scalar_type() != at::kFloat8_e8m0fnu)
    raise(PyExc_NotImplementedError, std::string("stk_amd: 8-bit weights have scales of float32 or float8_e8m0fnu, got ") + c10::toString(scales_.scalar_type()));
  const c10::DeviceGuard guard(codes_.device());
  const int64_t experts = codes_.size(0), inputs = codes_.size(1), outputs = codes_.size(2);
  require(scales_.size(0) == experts && scales_.size(1) == (inputs + 127) / 128 && scales_.size(2) == (outputs + 127) / 128 && scales_.device() == codes_.device(),
          "pack_8bit: one scale for every block of 128 inputs and 128 outputs");
  const Tensor codes = codes_.contiguous(), scales = scales_.detach().contiguous();
  const auto bytes = codes.options().dtype(at::kByte);
  Tensor packed = at::empty({experts, stk_8bit_piece_bytes(1, inputs, outputs)}, bytes);
  const int64_t size = stk_8bit_scale_bytes(1, inputs, outputs, float_scales);
  Tensor packed_scales = float_scales ? at::empty({experts, size / 4}, scales.options()) : at::empty({experts, size}, bytes);
  check(stk_pack_8bit(ptr<uint8_t>(codes), ptr<void>(scales), float_scales, experts, inputs, outputs, ptr<void>(packed), ptr<void>(packed_scales), stream_of(codes)));
  return {packed, packed_scales};
}
// Packed weights as the calls take them: what pack_8bit or quantize_8bit made.
struct Packed8 {
  int64_t experts, inputs, outputs;
  bool float_scales;
  Packed8(const Tensor& packed, const Tensor& scales, int64_t inputs_, int64_t outputs_) : experts(0), inputs(inputs_), outputs(outputs_), float_scales(false) {
    need_gpu(packed), need_gpu(scales);
    float_scales = scales.scalar_type() == at::kFloat;
    require(packed.dim() == 2 && packed.scalar_type() == at::kByte && packed.is_contiguous() && scales.is_contiguous() && inputs > 0 && outputs > 0 &&
                (float_scales || scales.scalar_type() == at::kByte) && scales.device() == packed.device(),
            "packed 8-bit weights come from pack_8bit or quantize_8bit");
    experts = packed.size(0);
    require(packed.numel() == stk_8bit_piece_bytes(experts, inputs, outputs) &&
                scales.numel() * (float_scales ? 4 : 1) == stk_8bit_scale_bytes(experts, inputs, outputs, float_scales),
            "packed 8-bit weights come from pack_8bit or quantize_8bit");
  }
};
#define PACKED8_ARGS const Tensor &packed, const Tensor &scales, int64_t inputs, int64_t outputs
Tensor dequantize_8bit(PACKED8_ARGS, at::ScalarType dtype) {
  const Packed8 w(packed, scales, inputs, outputs);
  const c10::DeviceGuard guard(packed.device());
  Tensor out = at::empty({w.experts, inputs, outputs}, packed.options().dtype(dtype));
  check(stk_dequantize_8bit(ptr<void>(packed), ptr<void>(scales), w.float_scales, w.experts, inputs, outputs, ptr<void>(out), value_dtype(out), stream_of(packed)));
  return out;
}
// Rows of the products: `inputs` 16-bit values, next to each other.
Tensor rows8(const Tensor& x_, const Tensor& packed, int64_t inputs) {
  need_gpu(x_);
  require(x_.dim() == 2 && x_.size(1) == inputs, "incompatible dimensions");
  require(x_.device() == packed.device(), "operands are on one device");
  if (x_.scalar_type() != at::kHalf && x_.scalar_type() != at::kBFloat16)
    raise(PyExc_NotImplementedError, std::string("stk_amd: rows for 8-bit weights are float16 or bfloat16, got ") + c10::toString(x_.scalar_type()));
  const Tensor x = x_.detach();
  return (inputs == 1 || x.stride(1) == 1) && x.stride(0) >= 0 ? x : x.contiguous();
}
Tensor bytes_like(const Tensor& t, size_t bytes) { return at::empty({(int64_t)bytes}, t.options().dtype(at::kByte)); }
Tensor matmul_8bit(const Tensor& x_, PACKED8_ARGS, int activation) {
  const Packed8 w(packed, scales, inputs, outputs);
  require(w.experts == 1, "matmul_8bit: the weights of one matrix");
  const c10::DeviceGuard guard(packed.device());
  const Tensor x = rows8(x_, packed, inputs);
  const int64_t rows = x.size(0);
  Tensor out = at::empty({rows, outputs}, x.options());
  const size_t bytes = stk_matmul_8bit_workspace_bytes(rows, rows, 1, inputs, outputs);
  const Tensor ws = bytes_like(x, bytes);
  check(stk_matmul_8bit(ptr<void>(x), rows, x.stride(0), ptr<void>(packed), ptr<void>(scales), w.float_scales, inputs, outputs, ptr<void>(out), outputs, activation,
                        value_dtype(x), ptr<void>(ws), bytes, stream_of(x)));
  return out;
}
void check_routing8(const Tensor& indices, const Tensor& bins, const Packed8& w, const Tensor& packed) {
  need_gpu(indices), need_gpu(bins);
  for (const Tensor* t : {&indices, &bins})
    require(t->scalar_type() == at::kInt && t->is_contiguous() && t->device() == packed.device(), "the routing's arrays come from route");
  require(bins.numel() == w.experts, "one bin for each expert's weights");
}
Tensor gather_matmul_8bit(const Tensor& x_, const Tensor& indices, const Tensor& bins, int top_k, PACKED8_ARGS, int activation) {
  const Packed8 w(packed, scales, inputs, outputs);
  check_routing8(indices, bins, w, packed);
  const c10::DeviceGuard guard(packed.device());
  const Tensor x = rows8(x_, packed, inputs);
  const int64_t slots = indices.numel();
  require(top_k >= 1 && x.size(0) * top_k == slots, "one row per token");
  Tensor out = at::empty({slots, outputs}, x.options());
  const size_t bytes = stk_matmul_8bit_workspace_bytes(x.size(0), slots, w.experts, inputs, outputs);
  const Tensor ws = bytes_like(x, bytes);
  check(stk_gather_matmul_8bit(ptr<void>(x), x.size(0), x.stride(0), ptr<int32_t>(indices), ptr<int32_t>(bins), top_k, ptr<void>(packed), ptr<void>(scales),
                               w.float_scales, w.experts, inputs, outputs, ptr<void>(out), outputs, activation, value_dtype(x), ptr<void>(ws), bytes, stream_of(x)));
  return out;
}
Tensor matmul_8bit_scatter(const Tensor& x_, const Tensor& indices, const Tensor& bins, int top_k, PACKED8_ARGS, const OptTensor& weights) {
  const Packed8 w(packed, scales, inputs, outputs);
  check_routing8(indices, bins, w, packed);
  const c10::DeviceGuard guard(packed.device());
  const Tensor x = rows8(x_, packed, inputs);
  const int64_t slots = indices.numel();
  require(top_k >= 1 && slots % top_k == 0 && x.size(0) == slots, "one row per slot");
  const OptTensor by_slot = weights32(weights, slots);
  require(!by_slot || by_slot->device() == x.device(), "operands are on one device");
  Tensor out = at::empty({slots / top_k, outputs}, x.options());
  const size_t bytes = stk_matmul_8bit_scatter_workspace_bytes(slots, top_k, w.experts, inputs, outputs);
  const Tensor ws = bytes_like(x, bytes);
  check(stk_matmul_8bit_scatter(ptr<void>(x), x.stride(0), ptr<int32_t>(indices), ptr<int32_t>(bins), top_k, slots / top_k, ptr<float>(by_slot), ptr<void>(packed),
                                ptr<void>(scales), w.float_scales, w.experts, inputs, outputs, ptr<void>(out), outputs, value_dtype(x), ptr<void>(ws), bytes, stream_of(x)));
  return out;
}

// ------------------------------------------------------------------------------------------------ training with 8-bit products
typedef std::vector<OptTensor> Saved;
// Rows quantised along their values (codes, exponents) and, as rows or pieces, down the columns.
struct Quantised8 {
  Tensor codes, exponents, columns, column_exponents;
  Quantised8(const Rows& x, bool along, bool down, bool pieces) {
    const auto bytes = x.t.options().dtype(at::kByte);
    if (along) codes = at::empty({stk_8bit_row_bytes(x.rows, x.size)}, bytes), exponents = at::empty({stk_8bit_exponent_bytes(x.rows, x.size)}, bytes);
    if (down) {
      columns = at::empty({pieces ? stk_8bit_piece_bytes(1, x.rows, x.size) : stk_8bit_row_bytes(x.size, x.rows)}, bytes);
      column_exponents = at::empty({pieces ? stk_8bit_scale_bytes(1, x.rows, x.size, 0) : stk_8bit_exponent_bytes(x.size, x.rows)}, bytes);
    }
    const auto at = [](const Tensor& t) { return t.defined() ? ptr<void>(t) : nullptr; };
    if (x.rows > 0 && (along || down))
      check(stk_quantize_rows_8bit(ptr<void>(x.t), x.rows, x.size, x.stride, value_dtype(x.t), at(codes), at(exponents), at(columns), at(column_exponents), pieces,
                                   stream_of(x.t)));
  }
};
// y of x [..., inputs] and weights [inputs, outputs] or, with the bins of the padded layout, [experts, inputs, outputs]; then what the backward pass
// takes: the columns of x and their exponents where the gradient of the weights is wanted, the transposed weights where that of x is.
std::tuple<Tensor, Saved> linear_8bit_forward(const Tensor& x_, const Tensor& w_, const OptTensor& bins, bool want_x, bool want_w) {
  need_gpu(x_), need_gpu(w_);
  require(x_.dim() >= 1 && (bins ? x_.dim() == 2 && w_.dim() == 3 : w_.dim() == 2), "linear_8bit: x [..., inputs] and w [inputs, outputs], or the rows of a routing and w [experts, inputs, outputs]");
  const int64_t inputs = w_.size(-2), outputs = w_.size(-1), experts = bins ? w_.size(0) : 1;
  require(x_.size(-1) == inputs && inputs > 0 && outputs > 0 && experts > 0, "incompatible dimensions");
  require(x_.device() == w_.device(), "operands are on one device");
  if (x_.scalar_type() != w_.scalar_type() || (x_.scalar_type() != at::kHalf && x_.scalar_type() != at::kBFloat16))
    raise(PyExc_NotImplementedError, std::string("stk_amd: linear_8bit takes rows and weights that are both float16 or both bfloat16, got ") +
                                         c10::toString(x_.scalar_type()) + " and " + c10::toString(w_.scalar_type()));
  if (bins) {
    need_gpu(*bins);
    require(bins->scalar_type() == at::kInt && bins->is_contiguous() && bins->device() == x_.device() && bins->numel() == experts,
            "linear_8bit: one bin of the routing for each expert's weights");
  }
  const c10::DeviceGuard guard(x_.device());
  const Rows x(x_);
  auto sizes = x_.sizes().vec();
  sizes.back() = outputs;
  Tensor y = at::empty(sizes, x_.options());
  if (x.rows == 0) return {y, Saved(4)};
  const Quantised8 q(x, true, want_w, false);
  const auto [packed, scales, packed_t, scales_t] = quantize_8bit(bins ? w_ : w_.unsqueeze(0), want_x);
  check(stk_linear_8bit(ptr<void>(q.codes), ptr<void>(q.exponents), x.rows, ptr<int32_t>(bins), ptr<void>(packed), ptr<void>(scales), experts, inputs, outputs,
                        ptr<void>(y), outputs, value_dtype(x_), stream_of(x_)));
  Saved saved(4);
  if (want_w) saved[0] = q.columns, saved[1] = q.column_exponents;
  if (want_x) saved[2] = packed_t, saved[3] = scales_t;
  return {y, saved};
}
// (dx, dw), those that are wanted.
std::tuple<OptTensor, OptTensor> linear_8bit_backward(const Tensor& grad_, const Saved& saved, const OptTensor& bins, at::IntArrayRef x_sizes, at::IntArrayRef w_sizes,
                                                      bool want_x, bool want_w) {
  need_gpu(grad_);
  const c10::DeviceGuard guard(grad_.device());
  const Rows g(grad_);
  const int64_t inputs = w_sizes[w_sizes.size() - 2], outputs = w_sizes.back(), experts = bins ? w_sizes[0] : 1;
  OptTensor dx, dw;
  if (want_x) dx = at::empty(x_sizes, grad_.options());
  if (g.rows == 0) {
    if (want_w) dw = at::zeros(w_sizes, grad_.options());
    return {dx, dw};
  }
  const Quantised8 q(g, want_x, want_w, true);
  if (want_x)
    check(stk_linear_8bit(ptr<void>(q.codes), ptr<void>(q.exponents), g.rows, ptr<int32_t>(bins), ptr<void>(saved[2]), ptr<void>(saved[3]), experts, outputs, inputs,
                          ptr<void>(dx), inputs, value_dtype(grad_), stream_of(grad_)));
  if (want_w) {
    dw = at::empty(w_sizes, grad_.options());
    check(stk_weight_gradient_8bit(ptr<void>(saved[0]), ptr<void>(saved[1]), ptr<void>(q.columns), ptr<void>(q.column_exponents), g.rows, ptr<int32_t>(bins), experts,
                                   inputs, outputs, ptr<void>(dw), value_dtype(grad_), stream_of(grad_)));
  }
  return {dx, dw};
}
struct Linear8 : torch::autograd::Function<Linear8> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptTensor& bins) {
    auto [y, saved] = linear_8bit_forward(x, w, bins, x.requires_grad(), w.requires_grad());
    torch::autograd::variable_list keep;
    for (const OptTensor& t : saved) keep.push_back(t ? *t : Tensor());
    keep.push_back(bins ? *bins : Tensor());
    ctx->save_for_backward(keep);
    ctx->saved_data["x"] = x.sizes(), ctx->saved_data["w"] = w.sizes();
    return y;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto kept = ctx->get_saved_variables();
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor()};
    Saved saved;
    for (size_t i = 0; i < 4; i++) saved.push_back(kept[i].defined() ? OptTensor(kept[i]) : OptTensor());
    const OptTensor bins = kept[4].defined() ? OptTensor(kept[4]) : OptTensor();
    const auto x_sizes = ctx->saved_data["x"].toIntVector(), w_sizes = ctx->saved_data["w"].toIntVector();
    const auto [dx, dw] = linear_8bit_backward(grads[0], saved, bins, x_sizes, w_sizes, ctx->needs_input_grad(0), ctx->needs_input_grad(1));
    return once_differentiable({dx.value_or(Tensor()), dw.value_or(Tensor()), Tensor()}, "linear_8bit");
  }
};
Tensor linear_8bit_graph(const Tensor& x, const Tensor& w, const OptTensor& bins) {
  if (at::GradMode::is_enabled() && (x.requires_grad() || w.requires_grad())) return Linear8::apply(x, w, bins);
  return std::get<0>(linear_8bit_forward(x, w, bins, false, false));
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("abi_version", [] { return STK_AMD_ABI_VERSION; });
  m.def("sdd", &sdd, py::call_guard<py::gil_scoped_release>());
  m.def("dsd", &dsd, py::call_guard<py::gil_scoped_release>());
  m.def("dds", &dds, py::call_guard<py::gil_scoped_release>());
  m.def("dsd_dds", &dsd_dds, py::call_guard<py::gil_scoped_release>());
  m.def("dsd_dsd", &dsd_dsd, py::call_guard<py::gil_scoped_release>());
  m.def("sdd_dsd", &sdd_dsd, py::call_guard<py::gil_scoped_release>());
  m.def("build_plan", &build_plan, py::call_guard<py::gil_scoped_release>());
  m.def("capture_id", &capture_id, py::call_guard<py::gil_scoped_release>());
  m.def("follow", &follow, py::call_guard<py::gil_scoped_release>());
  m.def("row_indices", &row_indices, py::call_guard<py::gil_scoped_release>());
  m.def("transpose_meta", &transpose_meta, py::call_guard<py::gil_scoped_release>());
  m.def("dmoe_topology", &dmoe_topology, py::call_guard<py::gil_scoped_release>());
  m.def("to_dense", &to_dense, py::call_guard<py::gil_scoped_release>());
  m.def("to_sparse", &to_sparse, py::call_guard<py::gil_scoped_release>());
  m.def("activation_product", &activation_product, py::call_guard<py::gil_scoped_release>());
  m.def("route", &route, py::call_guard<py::gil_scoped_release>());
  m.def("padded_gather", &padded_gather, py::call_guard<py::gil_scoped_release>());
  m.def("padded_scatter", &padded_scatter, py::call_guard<py::gil_scoped_release>());
  m.def("padded_scatter_weight_gradient", &padded_scatter_weight_gradient, py::call_guard<py::gil_scoped_release>());
  m.def("sdd_gather", &sdd_gather, py::call_guard<py::gil_scoped_release>());
  m.def("sdd_gather_reads_plan", &stk_sdd_gather_reads_plan);
  m.def("dsd_scatter_few_case", &dsd_scatter_few_case);
  m.def("dsd_scatter_few", &dsd_scatter_few, py::call_guard<py::gil_scoped_release>());
  m.def("dsd_scatter", &dsd_scatter, py::call_guard<py::gil_scoped_release>());
  m.def("layer_norm", &layer_norm, py::call_guard<py::gil_scoped_release>());
  m.def("layer_norm_graph", &layer_norm_graph, py::call_guard<py::gil_scoped_release>());
  m.def("layer_norm_backward", &layer_norm_backward, py::call_guard<py::gil_scoped_release>());
  m.def("top_experts", &top_experts, py::call_guard<py::gil_scoped_release>());
  m.def("top_experts_graph", &top_experts_graph, py::call_guard<py::gil_scoped_release>());
  m.def("top_experts_backward", &top_experts_backward, py::call_guard<py::gil_scoped_release>());
  m.def("quantize_4bit", &quantize_4bit, py::call_guard<py::gil_scoped_release>());
  m.def("pack_4bit", &pack_4bit, py::call_guard<py::gil_scoped_release>());
  m.def("dequantize_4bit", &dequantize_4bit, py::call_guard<py::gil_scoped_release>());
  m.def("matmul_4bit", &matmul_4bit, py::call_guard<py::gil_scoped_release>());
  m.def("gather_matmul_4bit", &gather_matmul_4bit, py::call_guard<py::gil_scoped_release>());
  m.def("matmul_4bit_scatter", &matmul_4bit_scatter, py::call_guard<py::gil_scoped_release>());
  m.def("group_top_experts", &group_top_experts, py::call_guard<py::gil_scoped_release>());
  m.def("group_top_experts_graph", &group_top_experts_graph, py::call_guard<py::gil_scoped_release>());
  m.def("group_top_experts_backward", &group_top_experts_backward, py::call_guard<py::gil_scoped_release>());
  m.def("quantize_8bit", &quantize_8bit, py::call_guard<py::gil_scoped_release>());
  m.def("pack_8bit", &pack_8bit, py::call_guard<py::gil_scoped_release>());
  m.def("dequantize_8bit", &dequantize_8bit, py::call_guard<py::gil_scoped_release>());
  m.def("matmul_8bit", &matmul_8bit, py::call_guard<py::gil_scoped_release>());
  m.def("gather_matmul_8bit", &gather_matmul_8bit, py::call_guard<py::gil_scoped_release>());
  m.def("matmul_8bit_scatter", &matmul_8bit_scatter, py::call_guard<py::gil_scoped_release>());
  m.def("linear_8bit_graph", &linear_8bit_graph, py::call_guard<py::gil_scoped_release>());
  m.def("linear_8bit_forward", &linear_8bit_forward, py::call_guard<py::gil_scoped_release>());
  m.def("linear_8bit_backward", [](const Tensor& grad, const Saved& saved, const OptTensor& bins, const std::vector<int64_t>& x_sizes, const std::vector<int64_t>& w_sizes,
                                   bool want_x, bool want_w) { return linear_8bit_backward(grad, saved, bins, x_sizes, w_sizes, want_x, want_w); },
        py::call_guard<py::gil_scoped_release>());
}
