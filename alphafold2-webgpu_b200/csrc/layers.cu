// layers.cu -- entry points of the layers with learned weights (the dense
// layer and the gated transition, forward and backward) and of the gradient
// norm: argument checks, scratch, and the hand-over to the launchers in
// dense.cu and gradients.cu.
//
// No counterpart in the reference, which runs fixed weights forward only; the
// checks follow its conventions (positive safe integers, a RangeError-class
// status with the reason in the message).
#include <algorithm>
#include <cmath>
#include <new>
#include <string>
#include <vector>

#include "af2_internal.h"

namespace af2 {

// Calls on one stream need no order among themselves.  A call on another stream waits for an event
// after the last use: recorded then and there if that use was on a stream that lives as long as the
// context (its own and the legacy default stream, which nothing captures either), else after each use.
bool LayerScratch::lasting(cudaStream_t s) const { return s == ctx_->stream || s == cudaStreamLegacy; }

af2_status LayerScratch::acquire(void *workspace, size_t bytes) {
  if (workspace) {
    base_ = static_cast<uint8_t *>(workspace);
    return AF2_OK;
  }
  if (bytes == 0) return AF2_OK;
  if (!ctx_->layer_done) {
    cudaError_t e = cudaEventCreateWithFlags(&ctx_->layer_done, cudaEventDisableTiming);
    if (e != cudaSuccess) {
      ctx_->layer_done = nullptr;
      return cuda_fail(ctx_, e, "create the layer scratch's event");
    }
  }
  // A graph would keep the buffer's address, which the next call that needs more frees, and nothing would
  // order its replays with other calls.
  if (!lasting(stream_)) {
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    if (cudaError_t e = cudaStreamIsCapturing(stream_, &capture); e != cudaSuccess)
      return cuda_fail(ctx_, e, "query the stream's capture");
    if (capture != cudaStreamCaptureStatusNone)
      return fail(ctx_, AF2_ERR_UNSUPPORTED, "a call inside a stream capture cannot use the context's scratch; pass a "
                                             "workspace that the graph's owner keeps");
  }
  const bool grow = ctx_->layer_scratch.bytes < bytes;
  use_ = {stream_, 0, lasting(stream_)};
  if (!use_.lasting)
    if (cudaError_t e = cudaStreamGetId(stream_, &use_.id); e != cudaSuccess)
      return cuda_fail(ctx_, e, "query the stream's id");
  // earlier calls may still use the buffer: this one follows them, or the host does before it is freed
  const cudaError_t ordered = order_scratch(
      ctx_->layer_use, use_, grow,
      [&](const void *last) {
        return cudaEventRecord(ctx_->layer_done, static_cast<cudaStream_t>(const_cast<void *>(last)));
      },
      [&] { return cudaStreamWaitEvent(stream_, ctx_->layer_done, 0); },
      [&] { return cudaEventSynchronize(ctx_->layer_done); });
  if (ordered != cudaSuccess) return cuda_fail(ctx_, ordered, "order the layer scratch between streams");
  if (grow)
    if (af2_status st = ensure(ctx_, ctx_->layer_scratch, bytes, "layer scratch"); st != AF2_OK) return st;
  base_ = static_cast<uint8_t *>(ctx_->layer_scratch.ptr);
  owned_ = true;
  return AF2_OK;
}

af2_status LayerScratch::release() {
  if (!owned_) return AF2_OK;
  ctx_->layer_use = use_;
  if (use_.lasting) return AF2_OK;
  if (cudaError_t e = cudaEventRecord(ctx_->layer_done, stream_); e != cudaSuccess)
    return cuda_fail(ctx_, e, "record the layer scratch's use");
  return AF2_OK;
}

namespace {

constexpr int64_t kMaxRows = (int64_t(1) << 31) - 1024, kMaxWidth = 65536;

bool known_dtype(int dtype) { return dtype == AF2_F32 || dtype == AF2_F16 || dtype == AF2_BF16; }
size_t element_bytes(int dtype) { return dtype == AF2_F32 ? 4 : 2; }

// No exception leaves a C entry.
template <typename F>
af2_status guarded(af2_ctx *ctx, F &&f) {
  try {
    return f();
  } catch (const std::bad_alloc &) {
    return AF2_ERR_OUT_OF_MEMORY;
  } catch (...) {
    return AF2_ERR_CUDA;
  }
}

af2_status check_sizes(af2_ctx *ctx, int64_t rows, int64_t a, int64_t b, int dtype, const char *what) {
  if (rows < 0 || a <= 0 || b <= 0)
    return fail(ctx, AF2_ERR_INVALID_ARGUMENT,
                std::string(what) + " widths must be positive and its rows not negative; received " +
                    std::to_string(rows) + " rows, " + std::to_string(a) + " and " + std::to_string(b));
  if (!known_dtype(dtype)) return fail(ctx, AF2_ERR_INVALID_ARGUMENT, "dtype must be AF2_F32, AF2_F16 or AF2_BF16");
  if (rows > kMaxRows || a > kMaxWidth || b > kMaxWidth)
    return fail(ctx, AF2_ERR_UNSUPPORTED, std::string(what) + " beyond 2^31 - 1024 rows or widths of 65536");
  return AF2_OK;
}

af2_status check_activation(af2_ctx *ctx, int activation) {
  if (activation < AF2_ACTIVATION_NONE || activation > AF2_ACTIVATION_GELU)
    return fail(ctx, AF2_ERR_INVALID_ARGUMENT, "unknown activation " + std::to_string(activation));
  return AF2_OK;
}

struct NamedTensor {
  const char *name;
  const void *ptr;
  bool required;
};

// Required tensors are there, and each is aligned to its element.
template <int N>
af2_status check_tensors(af2_ctx *ctx, const NamedTensor (&tensors)[N], int dtype) {
  for (const NamedTensor &t : tensors) {
    if (!t.ptr && t.required) return fail(ctx, AF2_ERR_INVALID_ARGUMENT, std::string(t.name) + " is NULL");
    if (reinterpret_cast<uintptr_t>(t.ptr) % element_bytes(dtype) != 0)
      return fail(ctx, AF2_ERR_INVALID_ARGUMENT, std::string(t.name) + " is not aligned to its element type");
  }
  return AF2_OK;
}

af2_status check_block(af2_ctx *ctx, const void *ptr, const char *name) {
  if (reinterpret_cast<uintptr_t>(ptr) % 256 != 0)
    return fail(ctx, AF2_ERR_INVALID_ARGUMENT, std::string(name) + " must be 256-byte aligned");
  return AF2_OK;
}

// `rows` rows of `width` elements, `stride` from one to the next.
struct Rows {
  const void *ptr;
  int64_t rows, width, stride;
};

// Whether two tensors of one type share an element: exact for equal strides and where one has no gaps;
// otherwise (two with gaps of different sizes) not looked into.
bool overlap(const Rows &a, const Rows &b, size_t size) {
  if (!a.ptr || !b.ptr || a.rows == 0 || b.rows == 0) return false;
  const int64_t pa = static_cast<int64_t>(reinterpret_cast<uintptr_t>(a.ptr) / size),
                pb = static_cast<int64_t>(reinterpret_cast<uintptr_t>(b.ptr) / size);
  const int64_t end_a = pa + (a.rows - 1) * a.stride + a.width, end_b = pb + (b.rows - 1) * b.stride + b.width;
  if (pa >= end_b || pb >= end_a) return false;
  auto has_gaps = [](const Rows &r) { return r.rows > 1 && r.stride != r.width; };
  // a row of r that reaches past `from` and begins before `to`
  auto row_between = [](const Rows &r, int64_t p, int64_t from, int64_t to) {
    const int64_t before = from - p - r.width;  // rows that begin at p + k stride <= p + before end at or before `from`
    const int64_t first = before < 0 ? 0 : before / r.stride + 1;
    return first < r.rows && p + first * r.stride < to;
  };
  if (!has_gaps(a)) return row_between(b, pb, pa, end_a);
  if (!has_gaps(b)) return row_between(a, pa, pb, end_b);
  if (a.stride != b.stride) return false;
  // rows k of a and k - q, k - q - 1 of b are neighbours
  int64_t q = (pb - pa) / a.stride, column = (pb - pa) % a.stride;
  if (column < 0) column += a.stride, --q;
  auto meet = [&](int64_t shift) { return shift < a.rows && shift + b.rows > 0; };
  return (column < a.width && meet(q)) || (column + b.width > a.stride && meet(q + 1));
}

// Blocks write `out` while others read: it may overlap no input, but be the same rows as one of `same`.
template <int M, int N>
af2_status check_out(af2_ctx *ctx, const Rows &out, const Rows (&same)[M], const Rows (&inputs)[N], int dtype) {
  const size_t size = element_bytes(dtype);
  for (const Rows &in : inputs)
    if (overlap(out, in, size)) return fail(ctx, AF2_ERR_INVALID_ARGUMENT, "out overlaps an input");
  for (const Rows &in : same)
    if (overlap(out, in, size) && !(out.ptr == in.ptr && (out.stride == in.stride || out.rows == 1)))
      return fail(ctx, AF2_ERR_INVALID_ARGUMENT, "out overlaps an input without being it");
  return AF2_OK;
}

struct Strides {
  int activation = AF2_ACTIVATION_NONE;
  int64_t x = 0, residual = 0, out = 0, d_x = 0;
};

af2_status read_options(af2_ctx *ctx, const af2_layer_options *o, int64_t x_width, int64_t out_width, bool residual,
                        bool backward, Strides *s) {
  s->x = s->d_x = x_width;
  s->residual = s->out = out_width;
  if (!o) return AF2_OK;
  if (af2_status st = check_activation(ctx, o->activation); st != AF2_OK) return st;
  if (o->reserved != 0) return fail(ctx, AF2_ERR_INVALID_ARGUMENT, "the reserved option must be 0");
  const struct { const char *name; int64_t value, width; bool used; } strides[4] = {
      {"x_stride", o->x_stride, x_width, true},
      {"residual_stride", o->residual_stride, out_width, residual},
      {"out_stride", o->out_stride, out_width, true},
      {"d_x_stride", o->d_x_stride, x_width, backward}};
  for (const auto &v : strides)
    if (v.used && (v.value < v.width || v.value > (int64_t(1) << 40)))
      return fail(ctx, AF2_ERR_INVALID_ARGUMENT, std::string(v.name) + " " + std::to_string(v.value) +
                                                     " is outside the rows' width " + std::to_string(v.width) +
                                                     " to 2^40");
  s->activation = o->activation;
  s->x = o->x_stride;
  s->residual = o->residual_stride;
  s->out = o->out_stride;
  s->d_x = o->d_x_stride;
  return AF2_OK;
}

// Runs `pass` (see dense_forward) on p with the call's scratch.
template <typename P>
af2_status run_pass(af2_ctx *ctx, void *workspace, cudaStream_t stream, const P &p,
                    af2_status (*pass)(af2_ctx *, const P &, void *, uint64_t *, cudaStream_t)) {
  uint64_t bytes = 0;
  if (!workspace)
    if (af2_status st = pass(nullptr, p, nullptr, &bytes, stream); st != AF2_OK) return st;
  LayerScratch scratch(ctx, stream);
  if (af2_status st = scratch.acquire(workspace, bytes); st != AF2_OK) return st;
  const af2_status st = pass(ctx, p, scratch.base(), &bytes, stream);
  const af2_status rel = scratch.release();
  return st != AF2_OK ? st : rel;
}

// Stands for a tensor at an unknown address when scratch is sized: one that TMA cannot read in place.
void *const kAnywhere = reinterpret_cast<void *>(uintptr_t(4));

// The scratch of a backward pass whichever gradients are wanted.  Fewer products are planned otherwise
// than all of them -- alone, one has its depth cut further, and more split sums -- so each set of
// products is counted (everything else only grows with what is wanted): count(set, bytes) for the sets
// below `sets`.  Kept by shape, since that is up to twelve plans and a call with a caller's workspace asks.
template <typename F>
af2_status largest_set(const int64_t (&shape)[6], int sets, uint64_t *bytes, F &&count) {
  struct Kept {
    int64_t shape[6];  // [0] is not 0
    uint64_t bytes;
  };
  static thread_local Kept table[64];
  uint64_t hash = 0;
  for (int64_t v : shape) hash = (hash ^ static_cast<uint64_t>(v)) * 0x9e3779b97f4a7c15ull;
  Kept &kept = table[hash >> 58];
  if (!std::equal(shape, shape + 6, kept.shape)) {
    uint64_t most = 0;
    for (int set = 0; set < sets; ++set) {
      uint64_t n = 0;
      if (af2_status st = count(set, &n); st != AF2_OK) return st;
      most = std::max(most, n);
    }
    std::copy(shape, shape + 6, kept.shape);
    kept.bytes = most;
  }
  *bytes = kept.bytes;
  return AF2_OK;
}

cudaStream_t stream_of(af2_ctx *ctx, void *stream) {
  return stream ? static_cast<cudaStream_t>(stream) : ctx->stream;
}

// (The message is put together for a tensor that fails only: a set has hundreds.)
af2_status check_set(af2_ctx *ctx, const af2_tensor_ref *t, int64_t count, const char *what) {
  for (int64_t i = 0; i < count; ++i) {
    std::string wrong;
    if (!known_dtype(t[i].dtype))
      wrong = ": dtype must be AF2_F32, AF2_F16 or AF2_BF16";
    else if (t[i].count < 0 || t[i].count > (int64_t(1) << 44))
      wrong = " has " + std::to_string(t[i].count) + " elements";
    else if (t[i].count > 0 && !t[i].data)
      wrong = " is NULL";
    else if (reinterpret_cast<uintptr_t>(t[i].data) % element_bytes(t[i].dtype) != 0)
      wrong = " is not aligned to its element type";
    if (!wrong.empty())
      return fail(ctx, AF2_ERR_INVALID_ARGUMENT, std::string(what) + " " + std::to_string(i) + wrong);
  }
  return AF2_OK;
}

// What is written overlaps nothing else that is written, and no tensor but, as the same memory, its own:
// blocks scale their parts of the set in no order.  Parts of one buffer in their order, read from elsewhere
// or in place, need no table (384 tensors: 4 us less).
af2_status check_overlaps(af2_ctx *ctx, const af2_tensor_ref *tensors, const af2_tensor_ref *outputs, int64_t count) {
  const af2_tensor_ref *const out = outputs ? outputs : tensors;
  auto end_of = [](const af2_tensor_ref &t) {
    return reinterpret_cast<uintptr_t>(t.data) + t.count * element_bytes(t.dtype);
  };
  uintptr_t low = UINTPTR_MAX, high = 0;
  bool simple = true;  // in order, and no input between the first and the last
  for (int64_t i = 0; i < count && simple; ++i)
    if (out[i].count > 0) {
      const uintptr_t begin = reinterpret_cast<uintptr_t>(out[i].data);
      low = std::min(low, begin);
      simple = begin >= high;
      high = end_of(out[i]);
    }
  for (int64_t i = 0; outputs && i < count && simple; ++i)
    simple = tensors[i].count == 0 || reinterpret_cast<uintptr_t>(tensors[i].data) >= high || end_of(tensors[i]) <= low;
  if (simple) return AF2_OK;
  struct Span {
    uintptr_t begin, end;
    int64_t index;
  };
  auto spans = [&](const af2_tensor_ref *t) {
    std::vector<Span> s;
    s.reserve(static_cast<size_t>(count));
    for (int64_t i = 0; i < count; ++i)
      if (t[i].count > 0) s.push_back({reinterpret_cast<uintptr_t>(t[i].data), end_of(t[i]), i});
    std::sort(s.begin(), s.end(), [](const Span &a, const Span &b) { return a.begin < b.begin; });
    return s;
  };
  const std::vector<Span> written = spans(out);
  for (size_t i = 1; i < written.size(); ++i)
    if (written[i].begin < written[i - 1].end)
      return fail(ctx, AF2_ERR_INVALID_ARGUMENT,
                  std::string(outputs ? "outputs " : "tensors ") + std::to_string(written[i - 1].index) + " and " +
                      std::to_string(written[i].index) + " overlap");
  if (!outputs) return AF2_OK;
  size_t first = 0;  // written spans in order do not overlap: their ends are in order too
  for (const Span &t : spans(tensors)) {
    while (first < written.size() && written[first].end <= t.begin) ++first;
    for (size_t i = first; i < written.size() && written[i].begin < t.end; ++i)
      if (written[i].index != t.index || written[i].begin != t.begin)
        return fail(ctx, AF2_ERR_INVALID_ARGUMENT,
                    "output " + std::to_string(written[i].index) + " overlaps tensor " + std::to_string(t.index));
  }
  return AF2_OK;
}

}  // namespace
}  // namespace af2

using namespace af2;

extern "C" {

af2_status af2_dense_saved_bytes(const af2_linear_shape *shape, int dtype, int activation, uint64_t *bytes) {
  return guarded(nullptr, [&]() -> af2_status {
    if (!shape || !bytes) return AF2_ERR_INVALID_ARGUMENT;
    if (af2_status st = check_sizes(nullptr, shape->rows, shape->inner, shape->columns, dtype, ""); st != AF2_OK)
      return st;
    if (af2_status st = check_activation(nullptr, activation); st != AF2_OK) return st;
    *bytes = dense_saved_bytes(shape->rows, shape->columns, dtype, activation);
    return AF2_OK;
  });
}

af2_status af2_dense_workspace_bytes(const af2_linear_shape *shape, int dtype, int activation, int backward,
                                     uint64_t *bytes) {
  return guarded(nullptr, [&]() -> af2_status {
    if (!shape || !bytes) return AF2_ERR_INVALID_ARGUMENT;
    if (af2_status st = check_sizes(nullptr, shape->rows, shape->inner, shape->columns, dtype, ""); st != AF2_OK)
      return st;
    if (af2_status st = check_activation(nullptr, activation); st != AF2_OK) return st;
    void *const any = kAnywhere;
    const int64_t rows = shape->rows, in = shape->inner, cols = shape->columns;
    if (backward)
      return largest_set({1, rows, in, cols, dtype, activation}, 4, bytes, [&](int set, uint64_t *n) {
        return dense_backward(nullptr, {rows, in, cols, dtype, activation, any, any, any, any, cols, in, in,
                                        set & 1 ? any : nullptr, set & 2 ? any : nullptr, any},
                              nullptr, n, nullptr);
      });
    return dense_forward(nullptr, {rows, in, cols, dtype, activation, any, any, any, any, in, cols, cols, any, any},
                         nullptr, bytes, nullptr);
  });
}

af2_status af2_dense(af2_ctx *ctx, const af2_linear_shape *shape, int dtype, const void *x, const void *weight,
                     const void *bias, const void *residual, const af2_layer_options *options, void *out, void *saved,
                     void *workspace, void *stream) {
  if (!ctx) return AF2_ERR_INVALID_ARGUMENT;
  return guarded(ctx, [&]() -> af2_status {
    if (!shape) return fail(ctx, AF2_ERR_INVALID_ARGUMENT, "shape is NULL");
    af2_status st = check_sizes(ctx, shape->rows, shape->inner, shape->columns, dtype, "the dense layer's");
    if (st != AF2_OK) return st;
    const bool some = shape->rows > 0;
    const NamedTensor tensors[] = {{"x", x, some},       {"weight", weight, true},
                                   {"bias", bias, false}, {"residual", residual, false},
                                   {"out", out, some}};
    if ((st = check_tensors(ctx, tensors, dtype)) != AF2_OK) return st;
    Strides s;
    if ((st = read_options(ctx, options, shape->inner, shape->columns, residual != nullptr, false, &s)) != AF2_OK)
      return st;
    if ((st = check_block(ctx, saved, "saved")) != AF2_OK || (st = check_block(ctx, workspace, "workspace")) != AF2_OK)
      return st;
    if (!some) return AF2_OK;
    const int64_t rows = shape->rows, in = shape->inner, columns = shape->columns;
    const Rows same[] = {{residual, rows, columns, s.residual}};
    const Rows inputs[] = {{x, rows, in, s.x}, {weight, in, columns, columns}, {bias, 1, columns, columns}};
    if ((st = check_out(ctx, {out, rows, columns, s.out}, same, inputs, dtype)) != AF2_OK) return st;
    cudaSetDevice(ctx->device);
    const DenseForward p{shape->rows, shape->inner, shape->columns, dtype, s.activation, x,   weight,
                         bias,        residual,     s.x,            s.residual, s.out,  out, saved};
    const cudaStream_t cs = stream_of(ctx, stream);
    return run_pass(ctx, workspace, cs, p, dense_forward);
  });
}

af2_status af2_dense_backward(af2_ctx *ctx, const af2_linear_shape *shape, int dtype, const void *d_out, const void *x,
                              const void *weight, const void *saved, const af2_layer_options *options, void *d_x,
                              void *d_weight, void *d_bias, void *workspace, void *stream) {
  if (!ctx) return AF2_ERR_INVALID_ARGUMENT;
  return guarded(ctx, [&]() -> af2_status {
    if (!shape) return fail(ctx, AF2_ERR_INVALID_ARGUMENT, "shape is NULL");
    af2_status st = check_sizes(ctx, shape->rows, shape->inner, shape->columns, dtype, "the dense layer's");
    if (st != AF2_OK) return st;
    Strides s;
    if ((st = read_options(ctx, options, shape->inner, shape->columns, false, d_x != nullptr, &s)) != AF2_OK)
      return st;
    const bool some = shape->rows > 0;
    const NamedTensor tensors[] = {
        {"d_out", d_out, some},
        {"x", x, some && d_weight},
        {"weight", weight, some && d_x},
        {"saved", saved, some && s.activation != AF2_ACTIVATION_NONE},
        {"d_x", d_x, false},
        {"d_weight", d_weight, false},
        {"d_bias", d_bias, false}};
    if ((st = check_tensors(ctx, tensors, dtype)) != AF2_OK) return st;
    if ((st = check_block(ctx, saved, "saved")) != AF2_OK || (st = check_block(ctx, workspace, "workspace")) != AF2_OK)
      return st;
    cudaSetDevice(ctx->device);
    const DenseBackward p{shape->rows, shape->inner, shape->columns, dtype, s.activation, d_out, x,       weight,
                          saved,       s.out,        s.x,            s.d_x, d_x,          d_weight, d_bias};
    const cudaStream_t cs = stream_of(ctx, stream);
    return run_pass(ctx, workspace, cs, p, dense_backward);
  });
}

af2_status af2_gated_transition_saved_bytes(const af2_transition_shape *shape, int dtype, uint64_t *bytes) {
  return guarded(nullptr, [&]() -> af2_status {
    if (!shape || !bytes) return AF2_ERR_INVALID_ARGUMENT;
    if (af2_status st = check_sizes(nullptr, shape->rows, shape->channels, shape->hidden_channels, dtype, "");
        st != AF2_OK)
      return st;
    *bytes = gated_saved_bytes(shape->rows, shape->hidden_channels, dtype);
    return AF2_OK;
  });
}

af2_status af2_gated_transition_workspace_bytes(const af2_transition_shape *shape, int dtype, int backward,
                                                uint64_t *bytes) {
  return guarded(nullptr, [&]() -> af2_status {
    if (!shape || !bytes) return AF2_ERR_INVALID_ARGUMENT;
    if (af2_status st = check_sizes(nullptr, shape->rows, shape->channels, shape->hidden_channels, dtype, "");
        st != AF2_OK)
      return st;
    void *const any = kAnywhere;
    const int64_t rows = shape->rows, c = shape->channels, h = shape->hidden_channels;
    const af2_gated_weights w{any, any, any, any, any, any};
    if (backward)
      return largest_set({2, rows, c, h, dtype, 0}, 12, bytes, [&](int set, uint64_t *n) {
        // x, the output's weight, and none, one or both of the gate's and the value's
        return gated_backward(nullptr, {rows, c, h, dtype, 0, any, any, any, w,
                                        {set & 1 ? any : nullptr, set >= 4 ? any : nullptr, any,
                                         set >= 8 ? any : nullptr, any, set & 2 ? any : nullptr, any}, c, c, c},
                              nullptr, n, nullptr);
      });
    uint64_t saving = 0;  // the forward pass that saves nothing needs the most
    if (af2_status st = gated_forward(nullptr, {rows, c, h, dtype, 0, any, any, w, c, c, c, any, any}, nullptr, &saving,
                                      nullptr);
        st != AF2_OK)
      return st;
    const af2_status st = gated_forward(nullptr, {rows, c, h, dtype, 0, any, any, w, c, c, c, any, nullptr}, nullptr,
                                        bytes, nullptr);
    if (*bytes < saving) *bytes = saving;
    return st;
  });
}

af2_status af2_gated_transition(af2_ctx *ctx, const af2_transition_shape *shape, int dtype, const void *x,
                                const af2_gated_weights *weights, const void *residual,
                                const af2_layer_options *options, void *out, void *saved, void *workspace,
                                void *stream) {
  if (!ctx) return AF2_ERR_INVALID_ARGUMENT;
  return guarded(ctx, [&]() -> af2_status {
    if (!shape || !weights) return fail(ctx, AF2_ERR_INVALID_ARGUMENT, "shape or weights is NULL");
    af2_status st = check_sizes(ctx, shape->rows, shape->channels, shape->hidden_channels, dtype,
                                "the gated transition's");
    if (st != AF2_OK) return st;
    const bool some = shape->rows > 0;
    const NamedTensor tensors[] = {{"x", x, some},
                                   {"gate_weight", weights->gate_weight, true},
                                   {"gate_bias", weights->gate_bias, false},
                                   {"value_weight", weights->value_weight, true},
                                   {"value_bias", weights->value_bias, false},
                                   {"output_weight", weights->output_weight, true},
                                   {"output_bias", weights->output_bias, false},
                                   {"residual", residual, false},
                                   {"out", out, some}};
    if ((st = check_tensors(ctx, tensors, dtype)) != AF2_OK) return st;
    Strides s;
    if ((st = read_options(ctx, options, shape->channels, shape->channels, residual != nullptr, false, &s)) != AF2_OK)
      return st;
    if ((st = check_block(ctx, saved, "saved")) != AF2_OK || (st = check_block(ctx, workspace, "workspace")) != AF2_OK)
      return st;
    if (!some) return AF2_OK;
    const int64_t rows = shape->rows, c = shape->channels, h = shape->hidden_channels;
    // (x is read into the hidden activations before the same rows of out are written, whichever kernel runs)
    const Rows same[] = {{residual, rows, c, s.residual}, {x, rows, c, s.x}};
    const Rows inputs[] = {{weights->gate_weight, c, h, h},
                           {weights->gate_bias, 1, h, h},
                           {weights->value_weight, c, h, h},
                           {weights->value_bias, 1, h, h},
                           {weights->output_weight, h, c, c},
                           {weights->output_bias, 1, c, c}};
    if ((st = check_out(ctx, {out, rows, c, s.out}, same, inputs, dtype)) != AF2_OK) return st;
    cudaSetDevice(ctx->device);
    const GatedForward p{shape->rows, shape->channels, shape->hidden_channels, dtype, s.activation, x,
                         residual,    *weights,        s.x,                    s.residual, s.out,   out, saved};
    const cudaStream_t cs = stream_of(ctx, stream);
    return run_pass(ctx, workspace, cs, p, gated_forward);
  });
}

af2_status af2_gated_transition_backward(af2_ctx *ctx, const af2_transition_shape *shape, int dtype,
                                         const void *d_out, const void *x, const af2_gated_weights *weights,
                                         const void *saved, const af2_layer_options *options,
                                         const af2_gated_gradients *gradients, void *workspace, void *stream) {
  if (!ctx) return AF2_ERR_INVALID_ARGUMENT;
  return guarded(ctx, [&]() -> af2_status {
    if (!shape || !weights || !gradients)
      return fail(ctx, AF2_ERR_INVALID_ARGUMENT, "shape, weights or gradients is NULL");
    af2_status st = check_sizes(ctx, shape->rows, shape->channels, shape->hidden_channels, dtype,
                                "the gated transition's");
    if (st != AF2_OK) return st;
    const bool some = shape->rows > 0;
    const NamedTensor tensors[] = {{"d_out", d_out, some},
                                   {"x", x, some},
                                   {"saved", saved, some},
                                   {"gate_weight", weights->gate_weight, some},
                                   {"value_weight", weights->value_weight, some},
                                   {"output_weight", weights->output_weight, some},
                                   {"the gradient of x", gradients->x, false},
                                   {"the gradient of gate_weight", gradients->gate_weight, false},
                                   {"the gradient of gate_bias", gradients->gate_bias, false},
                                   {"the gradient of value_weight", gradients->value_weight, false},
                                   {"the gradient of value_bias", gradients->value_bias, false},
                                   {"the gradient of output_weight", gradients->output_weight, false},
                                   {"the gradient of output_bias", gradients->output_bias, false}};
    if ((st = check_tensors(ctx, tensors, dtype)) != AF2_OK) return st;
    Strides s;
    if ((st = read_options(ctx, options, shape->channels, shape->channels, false, gradients->x != nullptr, &s)) !=
        AF2_OK)
      return st;
    if ((st = check_block(ctx, saved, "saved")) != AF2_OK || (st = check_block(ctx, workspace, "workspace")) != AF2_OK)
      return st;
    cudaSetDevice(ctx->device);
    const GatedBackward p{shape->rows, shape->channels, shape->hidden_channels, dtype, s.activation, d_out, x,
                          saved,       *weights,        *gradients,             s.out, s.x,          s.d_x};
    const cudaStream_t cs = stream_of(ctx, stream);
    return run_pass(ctx, workspace, cs, p, gated_backward);
  });
}

af2_status af2_gradient_norm_workspace_bytes(int64_t count, uint64_t *bytes) {
  if (!bytes || count < 0 || count > (int64_t(1) << 24)) return AF2_ERR_INVALID_ARGUMENT;
  *bytes = gradient_norm_workspace_bytes(count);
  return AF2_OK;
}

static af2_status gradient_call(af2_ctx *ctx, const af2_tensor_ref *tensors, const af2_tensor_ref *outputs,
                                int64_t count, bool clip, double max_norm, float *norm, void *workspace,
                                void *stream) {
  if (!ctx) return AF2_ERR_INVALID_ARGUMENT;
  return guarded(ctx, [&]() -> af2_status {
    if (count < 0 || count > (int64_t(1) << 24))
      return fail(ctx, AF2_ERR_INVALID_ARGUMENT, "the set has " + std::to_string(count) + " tensors");
    if (count > 0 && !tensors) return fail(ctx, AF2_ERR_INVALID_ARGUMENT, "tensors is NULL");
    if (!norm || reinterpret_cast<uintptr_t>(norm) % 4 != 0)
      return fail(ctx, AF2_ERR_INVALID_ARGUMENT, "norm must be an f32 on the device");
    if (clip && (!(max_norm >= 0) || !std::isfinite(max_norm)))
      return fail(ctx, AF2_ERR_INVALID_ARGUMENT, "max_norm must be finite and not negative; received " +
                                                     std::to_string(max_norm));
    af2_status st = check_set(ctx, tensors, count, "tensor");
    if (st != AF2_OK) return st;
    if (outputs) {
      if ((st = check_set(ctx, outputs, count, "output")) != AF2_OK) return st;
      for (int64_t i = 0; i < count; ++i)
        if (outputs[i].count != tensors[i].count || outputs[i].dtype != tensors[i].dtype)
          return fail(ctx, AF2_ERR_INVALID_ARGUMENT,
                      "output " + std::to_string(i) + " differs from its tensor in size or type");
    }
    if (clip && (st = check_overlaps(ctx, tensors, outputs, count)) != AF2_OK) return st;
    if ((st = check_block(ctx, workspace, "workspace")) != AF2_OK) return st;
    cudaSetDevice(ctx->device);
    const cudaStream_t cs = stream_of(ctx, stream);
    LayerScratch scratch(ctx, cs);
    if ((st = scratch.acquire(workspace, gradient_norm_workspace_bytes(count))) != AF2_OK) return st;
    st = gradient_norm_launch(ctx, tensors, outputs, count, clip, static_cast<float>(max_norm), norm, scratch.base(), cs);
    const af2_status rel = scratch.release();
    return st != AF2_OK ? st : rel;
  });
}

af2_status af2_gradient_norm(af2_ctx *ctx, const af2_tensor_ref *tensors, int64_t count, float *norm, void *workspace,
                             void *stream) {
  return gradient_call(ctx, tensors, nullptr, count, false, 0.0, norm, workspace, stream);
}

af2_status af2_clip_gradients(af2_ctx *ctx, const af2_tensor_ref *tensors, const af2_tensor_ref *outputs,
                              int64_t count, double max_norm, float *norm, void *workspace, void *stream) {
  return gradient_call(ctx, tensors, outputs, count, true, max_norm, norm, workspace, stream);
}

}  // extern "C"
