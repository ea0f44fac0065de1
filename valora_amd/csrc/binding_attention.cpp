// Torch binding of the attention block's operators (include/mlora.h): rotary positions into the paged cache, attention over it,
// eviction from it.  Operands are checked here, the work is one call through the C ABI on the current stream of the tensors'
// device.
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <cmath>

#include "binding_common.h"

namespace {

hipStream_t stream_of(const c10::Device &d) { return c10::hip::getCurrentHIPStream(d.index()).stream(); }

void check_on(const at::Tensor &t, const c10::Device &d, const char *name) {
  if (!t.is_cuda()) raise(std::string(name) + " must be a CUDA tensor");
  if (t.device() != d) raise(std::string(name) + " is on " + t.device().str() + ", expected " + d.str());
}

void check_type(const at::Tensor &t, at::ScalarType want, const char *name) {
  if (t.scalar_type() != want)
    raise(std::string("expected scalar type ") + c10::toString(want) + " but found " + c10::toString(t.scalar_type()) + " (" + name + ")");
}

// [rows, heads, head_dim], or [rows, heads * head_dim]: heads and strides in elements
struct Heads {
  char *data;
  int64_t rows, heads, row_stride, head_stride;
};

Heads heads_of(const at::Tensor &t, int64_t head_dim, const char *name) {
  Heads h{static_cast<char *>(t.data_ptr()), t.dim() > 0 ? t.size(0) : 0, 0, 0, 0};
  if (t.dim() == 3 && t.size(2) == head_dim) {
    h.heads = t.size(1);
    h.head_stride = t.stride(1);
  } else if (t.dim() == 2 && t.size(1) % head_dim == 0) {
    h.heads = t.size(1) / head_dim;
    h.head_stride = head_dim;
  } else {
    raise(std::string(name) + " must be [rows, heads, " + std::to_string(head_dim) + "] or [rows, heads * " + std::to_string(head_dim) + "]");
  }
  h.row_stride = t.stride(0);
  if (t.numel() > 0 && t.stride(-1) != 1) raise(std::string(name) + ": elements of a head must be contiguous");
  return h;
}

// heads of a row side by side, as the attention kernels read them
Heads dense_heads(const at::Tensor &t, int64_t head_dim, int64_t heads, const char *name) {
  Heads h = heads_of(t, head_dim, name);
  if (h.heads != heads) raise(std::string(name) + " has " + std::to_string(h.heads) + " heads, the plan " + std::to_string(heads));
  if (heads > 1 && t.numel() > 0 && h.head_stride != head_dim) raise(std::string(name) + ": heads of a row must be contiguous");
  if (h.rows <= 1 && h.row_stride < heads * head_dim) h.row_stride = heads * head_dim;   // (a lone row's stride says nothing)
  return h;
}

void no_kernel(const char *what, const at::Tensor &t) { raise(std::string("No suitable kernel. ") + what + " dtype=" + dtype_name(t)); }

// ---- the 8-bit cache: codes [pages, kv_heads, page_size, head_dim], powers [pages, kv_heads, page_size, 2]; a page is dense --------------
mlora_cache8 cache8_of(const at::Tensor &key_codes, const at::Tensor &value_codes, const at::Tensor &powers, const c10::Device &dev) {
  mlora_cache8 c{};
  const auto page = [&](const at::Tensor &t, at::ScalarType type, const char *name) {
    check_on(t, dev, name);
    check_type(t, type, name);
    if (t.dim() != 4) raise(std::string(name) + " must be [pages, kv_heads, page_size, " + (type == at::kFloat8_e8m0fnu ? "2]" : "head_dim]"));
    int64_t dense = 1;
    for (int i = 3; i >= 1; --i) {
      if (t.size(i) > 1 && t.stride(i) != dense && t.numel() > 0) raise(std::string(name) + ": a page must be contiguous");
      dense *= t.size(i);
    }
    if (t.size(0) > 1 && t.stride(0) < dense) raise(std::string(name) + ": pages overlap");
    return t.size(0) > 1 ? t.stride(0) : dense;
  };
  c.key_stride = page(key_codes, at::kFloat8_e4m3fn, "key_codes");
  c.value_stride = page(value_codes, at::kFloat8_e4m3fn, "value_codes");
  c.powers_stride = page(powers, at::kFloat8_e8m0fnu, "powers");
  if (key_codes.sizes() != value_codes.sizes()) raise("key_codes and value_codes must have the same shape");
  if (powers.size(0) != key_codes.size(0) || powers.size(1) != key_codes.size(1) || powers.size(2) != key_codes.size(2) || powers.size(3) != 2)
    raise("powers must be [pages, kv_heads, page_size, 2] of the codes");
  for (const int i : {1, 2, 3})
    if (key_codes.size(i) > 4096) raise("No suitable kernel. codes of " + std::to_string(key_codes.size(i)) + " heads, tokens or elements");
  c.key_codes = key_codes.data_ptr();
  c.value_codes = value_codes.data_ptr();
  c.powers = powers.data_ptr();
  c.n_pages = key_codes.size(0);
  c.kv_heads = (int32_t)key_codes.size(1);
  c.page_size = (int32_t)key_codes.size(2);
  c.head_dim = (int32_t)key_codes.size(3);
  return c;
}

py::tuple cache8_read(const at::Tensor &key_codes, const at::Tensor &value_codes, const at::Tensor &powers, const at::Tensor &loc,
                      at::ScalarType type, const c10::optional<at::Tensor> &k_out, const c10::optional<at::Tensor> &v_out) {
  if (!key_codes.is_cuda()) raise("key_codes must be a CUDA tensor");
  const c10::Device dev = key_codes.device();
  const mlora_cache8 c = cache8_of(key_codes, value_codes, powers, dev);
  check_on(loc, dev, "loc");
  check_type(loc, at::kLong, "loc");
  if (loc.dim() != 1 || !loc.is_contiguous()) raise("loc must be a contiguous 1D tensor");
  const int64_t n = loc.numel();
  if (type != at::kHalf && type != at::kBFloat16) raise(std::string("No suitable kernel. cache8_read dtype=torch.") + c10::toString(type));
  const auto result = [&](const c10::optional<at::Tensor> &given, const char *name) {
    if (!given.has_value()) return at::empty({n, c.kv_heads, c.head_dim}, key_codes.options().dtype(type));
    check_on(*given, dev, name);
    check_type(*given, type, name);
    return *given;
  };
  const at::Tensor k = result(k_out, "k_out"), v = result(v_out, "v_out");
  const Heads hk = dense_heads(k, c.head_dim, c.kv_heads, "k_out"), hv = dense_heads(v, c.head_dim, c.kv_heads, "v_out");
  if (hk.rows != n || hv.rows != n) raise("k_out and v_out must have a row per slot");
  if (n > 0 && hk.data == hv.data) raise("k_out must not be v_out");
  const c10::DeviceGuard on(dev);
  const hipStream_t st = stream_of(dev);
  const mlora_dtype code = dtype_code(k);
  check_unlocked([&] {
    return mlora_cache_read_codes(st, &c, static_cast<const int64_t *>(loc.data_ptr()), n, hk.data, hk.row_stride, hv.data, hv.row_stride, code);
  });
  return py::make_tuple(k, v);
}

// ---- rotary ----------------------------------------------------------------------------------------------------------------
// freqs: float64 [rotary_dim / 2] in turns per position
struct NativeRotary {
  at::Tensor freqs;
  int64_t head_dim, rotary_dim;
  bool interleaved;
  double gain;

  NativeRotary(const at::Tensor &f, int64_t head_dim_, bool interleaved_, double gain_)
      : freqs(f.contiguous()), head_dim(head_dim_), rotary_dim(2 * f.numel()), interleaved(interleaved_), gain(gain_) {
    if (!f.is_cuda()) raise("freqs must be a CUDA tensor");
    check_type(f, at::kDouble, "freqs");
  }

  mlora_rotary_part part(const at::Tensor &src, const at::Tensor &dst, int64_t T, bool turn, bool to_rows, const char *name) const {
    check_on(src, freqs.device(), name);
    check_on(dst, freqs.device(), name);
    const Heads s = heads_of(src, head_dim, name), d = heads_of(dst, head_dim, name);
    if (s.rows != T) raise(std::string(name) + " has " + std::to_string(s.rows) + " tokens, positions " + std::to_string(T));
    if (s.heads != d.heads || (!to_rows && d.rows != T)) raise(std::string(name) + ": source and destination differ in shape");
    if (src.scalar_type() != dst.scalar_type()) no_kernel(name, dst);
    if (s.data == d.data && (s.row_stride != d.row_stride || s.head_stride != d.head_stride))
      raise(std::string(name) + ": a destination that is the source must have its strides");
    mlora_rotary_part p{};
    p.src = s.data;
    p.dst = d.data;
    p.src_token_stride = s.row_stride;
    p.src_head_stride = s.head_stride;
    p.dst_token_stride = d.row_stride;
    p.dst_head_stride = d.head_stride;
    if (s.heads > 65536) raise(std::string(name) + ": too many heads");
    p.heads = (int32_t)s.heads;
    p.flags = (turn ? MLORA_ROTARY_TURN : 0) | (to_rows ? MLORA_ROTARY_TO_ROWS : 0);
    return p;
  }

  int64_t tokens(const at::Tensor &positions) const {
    check_on(positions, freqs.device(), "positions");
    check_type(positions, at::kLong, "positions");
    if (positions.dim() != 1 || !positions.is_contiguous()) raise("positions must be a contiguous 1D tensor");
    return positions.numel();
  }

  void call(const mlora_rotary_part *parts, int n, const at::Tensor &positions, const int64_t *loc, int64_t n_rows, const at::Tensor &like) const {
    const mlora_dtype code = dtype_code(like);
    if ((int)code < 0) no_kernel("rotary", like);
    const c10::DeviceGuard on(freqs.device());
    const hipStream_t st = stream_of(freqs.device());
    check_unlocked([&] {
      return mlora_rotary(st, parts, n, static_cast<const int64_t *>(positions.data_ptr()), loc, n_rows, positions.numel(),
                          (int32_t)head_dim, (int32_t)rotary_dim, interleaved, static_cast<const double *>(freqs.data_ptr()),
                          (float)gain, code);
    });
  }

  void apply(const at::Tensor &positions, const at::Tensor &q, const c10::optional<at::Tensor> &k,
             const c10::optional<at::Tensor> &q_out, const c10::optional<at::Tensor> &k_out) const {
    const int64_t T = tokens(positions);
    mlora_rotary_part parts[2];
    int n = 0;
    parts[n++] = part(q, q_out.has_value() ? *q_out : q, T, true, false, "q");
    if (k.has_value()) {
      if (k->scalar_type() != q.scalar_type()) no_kernel("k", *k);
      parts[n++] = part(*k, k_out.has_value() ? *k_out : *k, T, true, false, "k");
    } else if (k_out.has_value()) {
      raise("k_out without k");
    }
    call(parts, n, positions, nullptr, 0, q);
  }

  void store(const at::Tensor &positions, const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &key_buffer,
             const at::Tensor &value_buffer, const at::Tensor &loc, const c10::optional<at::Tensor> &q_out) const {
    const int64_t T = tokens(positions);
    if (k.scalar_type() != q.scalar_type()) no_kernel("k", k);
    if (v.scalar_type() != q.scalar_type()) no_kernel("v", v);
    const mlora_rotary_part parts[3] = {part(q, q_out.has_value() ? *q_out : q, T, true, false, "q"),
                                        part(k, key_buffer, T, true, true, "key_buffer"),
                                        part(v, value_buffer, T, false, true, "value_buffer")};
    check_on(loc, freqs.device(), "loc");
    check_type(loc, at::kLong, "loc");
    if (loc.dim() != 1 || loc.numel() != T || !loc.is_contiguous()) raise("loc must be a contiguous 1D tensor with a row per token");
    if (key_buffer.size(0) != value_buffer.size(0)) raise("key_buffer and value_buffer must have the same rows");
    call(parts, 3, positions, static_cast<const int64_t *>(loc.data_ptr()), key_buffer.size(0), q);
  }

  void store8(const at::Tensor &positions, const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &key_codes,
              const at::Tensor &value_codes, const at::Tensor &powers, const at::Tensor &loc, const c10::optional<at::Tensor> &q_out) const {
    const int64_t T = tokens(positions);
    const c10::Device dev = freqs.device();
    const mlora_dtype code = dtype_code(q);
    if ((int)code < 0) no_kernel("rotary", q);
    if (k.scalar_type() != q.scalar_type()) no_kernel("k", k);
    if (v.scalar_type() != q.scalar_type()) no_kernel("v", v);
    const mlora_rotary_part part_q = part(q, q_out.has_value() ? *q_out : q, T, true, false, "q");
    const mlora_cache8 c = cache8_of(key_codes, value_codes, powers, dev);
    if (c.head_dim != head_dim) raise("the codes' head_dim=" + std::to_string(c.head_dim) + " is not the rotary's " + std::to_string(head_dim));
    check_on(k, dev, "k");
    check_on(v, dev, "v");
    const Heads hk = heads_of(k, head_dim, "k"), hv = heads_of(v, head_dim, "v");
    if (hk.rows != T || hv.rows != T) raise("k and v must have a row per position");
    if (hk.heads != c.kv_heads || hv.heads != c.kv_heads) raise("k and v must have the codes' " + std::to_string(c.kv_heads) + " heads");
    check_on(loc, dev, "loc");
    check_type(loc, at::kLong, "loc");
    if (loc.dim() != 1 || loc.numel() != T || !loc.is_contiguous()) raise("loc must be a contiguous 1D tensor with a slot per token");
    const c10::DeviceGuard on(dev);
    const hipStream_t st = stream_of(dev);
    check_unlocked([&] {
      return mlora_rotary_store_codes(st, &part_q, hk.data, hk.row_stride, hk.head_stride, hv.data, hv.row_stride, hv.head_stride, &c,
                                 static_cast<const int64_t *>(positions.data_ptr()), static_cast<const int64_t *>(loc.data_ptr()), T,
                                 (int32_t)rotary_dim, interleaved, static_cast<const double *>(freqs.data_ptr()), (float)gain, code);
    });
  }
};

// ---- attention -------------------------------------------------------------------------------------------------------------
struct NativeAttentionPlan {
  mlora_attention_plan plan{};
  at::Tensor start, seq, kv, buf, workspace, weights_workspace;

  NativeAttentionPlan(const at::Tensor &b_start_loc, const at::Tensor &b_seq_len, const at::Tensor &b_kv_len, int64_t n_tokens,
                      int64_t max_seq_len, int64_t max_kv_len, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t page_size,
                      int64_t window)
      : start(b_start_loc), seq(b_seq_len), kv(b_kv_len) {
    if (!start.is_cuda()) raise("b_start_loc must be a CUDA tensor");
    for (const auto &t : {std::make_pair(&start, "b_start_loc"), std::make_pair(&seq, "b_seq_len"), std::make_pair(&kv, "b_kv_len")}) {
      check_on(*t.first, start.device(), t.second);
      check_type(*t.first, at::kInt, t.second);
      if (t.first->dim() != 1 || !t.first->is_contiguous() || t.first->numel() != start.numel())
        raise(std::string(t.second) + " must be a contiguous 1D tensor with an entry per request");
    }
    for (const int64_t v : {q_heads, kv_heads, head_dim, page_size, window})
      if (v > INT32_MAX || v < INT32_MIN) raise("attention plan: heads, head_dim, page_size or window out of range");
    plan.n_req = start.numel();
    plan.n_tokens = n_tokens;
    plan.max_seq_len = max_seq_len;
    plan.max_kv_len = max_kv_len;
    plan.q_heads = (int32_t)q_heads;
    plan.kv_heads = (int32_t)kv_heads;
    plan.head_dim = (int32_t)head_dim;
    plan.page_size = (int32_t)page_size;
    plan.window = (int32_t)window;
    const size_t bytes = mlora_attention_plan_bytes(&plan);
    if (bytes == 0) check_rc(MLORA_ERR_INVALID);
    // they stay where they are for as long as the plan lives: a graph captured from it keeps pointing at live memory
    buf = at::empty({(int64_t)bytes}, start.options().dtype(at::kByte));
    workspace = at::empty({(int64_t)mlora_attention_workspace_bytes(&plan, 0)}, start.options().dtype(at::kByte));
    plan.dev = buf.data_ptr();
    plan.bytes = bytes;
    rebuild();
  }

  void rebuild() {
    const c10::DeviceGuard on(start.device());
    const hipStream_t st = stream_of(start.device());
    check_unlocked([&] {
      return mlora_build_attention_plan(st, &plan, static_cast<const int32_t *>(start.data_ptr()),
                                        static_cast<const int32_t *>(seq.data_ptr()), static_cast<const int32_t *>(kv.data_ptr()));
    });
  }

  // What attend and attend8 take beside the cache; `call` makes the call of the C ABI
  template <typename F>
  void attend_over(const at::Tensor &out, const at::Tensor &q, const at::Tensor &table, const c10::optional<double> &scale,
                   const c10::optional<at::Tensor> &weights, F call) {
    const c10::Device dev = start.device();
    const mlora_dtype code = dtype_code(q);
    const Heads ho = dense_heads(out, plan.head_dim, plan.q_heads, "out"), hq = dense_heads(q, plan.head_dim, plan.q_heads, "q");
    if (ho.rows != plan.n_tokens || hq.rows != plan.n_tokens)
      raise("q and out must have the plan's " + std::to_string(plan.n_tokens) + " tokens");
    if (ho.data == hq.data && plan.n_tokens > 0) raise("out must not be q");
    check_type(table, at::kInt, "table");
    if (table.dim() != 2 || table.size(0) != plan.n_req || (table.numel() > 0 && table.stride(1) != 1))
      raise("table must be [requests, pages] with contiguous rows");
    float *w = nullptr;
    int64_t w_stride = 0;
    if (weights.has_value()) {
      check_on(*weights, dev, "weights");
      check_type(*weights, at::kFloat, "weights");
      if (weights->dim() != 2 || weights->size(0) != plan.n_req || weights->size(1) < plan.max_kv_len ||
          (weights->numel() > 0 && weights->stride(1) != 1))
        raise("weights must be [requests, at least max_kv_len] with contiguous rows");
      w = static_cast<float *>(weights->data_ptr());
      w_stride = plan.n_req > 1 ? weights->stride(0) : weights->size(1);
      if (w_stride < plan.max_kv_len) raise("weights: rows overlap");
    }
    if (w && !weights_workspace.defined())      // (up to 256 MB, for those who ask for weights)
      weights_workspace = at::empty({(int64_t)mlora_attention_workspace_bytes(&plan, 1)}, start.options().dtype(at::kByte));
    const at::Tensor room = w ? weights_workspace : workspace;
    const float s = scale.has_value() ? (float)*scale : 1.0f / std::sqrt((float)plan.head_dim);
    const c10::DeviceGuard on(dev);
    const hipStream_t st = stream_of(dev);
    check_unlocked([&] {
      return call(st, room.data_ptr(), (size_t)room.numel(), ho, hq, static_cast<const int32_t *>(table.data_ptr()),
                  plan.n_req > 1 ? table.stride(0) : table.size(1), table.size(1), s, w, w_stride, code);
    });
  }

  void attend(const at::Tensor &out, const at::Tensor &q, const at::Tensor &key_buffer, const at::Tensor &value_buffer,
              const at::Tensor &table, const c10::optional<double> &scale, const c10::optional<at::Tensor> &weights) {
    const c10::Device dev = start.device();
    check_on(out, dev, "out");
    check_on(q, dev, "q");
    check_on(key_buffer, dev, "key_buffer");
    check_on(value_buffer, dev, "value_buffer");
    check_on(table, dev, "table");
    if ((int)dtype_code(q) < 0) no_kernel("q", q);
    if (out.scalar_type() != q.scalar_type()) no_kernel("out", out);
    if (key_buffer.scalar_type() != q.scalar_type()) no_kernel("key_buffer", key_buffer);
    if (value_buffer.scalar_type() != q.scalar_type()) no_kernel("value_buffer", value_buffer);
    const Heads hk = dense_heads(key_buffer, plan.head_dim, plan.kv_heads, "key_buffer"),
                hv = dense_heads(value_buffer, plan.head_dim, plan.kv_heads, "value_buffer");
    if (hk.rows != hv.rows) raise("key_buffer and value_buffer must have the same rows");
    attend_over(out, q, table, scale, weights,
                [&](hipStream_t st, void *room, size_t bytes, const Heads &ho, const Heads &hq, const int32_t *pages, int64_t stride, int64_t width,
                    float by, float *w, int64_t w_stride, mlora_dtype code) {
                  return mlora_paged_attention(st, &plan, room, bytes, ho.data, ho.row_stride, hq.data, hq.row_stride, hk.data, hk.row_stride,
                                               hv.data, hv.row_stride, hk.rows, pages, stride, width, by, w, w_stride, code);
                });
  }

  void attend8(const at::Tensor &out, const at::Tensor &q, const at::Tensor &key_codes, const at::Tensor &value_codes, const at::Tensor &powers,
               const at::Tensor &table, const c10::optional<double> &scale, const c10::optional<at::Tensor> &weights) {
    const c10::Device dev = start.device();
    check_on(out, dev, "out");
    check_on(q, dev, "q");
    check_on(table, dev, "table");
    if ((int)dtype_code(q) < 0) no_kernel("q", q);
    if (out.scalar_type() != q.scalar_type()) no_kernel("out", out);
    const mlora_cache8 c = cache8_of(key_codes, value_codes, powers, dev);
    attend_over(out, q, table, scale, weights,
                [&](hipStream_t st, void *room, size_t bytes, const Heads &ho, const Heads &hq, const int32_t *pages, int64_t stride, int64_t width,
                    float by, float *w, int64_t w_stride, mlora_dtype code) {
                  return mlora_paged_attention_codes(st, &plan, room, bytes, ho.data, ho.row_stride, hq.data, hq.row_stride, &c, pages, stride, width,
                                                by, w, w_stride, code);
                });
  }
};

// ---- eviction --------------------------------------------------------------------------------------------------------------
py::tuple cache_evict(const at::Tensor &table, const at::Tensor &kv_len, const at::Tensor &weights, int64_t budget, int64_t recent,
                      int64_t sinks, int64_t page_size) {
  if (!table.is_cuda()) raise("table must be a CUDA tensor");
  const c10::Device dev = table.device();
  check_on(kv_len, dev, "b_kv_len");
  check_on(weights, dev, "weights");
  check_type(table, at::kInt, "table");
  check_type(kv_len, at::kInt, "b_kv_len");
  check_type(weights, at::kFloat, "weights");
  if (table.dim() != 2 || (table.numel() > 0 && table.stride(1) != 1)) raise("table must be [requests, pages] with contiguous rows");
  const int64_t n = table.size(0), width = table.size(1);
  if (kv_len.dim() != 1 || kv_len.numel() != n || !kv_len.is_contiguous()) raise("b_kv_len must be a contiguous 1D tensor with an entry per request");
  if (page_size < 1 || page_size > 256) raise("No suitable kernel. cache_evict: page_size=" + std::to_string(page_size) + " (a power of two up to 256)");
  if (weights.dim() != 2 || weights.size(0) != n || weights.size(1) != width * page_size || (weights.numel() > 0 && weights.stride(1) != 1))
    raise("weights must be [requests, pages * page_size] with contiguous rows");
  at::Tensor new_table = at::empty({n, width}, table.options()), new_len = at::empty({n}, kv_len.options()),
             new_weights = at::empty({n, width * page_size}, weights.options()), freed = at::empty({n, width}, table.options());
  const c10::DeviceGuard on(dev);
  const hipStream_t st = stream_of(dev);
  check_unlocked([&] {
    return mlora_cache_evict(st, static_cast<const int32_t *>(table.data_ptr()), n > 1 ? table.stride(0) : width,
                             static_cast<const int32_t *>(kv_len.data_ptr()), static_cast<const float *>(weights.data_ptr()),
                             n > 1 ? weights.stride(0) : width * page_size, n, width, (int32_t)page_size, budget, recent, sinks,
                             static_cast<int32_t *>(new_table.data_ptr()), static_cast<int32_t *>(new_len.data_ptr()),
                             static_cast<float *>(new_weights.data_ptr()), static_cast<int32_t *>(freed.data_ptr()));
  });
  return py::make_tuple(new_table, new_len, new_weights, freed);
}

}  // namespace

void bind_attention(py::module_ &m) {
  py::class_<NativeRotary>(m, "NativeRotary")
      .def(py::init<const at::Tensor &, int64_t, bool, double>())
      .def("apply", &NativeRotary::apply)
      .def("store", &NativeRotary::store)
      .def("store8", &NativeRotary::store8);
  py::class_<NativeAttentionPlan>(m, "NativeAttentionPlan")
      .def(py::init<const at::Tensor &, const at::Tensor &, const at::Tensor &, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t,
                    int64_t, int64_t>())
      .def("rebuild", &NativeAttentionPlan::rebuild)
      .def("attend", &NativeAttentionPlan::attend)
      .def("attend8", &NativeAttentionPlan::attend8)
      .def_readonly("buf", &NativeAttentionPlan::buf)
      .def_readonly("workspace", &NativeAttentionPlan::workspace);
  m.def("cache_evict", &cache_evict);
  m.def("cache8_read", &cache8_read);
}
