// pad_torch_op.cpp -- the thin torch operator over the C ABI of
// libpad_b200.so (include/pad_b200.h): torch.ops.pad_b200.*.
//
// It plays the part of the reference's pybind binding `forward_v4`
// (cuda/binding.cpp:13-14, cuda/kernels.h:60-70) and of the launcher glue
// around it (cuda/kernel_v4_split_k.cu:205-268): it takes tensors, makes
// block_table / seq_lens int32 (src/kernel_cuda_v4.py:58-59), allocates `out`,
// keeps one reusable workspace and one error-flag word per (device, stream),
// and calls the C entry point on the current stream of the inputs' device.
// Everything here is host code; the kernels are in libpad_b200.so.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/library.h>

#include <algorithm>
#include <cstdint>
#include <initializer_list>
#include <map>
#include <mutex>
#include <tuple>
#include <utility>

#include "pad_b200.h"

namespace {

struct StreamState {
  at::Tensor workspace;  // uint8, grown on demand, never shrunk
  at::Tensor flags;      // int32[1], PAD_FLAG_* bits OR-ed in by the kernels
};

std::mutex g_mu;
std::map<std::pair<int, cudaStream_t>, StreamState> g_state;

StreamState& state_for(const at::Device& dev, cudaStream_t s) {
  std::lock_guard<std::mutex> lk(g_mu);
  auto key = std::make_pair(static_cast<int>(dev.index()), s);
  auto it = g_state.find(key);
  if (it == g_state.end()) {
    StreamState st;
    st.workspace = at::empty({0}, at::TensorOptions().dtype(at::kByte).device(dev));
    st.flags = at::zeros({1}, at::TensorOptions().dtype(at::kInt).device(dev));
    it = g_state.emplace(key, std::move(st)).first;
  }
  return it->second;
}

void check(int status, const char* what) {
  TORCH_CHECK(status == PAD_OK, "libpad_b200 ", what, ": ", pad_status_string(status), ": ", pad_last_error());
}

at::Tensor as_int32_rows(const at::Tensor& t, const at::Device& dev) {
  at::Tensor r = t.device() == dev && t.scalar_type() == at::kInt ? t : t.to(dev, at::kInt);
  return r.dim() >= 1 && r.stride(-1) == 1 ? r : r.contiguous();
}

// q needs a contiguous head_dim axis, 16-byte aligned rows and base.
at::Tensor tma_ready(const at::Tensor& q) {
  const bool ok = q.stride(2) == 1 && q.stride(0) % 8 == 0 && q.stride(1) % 8 == 0 &&
                  reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 == 0;
  return ok ? q : q.contiguous();
}

at::Tensor prepare_out(const c10::optional<at::Tensor>& out, const at::Tensor& q) {
  if (!out.has_value()) return at::empty(q.sizes(), q.options().dtype(at::kHalf));
  const at::Tensor& o = *out;
  TORCH_CHECK(o.sizes() == q.sizes() && o.scalar_type() == at::kHalf && o.device() == q.device(),
              "out must be an fp16 tensor shaped like q on q's device");
  return o;
}

// Calls `launch(ws_ptr, ws_bytes)`; when the workspace is too small the
// library reports PAD_ERR_WORKSPACE before launching anything, so grow it to
// `need()` and call again.
template <class Launch, class Need>
void with_workspace(StreamState& st, Launch launch, Need need) {
  int rc = launch(st.workspace.data_ptr(), (size_t)st.workspace.numel());
  if (rc == PAD_ERR_WORKSPACE) {
    size_t bytes = 0;
    check(need(&bytes), "workspace size");
    const int64_t grow = std::max<int64_t>((int64_t)bytes, 2 * st.workspace.numel());
    st.workspace = at::empty({grow}, st.workspace.options());
    rc = launch(st.workspace.data_ptr(), (size_t)st.workspace.numel());
  }
  check(rc, "decode");
}

at::Tensor decode(const at::Tensor& q_in, const at::Tensor& k, const at::Tensor& v, const at::Tensor& bt_in,
                  const at::Tensor& sl_in, int64_t num_splits, double scale, const c10::optional<at::Tensor>& out_in) {
  TORCH_CHECK(q_in.dim() == 3 && k.dim() == 4 && v.sizes() == k.sizes(), "bad q / k_cache / v_cache shapes");
  const at::Device dev = q_in.device();
  c10::cuda::CUDAGuard guard(dev);
  const at::Tensor q = tma_ready(q_in);
  const at::Tensor bt = as_int32_rows(bt_in, dev);
  const at::Tensor sl = as_int32_rows(sl_in, dev);
  at::Tensor out = prepare_out(out_in, q_in);
  const int64_t batch = q.size(0);
  if (batch == 0) return out;
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  StreamState& st = state_for(dev, stream);
  const int64_t qs[3] = {q.stride(0), q.stride(1), q.stride(2)};
  const int64_t ks[4] = {k.stride(0), k.stride(1), k.stride(2), k.stride(3)};
  const int64_t vs[4] = {v.stride(0), v.stride(1), v.stride(2), v.stride(3)};
  const int64_t os[3] = {out.stride(0), out.stride(1), out.stride(2)};
  const int64_t hq = q.size(1), d = q.size(2), pages = k.size(0), ps = k.size(1), hkv = k.size(2);
  const int64_t maxp = bt.size(1);
  with_workspace(
      st,
      [&](void* ws, size_t wsb) {
        return pad_paged_attention_decode(q.data_ptr(), k.data_ptr(), v.data_ptr(), bt.data_ptr<int32_t>(),
                                          sl.data_ptr<int32_t>(), out.data_ptr(), batch, hq, hkv, d, pages, ps, maxp,
                                          qs, ks, vs, bt.stride(0), os, (float)scale, num_splits, ws, wsb, stream,
                                          st.flags.data_ptr<int32_t>());
      },
      [&](size_t* bytes) {
        return pad_decode_workspace_bytes((int)dev.index(), batch, hkv, hq / hkv, d, ps, maxp, num_splits, bytes);
      });
  return out;
}

at::Tensor decode_csr(const at::Tensor& q_in, const at::Tensor& k, const at::Tensor& v, const at::Tensor& indptr_in,
                      const at::Tensor& indices_in, const at::Tensor& last_in, int64_t num_splits, double scale,
                      const c10::optional<at::Tensor>& out_in) {
  TORCH_CHECK(q_in.dim() == 3 && k.dim() == 4 && v.sizes() == k.sizes(), "bad q / k_cache / v_cache shapes");
  const at::Device dev = q_in.device();
  c10::cuda::CUDAGuard guard(dev);
  const at::Tensor q = tma_ready(q_in);
  const at::Tensor indptr = as_int32_rows(indptr_in, dev);
  at::Tensor indices = as_int32_rows(indices_in, dev);
  const at::Tensor last = as_int32_rows(last_in, dev);
  at::Tensor out = prepare_out(out_in, q_in);
  const int64_t batch = q.size(0);
  if (batch == 0) return out;
  const int64_t nnz = std::max<int64_t>(indices.numel(), 1);
  if (indices.numel() == 0) indices = at::zeros({1}, indices.options());
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  StreamState& st = state_for(dev, stream);
  const int64_t qs[3] = {q.stride(0), q.stride(1), q.stride(2)};
  const int64_t ks[4] = {k.stride(0), k.stride(1), k.stride(2), k.stride(3)};
  const int64_t vs[4] = {v.stride(0), v.stride(1), v.stride(2), v.stride(3)};
  const int64_t os[3] = {out.stride(0), out.stride(1), out.stride(2)};
  const int64_t hq = q.size(1), d = q.size(2), pages = k.size(0), ps = k.size(1), hkv = k.size(2);
  with_workspace(
      st,
      [&](void* ws, size_t wsb) {
        return pad_paged_attention_decode_csr(q.data_ptr(), k.data_ptr(), v.data_ptr(), indptr.data_ptr<int32_t>(),
                                              indices.data_ptr<int32_t>(), last.data_ptr<int32_t>(), out.data_ptr(),
                                              batch, hq, hkv, d, pages, ps, nnz, qs, ks, vs, os, (float)scale,
                                              num_splits, ws, wsb, stream, st.flags.data_ptr<int32_t>());
      },
      [&](size_t* bytes) {
        return pad_decode_csr_workspace_bytes((int)dev.index(), batch, hkv, hq / hkv, d, ps, nnz, num_splits, bytes);
      });
  return out;
}

void kv_append(const at::Tensor& k_new_in, const at::Tensor& v_new_in, const at::Tensor& k_cache,
               const at::Tensor& v_cache, const at::Tensor& bt_in, const at::Tensor& pos_in) {
  TORCH_CHECK(k_new_in.dim() == 3 && k_cache.dim() == 4, "k_new must be [B, Hkv, D], the caches 4-D");
  const at::Device dev = k_cache.device();
  c10::cuda::CUDAGuard guard(dev);
  const at::Tensor bt = as_int32_rows(bt_in, dev);
  const at::Tensor pos = as_int32_rows(pos_in, dev);
  const at::Tensor kn = k_new_in.stride(2) == 1 ? k_new_in : k_new_in.contiguous();
  const at::Tensor vn = v_new_in.stride(2) == 1 ? v_new_in : v_new_in.contiguous();
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  StreamState& st = state_for(dev, stream);
  const int64_t kns[3] = {kn.stride(0), kn.stride(1), kn.stride(2)};
  const int64_t vns[3] = {vn.stride(0), vn.stride(1), vn.stride(2)};
  const int64_t ks[4] = {k_cache.stride(0), k_cache.stride(1), k_cache.stride(2), k_cache.stride(3)};
  const int64_t vs[4] = {v_cache.stride(0), v_cache.stride(1), v_cache.stride(2), v_cache.stride(3)};
  check(pad_paged_kv_append(kn.data_ptr(), vn.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                            bt.data_ptr<int32_t>(), pos.data_ptr<int32_t>(), kn.size(0), kn.size(1), kn.size(2),
                            k_cache.size(0), k_cache.size(1), bt.size(1), kns, vns, ks, vs, bt.stride(0), stream,
                            st.flags.data_ptr<int32_t>()),
        "kv_append");
}

// A tensor's strides as the C entry points take them. The stride of an axis of
// one element means nothing (torch keeps any number there): it becomes what a
// dense tensor would have.
struct Strides {
  int64_t s[4] = {0, 0, 0, 0};
  explicit Strides(const at::Tensor& t) {
    int64_t dense = 1;
    for (int64_t i = std::min<int64_t>(t.dim(), 4) - 1; i >= 0; --i) {
      s[i] = t.size(i) == 1 ? dense : t.stride(i);
      dense = s[i] * std::max<int64_t>(t.size(i), 1);
    }
  }
};

// q as the kernels read it: rows of 16-byte pieces (a copy where it is not).
at::Tensor aligned_rows(const at::Tensor& q) {
  const Strides st(q);
  const bool ok = st.s[2] == 1 && st.s[0] % 8 == 0 && st.s[1] % 8 == 0 && st.s[0] > 0 && st.s[1] > 0 &&
                  reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 == 0;
  return ok ? q : q.clone(at::MemoryFormat::Contiguous);
}

void check_on(const at::Device& dev, std::initializer_list<const at::Tensor*> all, const char* what) {
  for (const at::Tensor* t : all)
    TORCH_CHECK(t->device() == dev, "libpad_b200 ", what, ": every tensor must be on ", dev.str());
}

// The 4-bit caches of one call: codes [P, page, Hkv, D/2], scales [P, page, Hkv, 4].
void check_fp4(const at::Tensor& k, const at::Tensor& ks, const at::Tensor& v, const at::Tensor& vs, const char* what) {
  TORCH_CHECK(k.dim() == 4 && ks.dim() == 4 && v.sizes() == k.sizes() && vs.sizes() == ks.sizes() &&
                  ks.size(0) == k.size(0) && ks.size(1) == k.size(1) && ks.size(2) == k.size(2) && ks.size(3) == 4,
              "libpad_b200 ", what, ": codes must be [pages, page_size, Hkv, D/2], scales [pages, page_size, Hkv, 4]");
  for (const at::Tensor* t : {&k, &ks, &v, &vs})
    TORCH_CHECK(t->scalar_type() == at::kByte, "libpad_b200 ", what, ": codes and scales must be uint8");
}

void kv_append_fp4(const at::Tensor& k_new, const at::Tensor& v_new, const at::Tensor& k, const at::Tensor& ks,
                   const at::Tensor& v, const at::Tensor& vs, const at::Tensor& bt_in, const at::Tensor& pos_in,
                   const c10::optional<at::Tensor>& ids_in) {
  const at::Device dev = k.device();
  check_fp4(k, ks, v, vs, "kv_append_fp4");
  check_on(dev, {&k_new, &v_new, &ks, &v, &vs}, "kv_append_fp4");
  TORCH_CHECK(k_new.dim() == 3 && v_new.sizes() == k_new.sizes() && k_new.scalar_type() == at::kHalf &&
                  v_new.scalar_type() == at::kHalf && k_new.size(1) == k.size(2) && k_new.size(2) == 2 * k.size(3),
              "libpad_b200 kv_append_fp4: k_new and v_new must be fp16 [tokens, Hkv, D] of the cache's heads");
  TORCH_CHECK(bt_in.dim() == 2 && pos_in.dim() == 1 && pos_in.size(0) == k_new.size(0) &&
                  (!ids_in.has_value() || (ids_in->dim() == 1 && ids_in->size(0) == k_new.size(0))),
              "libpad_b200 kv_append_fp4: block_table must be [B, max_pages], positions and seq_ids [tokens]");
  c10::cuda::CUDAGuard guard(dev);
  const at::Tensor bt = as_int32_rows(bt_in, dev), pos = as_int32_rows(pos_in, dev);
  const at::Tensor ids = ids_in.has_value() ? as_int32_rows(*ids_in, dev) : at::Tensor();
  const at::Tensor kn = Strides(k_new).s[2] == 1 ? k_new : k_new.contiguous();
  const at::Tensor vn = Strides(v_new).s[2] == 1 ? v_new : v_new.contiguous();
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  StreamState& st = state_for(dev, stream);
  const Strides kns(kn), vns(vn), k_s(k), ks_s(ks), v_s(v), vs_s(vs);
  check(pad_paged_kv_append_fp4(kn.data_ptr(), vn.data_ptr(), k.data_ptr(), ks.data_ptr(), v.data_ptr(), vs.data_ptr(),
                                bt.data_ptr<int32_t>(), pos.data_ptr<int32_t>(),
                                ids.defined() ? ids.data_ptr<int32_t>() : nullptr, kn.size(0), bt.size(0), kn.size(1),
                                kn.size(2), k.size(0), k.size(1), bt.size(1), kns.s, vns.s, k_s.s, ks_s.s, v_s.s,
                                vs_s.s, Strides(bt).s[0], stream, st.flags.data_ptr<int32_t>()),
        "kv_append_fp4");
}

std::tuple<at::Tensor, at::Tensor> kv_read_fp4(const at::Tensor& k, const at::Tensor& ks, const at::Tensor& v,
                                               const at::Tensor& vs, const at::Tensor& bt_in, const at::Tensor& pos_in,
                                               const c10::optional<at::Tensor>& ids_in) {
  const at::Device dev = k.device();
  check_fp4(k, ks, v, vs, "kv_read_fp4");
  check_on(dev, {&ks, &v, &vs}, "kv_read_fp4");
  TORCH_CHECK(bt_in.dim() == 2 && pos_in.dim() == 1 &&
                  (!ids_in.has_value() || (ids_in->dim() == 1 && ids_in->size(0) == pos_in.size(0))),
              "libpad_b200 kv_read_fp4: block_table must be [B, max_pages], positions and seq_ids [tokens]");
  c10::cuda::CUDAGuard guard(dev);
  const at::Tensor bt = as_int32_rows(bt_in, dev), pos = as_int32_rows(pos_in, dev);
  const at::Tensor ids = ids_in.has_value() ? as_int32_rows(*ids_in, dev) : at::Tensor();
  const int64_t tokens = pos.size(0), hkv = k.size(2), d = 2 * k.size(3);
  at::Tensor ko = at::empty({tokens, hkv, d}, k.options().dtype(at::kHalf)), vo = at::empty_like(ko);
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  StreamState& st = state_for(dev, stream);
  const Strides kos(ko), vos(vo), k_s(k), ks_s(ks), v_s(v), vs_s(vs);
  check(pad_paged_kv_read_fp4(k.data_ptr(), ks.data_ptr(), v.data_ptr(), vs.data_ptr(), bt.data_ptr<int32_t>(),
                              pos.data_ptr<int32_t>(), ids.defined() ? ids.data_ptr<int32_t>() : nullptr,
                              ko.data_ptr(), vo.data_ptr(), tokens, bt.size(0), hkv, d, k.size(0), k.size(1),
                              bt.size(1), k_s.s, ks_s.s, v_s.s, vs_s.s, kos.s, vos.s, Strides(bt).s[0], stream,
                              st.flags.data_ptr<int32_t>()),
        "kv_read_fp4");
  return {ko, vo};
}

// weights / slot_positions of a cache: [pages, Hkv, page_size] of one type.
void check_slots(const at::Tensor& t, at::ScalarType type, int64_t pages, int64_t hkv, int64_t ps, const char* what) {
  TORCH_CHECK(t.dim() == 3 && t.scalar_type() == type && t.size(0) == pages && t.size(1) == hkv && t.size(2) == ps,
              "libpad_b200 ", what, ": weights (fp32) and slot_positions (int32) must be [pages, Hkv, page_size]");
}

// What a decode with attention weights takes beside the decode's arguments.
struct Tracked {
  at::Tensor total, num_new_of;
  Strides ws, ps;
  Tracked(const at::Tensor& weights, const c10::optional<at::Tensor>& positions,
          const c10::optional<at::Tensor>& total_in, int64_t num_new, const c10::optional<at::Tensor>& num_new_in,
          int64_t pages, int64_t hkv, int64_t page_size, int64_t batch, const at::Device& dev, const char* what)
      : ws(weights), ps(positions.has_value() ? *positions : weights) {
    check_slots(weights, at::kFloat, pages, hkv, page_size, what);
    check_on(dev, {&weights}, what);
    TORCH_CHECK(num_new >= 0, "libpad_b200 ", what, ": num_new must not be negative");
    TORCH_CHECK(positions.has_value() == total_in.has_value(), "libpad_b200 ", what,
                ": slot_positions and total_lens go together");
    if (positions.has_value()) {
      check_slots(*positions, at::kInt, pages, hkv, page_size, what);
      check_on(dev, {&*positions}, what);
      TORCH_CHECK(total_in->dim() == 1 && total_in->size(0) == batch, "libpad_b200 ", what,
                  ": total_lens must be [B]");
      total = as_int32_rows(*total_in, dev);
    }
    if (num_new_in.has_value()) {
      const at::Tensor& n = *num_new_in;
      TORCH_CHECK(n.dim() == 1 && n.size(0) == batch && at::isIntegralType(n.scalar_type(), false), "libpad_b200 ",
                  what, ": num_new must be a number or an integer tensor [B]");
      num_new_of = as_int32_rows(n.scalar_type() == at::kLong ? n.clamp(0, INT32_MAX) : n, dev);
    }
  }
  const int32_t* total_ptr() const { return total.defined() ? total.data_ptr<int32_t>() : nullptr; }
};

// Decode, and the attention weights of the cached tokens. The workspace, tens
// of times the decode's own, is the call's: two captured graphs never share one.
at::Tensor decode_weights(const at::Tensor& q_in, const at::Tensor& k, const at::Tensor& v, const at::Tensor& bt_in,
                          const at::Tensor& sl_in, int64_t num_splits, double scale,
                          const c10::optional<at::Tensor>& out_in, const at::Tensor& weights, int64_t num_new,
                          const c10::optional<at::Tensor>& positions, const c10::optional<at::Tensor>& total_in,
                          const c10::optional<at::Tensor>& num_new_in) {
  TORCH_CHECK(q_in.dim() == 3 && k.dim() == 4 && v.sizes() == k.sizes() && k.size(2) > 0 && k.size(3) == q_in.size(2),
              "libpad_b200 decode_weights: bad q / k_cache / v_cache shapes");
  TORCH_CHECK(q_in.scalar_type() == at::kHalf && k.scalar_type() == at::kHalf && v.scalar_type() == at::kHalf,
              "libpad_b200 decode_weights: q, k_cache and v_cache must be fp16");
  TORCH_CHECK(bt_in.dim() == 2 && bt_in.size(0) == q_in.size(0) && sl_in.dim() == 1 && sl_in.size(0) == q_in.size(0),
              "libpad_b200 decode_weights: block_table must be [B, max_pages], seq_lens [B]");
  const at::Device dev = q_in.device();
  check_on(dev, {&k, &v}, "decode_weights");
  c10::cuda::CUDAGuard guard(dev);
  const int64_t batch = q_in.size(0), hq = q_in.size(1), d = q_in.size(2), pages = k.size(0), ps = k.size(1),
                hkv = k.size(2);
  const Tracked tr(weights, positions, total_in, num_new, num_new_in, pages, hkv, ps, batch, dev, "decode_weights");
  const at::Tensor q = aligned_rows(q_in);
  const at::Tensor bt = as_int32_rows(bt_in, dev), sl = as_int32_rows(sl_in, dev);
  at::Tensor out = prepare_out(out_in, q_in);
  if (batch == 0) return out;
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  StreamState& st = state_for(dev, stream);
  const Strides qs(q), ks(k), vs(v), os(out);
  size_t bytes = 0;
  check(pad_decode_weights_workspace_bytes((int)dev.index(), batch, hkv, hq / hkv, d, pages, ps, bt.size(1),
                                           num_splits, &bytes),
        "workspace size");
  const at::Tensor ws = at::empty({(int64_t)bytes}, st.flags.options().dtype(at::kByte));
  auto call = [&](auto entry, auto news) {
    return entry(q.data_ptr(), k.data_ptr(), v.data_ptr(), bt.data_ptr<int32_t>(), sl.data_ptr<int32_t>(),
                 out.data_ptr(), weights.data_ptr<float>(),
                 positions.has_value() ? positions->data_ptr<int32_t>() : nullptr, tr.total_ptr(), news, batch, hq, hkv,
                 d, pages, ps, bt.size(1), qs.s, ks.s, vs.s, Strides(bt).s[0], os.s, tr.ws.s, tr.ps.s, (float)scale,
                 num_splits, ws.data_ptr(), bytes, stream, st.flags.data_ptr<int32_t>());
  };
  check(tr.num_new_of.defined()
            ? call(pad_paged_attention_decode_weights_by_seq, (const int32_t*)tr.num_new_of.data_ptr<int32_t>())
            : call(pad_paged_attention_decode_weights, num_new),
        "decode_weights");
  return out;
}

at::Tensor decode_fp4(const at::Tensor& q_in, const at::Tensor& k, const at::Tensor& ks, const at::Tensor& v,
                      const at::Tensor& vs, const at::Tensor& bt_in, const at::Tensor& sl_in, int64_t num_splits,
                      double scale, const c10::optional<at::Tensor>& out_in, const c10::optional<at::Tensor>& weights,
                      int64_t num_new, const c10::optional<at::Tensor>& positions,
                      const c10::optional<at::Tensor>& total_in, const c10::optional<at::Tensor>& num_new_in) {
  const at::Device dev = q_in.device();
  check_fp4(k, ks, v, vs, "decode_fp4");
  check_on(dev, {&k, &ks, &v, &vs}, "decode_fp4");
  TORCH_CHECK(q_in.dim() == 3 && q_in.scalar_type() == at::kHalf && q_in.size(2) == 2 * k.size(3) && k.size(2) > 0,
              "libpad_b200 decode_fp4: q must be fp16 [B, Hq, D] of the cache's head_dim");
  TORCH_CHECK(bt_in.dim() == 2 && bt_in.size(0) == q_in.size(0) && sl_in.dim() == 1 && sl_in.size(0) == q_in.size(0),
              "libpad_b200 decode_fp4: block_table must be [B, max_pages], seq_lens [B]");
  TORCH_CHECK(weights.has_value() || !positions.has_value(), "libpad_b200 decode_fp4: slot_positions need weights");
  c10::cuda::CUDAGuard guard(dev);
  const int64_t batch = q_in.size(0), hq = q_in.size(1), d = q_in.size(2), pages = k.size(0), ps = k.size(1),
                hkv = k.size(2);
  c10::optional<Tracked> tr;
  if (weights.has_value())
    tr.emplace(*weights, positions, total_in, num_new, num_new_in, pages, hkv, ps, batch, dev, "decode_fp4");
  const at::Tensor q = aligned_rows(q_in);
  const at::Tensor bt = as_int32_rows(bt_in, dev), sl = as_int32_rows(sl_in, dev);
  at::Tensor out = prepare_out(out_in, q_in);
  if (batch == 0) return out;
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  StreamState& st = state_for(dev, stream);
  const Strides qs(q), k_s(k), ks_s(ks), v_s(v), vs_s(vs), os(out);
  size_t bytes = 0;
  check(pad_decode_fp4_workspace_bytes((int)dev.index(), batch, hkv, hq / hkv, d, pages, ps, bt.size(1), num_splits,
                                       weights.has_value() ? 1 : 0, &bytes),
        "workspace size");
  const at::Tensor ws = at::empty({(int64_t)bytes}, k.options());
  auto call = [&](auto entry, auto news) {
    return entry(q.data_ptr(), k.data_ptr(), ks.data_ptr(), v.data_ptr(), vs.data_ptr(), bt.data_ptr<int32_t>(),
                 sl.data_ptr<int32_t>(), out.data_ptr(), tr ? weights->data_ptr<float>() : nullptr,
                 positions.has_value() ? positions->data_ptr<int32_t>() : nullptr, tr ? tr->total_ptr() : nullptr, news,
                 batch, hq, hkv, d, pages, ps, bt.size(1), qs.s, k_s.s, ks_s.s, v_s.s, vs_s.s, Strides(bt).s[0], os.s,
                 tr ? tr->ws.s : nullptr, tr ? tr->ps.s : nullptr, (float)scale, num_splits, ws.data_ptr(), bytes,
                 stream, st.flags.data_ptr<int32_t>());
  };
  check(tr && tr->num_new_of.defined()
            ? call(pad_paged_attention_decode_fp4_by_seq, (const int32_t*)tr->num_new_of.data_ptr<int32_t>())
            : call(pad_paged_attention_decode_fp4, num_new),
        "decode_fp4");
  return out;
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> kv_evict_plan(
    const at::Tensor& weights, const at::Tensor& bt_in, const at::Tensor& sl_in, int64_t budget, int64_t recent,
    const c10::optional<at::Tensor>& positions, const c10::optional<at::Tensor>& total_in) {
  const at::Device dev = weights.device();
  TORCH_CHECK(weights.dim() == 3 && bt_in.dim() == 2 && sl_in.dim() == 1 && sl_in.size(0) == bt_in.size(0),
              "libpad_b200 kv_evict_plan: weights must be [pages, Hkv, page_size], block_table [B, max_pages], "
              "seq_lens [B]");
  const int64_t pages = weights.size(0), hkv = weights.size(1), ps = weights.size(2), batch = bt_in.size(0);
  check_slots(weights, at::kFloat, pages, hkv, ps, "kv_evict_plan");
  TORCH_CHECK(positions.has_value() == total_in.has_value(),
              "libpad_b200 kv_evict_plan: slot_positions and total_lens go together");
  if (positions.has_value()) {
    check_slots(*positions, at::kInt, pages, hkv, ps, "kv_evict_plan");
    check_on(dev, {&*positions}, "kv_evict_plan");
    TORCH_CHECK(total_in->dim() == 1 && total_in->size(0) == batch, "libpad_b200 kv_evict_plan: total_lens must be [B]");
  }
  c10::cuda::CUDAGuard guard(dev);
  const at::Tensor bt = as_int32_rows(bt_in, dev), sl = as_int32_rows(sl_in, dev);
  const at::Tensor total = total_in.has_value() ? as_int32_rows(*total_in, dev) : at::Tensor();
  int64_t moves = 0;
  check(pad_evict_max_moves(budget, ps, bt.size(1), &moves), "kv_evict_plan");
  // one allocation for the plan, each part starting on 16 bytes; the lengths, which
  // a caller keeps, have their own
  const int64_t list = batch * hkv * moves, step = (list + 3) / 4 * 4;
  const auto opt = weights.options().dtype(at::kInt);
  const at::Tensor all = at::empty({2 * step + batch * hkv}, opt), lens = at::empty({batch}, opt);
  const at::Tensor src = all.as_strided({batch, hkv, moves}, {hkv * moves, moves, 1}, 0);
  const at::Tensor dst = all.as_strided({batch, hkv, moves}, {hkv * moves, moves, 1}, step);
  const at::Tensor counts = all.as_strided({batch, hkv}, {hkv, 1}, 2 * step);
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  StreamState& st = state_for(dev, stream);
  const Strides ws(weights), pst(positions.has_value() ? *positions : weights);
  check(pad_paged_kv_evict_plan(weights.data_ptr<float>(), positions.has_value() ? positions->data_ptr<int32_t>() : nullptr,
                                bt.data_ptr<int32_t>(), sl.data_ptr<int32_t>(),
                                total.defined() ? total.data_ptr<int32_t>() : nullptr, src.data_ptr<int32_t>(),
                                dst.data_ptr<int32_t>(), counts.data_ptr<int32_t>(), lens.data_ptr<int32_t>(), batch,
                                hkv, pages, ps, bt.size(1), budget, recent, ws.s, pst.s, Strides(bt).s[0], stream,
                                st.flags.data_ptr<int32_t>()),
        "kv_evict_plan");
  return {src, dst, counts, lens};
}

void kv_move(at::TensorList caches, const at::Tensor& bt_in, const at::Tensor& src, const at::Tensor& dst,
             const at::Tensor& counts, const c10::optional<at::Tensor>& weights,
             const c10::optional<at::Tensor>& positions) {
  TORCH_CHECK(caches.size() >= 1 && caches.size() <= 4, "libpad_b200 kv_move: 1 to 4 caches");
  const at::Tensor& first = caches[0];
  TORCH_CHECK(first.dim() == 4, "libpad_b200 kv_move: caches must be [pages, page_size, Hkv, row]");
  const at::Device dev = first.device();
  const int64_t pages = first.size(0), ps = first.size(1), hkv = first.size(2), batch = bt_in.size(0);
  void* ptr[4];
  int64_t bytes[4], strides[12];
  for (size_t c = 0; c < caches.size(); ++c) {
    const at::Tensor& t = caches[c];
    TORCH_CHECK(t.dim() == 4 && t.size(0) == pages && t.size(1) == ps && t.size(2) == hkv && Strides(t).s[3] == 1,
                "libpad_b200 kv_move: caches must be [pages, page_size, Hkv, row] with a contiguous row");
    check_on(dev, {&t}, "kv_move");
    const int64_t item = t.element_size();
    ptr[c] = t.data_ptr();
    bytes[c] = t.size(3) * item;
    const Strides st(t);
    for (int i = 0; i < 3; ++i) strides[3 * c + i] = st.s[i] * item;
  }
  TORCH_CHECK(bt_in.dim() == 2 && src.dim() == 3 && src.size(0) == batch && src.size(1) == hkv &&
                  dst.sizes() == src.sizes() && counts.dim() == 2 && counts.size(0) == batch &&
                  counts.size(1) == hkv && src.scalar_type() == at::kInt && dst.scalar_type() == at::kInt &&
                  counts.scalar_type() == at::kInt && src.is_contiguous() && dst.is_contiguous() &&
                  counts.is_contiguous(),
              "libpad_b200 kv_move: src, dst [B, Hkv, moves] and counts [B, Hkv] must be contiguous int32, as a plan "
              "returns them");
  check_on(dev, {&src, &dst, &counts}, "kv_move");
  if (weights.has_value()) {
    check_slots(*weights, at::kFloat, pages, hkv, ps, "kv_move");
    check_on(dev, {&*weights}, "kv_move");
  }
  if (positions.has_value()) {
    check_slots(*positions, at::kInt, pages, hkv, ps, "kv_move");
    check_on(dev, {&*positions}, "kv_move");
  }
  c10::cuda::CUDAGuard guard(dev);
  const at::Tensor bt = as_int32_rows(bt_in, dev);
  cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  StreamState& st = state_for(dev, stream);
  const Strides ws(weights.has_value() ? *weights : src), pst(positions.has_value() ? *positions : src);
  check(pad_paged_kv_move((int64_t)caches.size(), ptr, bytes, strides, bt.data_ptr<int32_t>(), src.data_ptr<int32_t>(),
                          dst.data_ptr<int32_t>(), counts.data_ptr<int32_t>(),
                          weights.has_value() ? weights->data_ptr<float>() : nullptr,
                          positions.has_value() ? positions->data_ptr<int32_t>() : nullptr, batch, hkv, pages, ps,
                          bt.size(1), src.size(2), ws.s, pst.s, Strides(bt).s[0], stream, st.flags.data_ptr<int32_t>()),
        "kv_move");
}

// The error-flag word of `device`'s current stream (the kernels OR
// PAD_FLAG_* bits into it; the caller reads and clears it).
at::Tensor error_flags(int64_t device) {
  const at::Device dev(at::kCUDA, (c10::DeviceIndex)device);
  c10::cuda::CUDAGuard guard(dev);
  return state_for(dev, c10::cuda::getCurrentCUDAStream(dev.index()).stream()).flags;
}

}  // namespace

TORCH_LIBRARY(pad_b200, m) {
  m.def("decode(Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_table, Tensor seq_lens, int num_splits, "
        "float scale, Tensor(a!)? out) -> Tensor");
  m.def("decode_csr(Tensor q, Tensor k_cache, Tensor v_cache, Tensor kv_indptr, Tensor kv_indices, "
        "Tensor kv_last_page_len, int num_splits, float scale, Tensor(a!)? out) -> Tensor");
  m.def("kv_append(Tensor k_new, Tensor v_new, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor block_table, "
        "Tensor positions) -> ()");
  m.def("decode_weights(Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_table, Tensor seq_lens, int num_splits, "
        "float scale, Tensor(a!)? out, Tensor(b!) weights, int num_new, Tensor(c!)? slot_positions, "
        "Tensor? total_lens, Tensor? num_new_of=None) -> Tensor");
  m.def("decode_fp4(Tensor q, Tensor k_cache, Tensor k_scales, Tensor v_cache, Tensor v_scales, Tensor block_table, "
        "Tensor seq_lens, int num_splits, float scale, Tensor(a!)? out, Tensor(b!)? weights, int num_new, "
        "Tensor(c!)? slot_positions, Tensor? total_lens, Tensor? num_new_of=None) -> Tensor");
  m.def("kv_append_fp4(Tensor k_new, Tensor v_new, Tensor(a!) k_cache, Tensor(b!) k_scales, Tensor(c!) v_cache, "
        "Tensor(d!) v_scales, Tensor block_table, Tensor positions, Tensor? seq_ids) -> ()");
  m.def("kv_read_fp4(Tensor k_cache, Tensor k_scales, Tensor v_cache, Tensor v_scales, Tensor block_table, "
        "Tensor positions, Tensor? seq_ids) -> (Tensor, Tensor)");
  m.def("kv_evict_plan(Tensor weights, Tensor block_table, Tensor seq_lens, int budget, int recent, "
        "Tensor? slot_positions, Tensor? total_lens) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("kv_move(Tensor(a!)[] caches, Tensor block_table, Tensor src, Tensor dst, Tensor counts, "
        "Tensor(b!)? weights, Tensor(c!)? slot_positions) -> ()");
  m.def("error_flags(int device) -> Tensor", &error_flags);
}

TORCH_LIBRARY_IMPL(pad_b200, CUDA, m) {
  m.impl("decode", &decode);
  m.impl("decode_csr", &decode_csr);
  m.impl("kv_append", &kv_append);
  m.impl("decode_weights", &decode_weights);
  m.impl("decode_fp4", &decode_fp4);
  m.impl("kv_append_fp4", &kv_append_fp4);
  m.impl("kv_read_fp4", &kv_read_fp4);
  m.impl("kv_evict_plan", &kv_evict_plan);
  m.impl("kv_move", &kv_move);
}
