// The short calls' host path: argument checks, allocations and launches of one call without going back to Python in
// between. A one-token decode is a few microseconds of device work, and the same sequence in Python (views, shape
// comparisons, a 20-argument foreign call) took 34 us, a layer step of it 165 us.
//
// Every function takes the plain case only -- dense, aligned CUDA tensors of the expected shapes and types on the
// current device -- and returns None for anything else, so that the general path in Python handles it or raises the
// error that belongs to it. Nothing is kept between calls.
#include <atomic>

#include <ATen/ATen.h>
#include <ATen/TracerMode.h>
#include <ATen/autocast_mode.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/AutogradState.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/utils/pybind.h>

#include "../../../include/gdn2_b200.h"

namespace py = pybind11;
using at::Tensor;

namespace {

// a tensor of this dtype on the current device, not wrapped by a transform or a subclass
bool unwrapped(const Tensor& t, at::ScalarType dt, c10::DeviceIndex dev) {
  return t.defined() && t.is_cuda() && t.get_device() == dev && t.scalar_type() == dt &&
         !t.is_conj() && !t.is_neg() && t.key_set().has(c10::DispatchKey::CUDA) && !t.key_set().has(c10::DispatchKey::Python) &&
         !t.key_set().has(c10::DispatchKey::FuncTorchBatched) && !t.key_set().has(c10::DispatchKey::FuncTorchGradWrapper) &&
         !t.key_set().has(c10::DispatchKey::Functionalize);
}
// dense and 16-byte aligned
bool dense(const Tensor& t) { return t.is_contiguous() && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0; }
bool plain(const Tensor& t, at::ScalarType dt, c10::DeviceIndex dev) { return unwrapped(t, dt, dev) && dense(t); }

int dtype_code(at::ScalarType dt) {
  return dt == at::kBFloat16 ? GDN2_BF16 : dt == at::kHalf ? GDN2_F16 : dt == at::kFloat ? GDN2_F32 : -1;
}

struct Problem {
  int64_t B, S, H, HK, DK, DV;
  int dtype;
  at::ScalarType type;
  c10::DeviceIndex dev;
};

// q, k, b, g [.., HK, DK] and v, w [.., H, DV] with `lead` leading dimensions (batch, and tokens when lead == 2)
bool plain_tokens(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& b, const Tensor& w, Problem& p,
                  int64_t lead) {
  if (q.dim() != lead + 2 || v.dim() != lead + 2 || !q.is_cuda()) return false;
  p.type = q.scalar_type();
  p.dtype = dtype_code(p.type);
  p.dev = c10::cuda::current_device();
  if (p.dtype < 0 || !plain(q, p.type, p.dev) || !plain(k, p.type, p.dev) || !plain(v, p.type, p.dev) || !plain(b, p.type, p.dev) ||
      !plain(w, p.type, p.dev) || !plain(g, at::kFloat, p.dev))
    return false;
  const auto qs = q.sizes(), vs = v.sizes();
  if (k.sizes() != qs || b.sizes() != qs || g.sizes() != qs || w.sizes() != vs) return false;
  p.B = qs[0];
  p.S = lead == 2 ? qs[1] : 1;
  if (vs[0] != p.B || (lead == 2 && vs[1] != p.S)) return false;
  p.HK = qs[lead]; p.DK = qs[lead + 1];
  p.H = vs[lead]; p.DV = vs[lead + 1];
  return p.B > 0 && p.S > 0 && p.HK > 0 && p.DK > 0 && p.DV > 0 && p.H > 0 && p.H % p.HK == 0;
}

bool plain_state(const Tensor& s, const Problem& p) {
  return plain(s, at::kFloat, p.dev) && s.dim() == 4 && s.size(0) == p.B && s.size(1) == p.H && s.size(2) == p.DK && s.size(3) == p.DV;
}

void* stream_of(const Problem& p) { return c10::cuda::getCurrentCUDAStream(p.dev).stream(); }

// gdn2_decode ([B, n, H, D] tokens) and gdn2_decode_step ([B, H, D]); the state is updated in place. Returns o or None.
std::optional<Tensor> decode(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& b, const Tensor& w,
                  const Tensor& state, std::optional<double> scale) {
  Problem p;
  if (!plain_tokens(q, k, v, g, b, w, p, q.dim() == 3 ? 1 : 2) || !plain_state(state, p)) return std::nullopt;
  Tensor o = at::empty(v.sizes(), v.options().requires_grad(false));
  const float sc = scale ? (float)*scale : (float)(1.0 / std::sqrt((double)p.DK));
  const int rc = gdn2_decode(q.data_ptr(), k.data_ptr(), v.data_ptr(), static_cast<const float*>(g.data_ptr()), b.data_ptr(),
                             w.data_ptr(), static_cast<float*>(state.data_ptr()), o.data_ptr(), p.B, p.S, p.H, p.HK, p.DK, p.DV,
                             p.S, p.S, sc, p.dtype, stream_of(p));
  if (rc != GDN2_OK) return std::nullopt;
  return o;
}

// Whether a prefill of at least 64 tokens is one call of gdn2_prefill_ragged: resolves `path` and gives its workspace
bool ragged_plan(const Problem& p, int& path, size_t& bytes) {
  const int64_t n_full = p.S / 64 * 64;
  if (path == GDN2_PATH_AUTO) path = p.DK == 128 && p.DV == 128 && p.dtype == GDN2_BF16 ? GDN2_PATH_TCGEN05 : GDN2_PATH_SIMT;
  // the caller overlaps the stages of long, uncut problems segment by segment
  if (path != GDN2_PATH_SIMT && n_full / 64 >= 32 && gdn2_prefill_scan_segments(p.B, n_full, p.H, p.DK, p.DV, p.dtype, path) <= 1)
    return false;
  bytes = gdn2_prefill_ragged_workspace_bytes(p.B, p.S, p.H, p.HK, p.DK, p.DV, p.dtype, path);
  return bytes != 0;
}
int64_t ragged_launches(const Problem& p, int path) {
  const int64_t n_full = p.S / 64 * 64;
  const bool tc = path != GDN2_PATH_SIMT;
  const int64_t scans = gdn2_prefill_scan_launches(p.B, n_full, p.H, p.DK, p.DV, p.dtype, path);
  return (tc ? 2 : 1) + scans + (tc && p.S > n_full);
}

// gdn2_prefill_ragged. `side`: the second stream (0: none). Returns (o, final state, kernels launched) or None.
std::optional<std::tuple<Tensor, Tensor, int64_t>> prefill(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& b, const Tensor& w,
                   std::optional<double> scale, const std::optional<Tensor>& state, int path, uint64_t side) {
  Problem p;
  if (q.dim() != 4 || !plain_tokens(q, k, v, g, b, w, p, 2)) return std::nullopt;
  if (state && !plain_state(*state, p)) return std::nullopt;
  size_t bytes = 0;
  if (p.S < 64 || !ragged_plan(p, path, bytes)) return std::nullopt;
  const auto opt = v.options().requires_grad(false);
  Tensor ws = at::empty({(int64_t)bytes}, opt.dtype(at::kByte));
  Tensor o = at::empty(v.sizes(), opt);
  Tensor fin = at::empty({p.B, p.H, p.DK, p.DV}, opt.dtype(at::kFloat));
  const float sc = scale ? (float)*scale : (float)(1.0 / std::sqrt((double)p.DK));
  const int rc = gdn2_prefill_ragged(
      q.data_ptr(), k.data_ptr(), v.data_ptr(), static_cast<const float*>(g.data_ptr()), b.data_ptr(), w.data_ptr(),
      state ? static_cast<const float*>(state->data_ptr()) : nullptr, o.data_ptr(), static_cast<float*>(fin.data_ptr()), ws.data_ptr(),
      bytes, p.B, p.S, p.H, p.HK, p.DK, p.DV, p.S, p.S, sc, p.dtype, path, p.S % 64 ? reinterpret_cast<void*>(side) : nullptr,
      stream_of(p));
  if (rc != GDN2_OK) return std::nullopt;
  return std::make_tuple(o, fin, ragged_launches(p, path));
}


// gdn2_prefill of a prompt shorter than a chunk: the decode of its tokens, `state` updated in place and returned (none: from zero).
// Returns (o, state) or None.
std::optional<std::tuple<Tensor, Tensor>> prefill_short(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& b,
                                                        const Tensor& w, std::optional<double> scale, const std::optional<Tensor>& state) {
  Problem p;
  if (q.dim() != 4 || !plain_tokens(q, k, v, g, b, w, p, 2) || p.S >= 64 || p.DK > 256) return std::nullopt;
  if (state && !plain_state(*state, p)) return std::nullopt;
  const auto opt = v.options().requires_grad(false);
  Tensor o = at::empty(v.sizes(), opt);
  Tensor st = state ? *state : at::zeros({p.B, p.H, p.DK, p.DV}, opt.dtype(at::kFloat));
  const float sc = scale ? (float)*scale : (float)(1.0 / std::sqrt((double)p.DK));
  const int rc = gdn2_decode_tail(q.data_ptr(), k.data_ptr(), v.data_ptr(), static_cast<const float*>(g.data_ptr()), b.data_ptr(), w.data_ptr(),
                                  static_cast<float*>(st.data_ptr()), o.data_ptr(), p.B, p.S, p.H, p.HK, p.DK, p.DV, p.S, p.S, sc, p.dtype,
                                  stream_of(p));
  if (rc != GDN2_OK) return std::nullopt;
  return std::make_tuple(o, st);
}

// What the layer's calls below share: x [B, n, hidden], the cache, the layer's tensors and sizes.
struct Layer {
  const Tensor &state, &w_cat, &A_log, &dt_bias, &norm_w, &o_w;
  const std::optional<Tensor> &conv_state, &conv_w, &conv_b;
  const std::vector<int64_t>& offs;
  int64_t H, HK, DK, DV, K;
  double erase_scale, eps, scale;
  int64_t CC() const { return 2 * HK * DK + H * DV; }       // convolved channels
};

bool plain_layer(Tensor& x, const Layer& l, Problem& p) {
  p.type = x.scalar_type();
  p.dtype = dtype_code(p.type);
  if (p.dtype < 0 || x.dim() != 3 || !x.is_cuda() || x.numel() == 0 || l.DK > 256 || l.DV > 256 || l.offs.size() != 7) return false;
  p.dev = c10::cuda::current_device();
  p.B = x.size(0); p.S = x.size(1); p.H = l.H; p.HK = l.HK; p.DK = l.DK; p.DV = l.DV;
  for (const Tensor* t : {&l.w_cat, &l.A_log, &l.dt_bias, &l.norm_w, &l.o_w})
    if (!plain(*t, p.type, p.dev)) return false;
  // one token out of a prompt that lies in memory whole (x[:, t]): its rows are brought together
  if (p.S == 1 && unwrapped(x, p.type, p.dev) && !dense(x)) x = x.clone(at::MemoryFormat::Contiguous);
  if (!plain(x, p.type, p.dev) || !plain_state(l.state, p) || x.size(2) != l.w_cat.size(1)) return false;
  return l.K >= 2 && l.conv_w && plain(*l.conv_w, p.type, p.dev) && (!l.conv_b || plain(*l.conv_b, p.type, p.dev)) && l.conv_state &&
         plain(*l.conv_state, p.type, p.dev) && l.conv_state->dim() == 3 && l.conv_state->size(0) == p.B &&
         l.conv_state->size(1) == l.CC() && l.conv_state->size(2) == l.K - 1;
}

// The layer stage by stage: projections, gdn2_layer_front, `attend` on the buffers of its inputs and output (true: done),
// gdn2_layer_back, output projection. Returns (out, new convolution cache, kernels of the front and the back launched) or None
// while nothing of the cache has changed, so that the general path can still take the call over.
struct Stages { char *q, *k, *b, *v, *w, *o; float* g; };
template <typename Attend>
std::optional<std::tuple<Tensor, Tensor, int64_t>> layer_stages(const Tensor& x, const Layer& l, const Problem& p, Attend attend) {
  Tensor proj = at::linear(x, l.w_cat);
  if (proj.scalar_type() != p.type || !proj.is_contiguous()) return std::nullopt;       // an autocast region
  const auto opt = x.options().requires_grad(false);
  // one allocation for what lives between the stages, every part 256-byte aligned
  const int64_t esz = p.dtype == GDN2_F32 ? 4 : 2, tokens = p.B * p.S;
  auto part = [](int64_t bytes) { return (bytes + 255) / 256 * 256; };
  const int64_t key = part(tokens * l.HK * l.DK * esz), decay = part(tokens * l.HK * l.DK * 4), value = part(tokens * l.H * l.DV * esz);
  Tensor mid = at::empty({3 * key + decay + 3 * value}, opt.dtype(at::kByte));
  Tensor conv = at::empty({p.B, l.CC(), l.K - 1}, opt);
  char* at_ = static_cast<char*>(mid.data_ptr());
  auto take = [&](int64_t bytes) { char* r = at_; at_ += bytes; return r; };
  Stages m;
  m.q = take(key); m.k = take(key); m.b = take(key); m.g = reinterpret_cast<float*>(take(decay));
  m.v = take(value); m.w = take(value); m.o = take(value);
  void* st = stream_of(p);
  gdn2_layer_front_args a{};
  a.proj = proj.data_ptr(); a.conv_state = l.conv_state->data_ptr(); a.conv_weight = l.conv_w->data_ptr();
  a.conv_bias = l.conv_b ? l.conv_b->data_ptr() : nullptr;
  a.A_log = l.A_log.data_ptr(); a.dt_bias = l.dt_bias.data_ptr();
  a.q = m.q; a.k = m.k; a.v = m.v; a.g = m.g; a.b = m.b; a.w = m.w; a.new_conv_state = conv.data_ptr();
  a.B = p.B; a.S = p.S; a.H = l.H; a.HK = l.HK; a.DK = l.DK; a.DV = l.DV; a.K = l.K; a.NP = proj.size(2);
  a.off_q = l.offs[0]; a.off_k = l.offs[1]; a.off_v = l.offs[2]; a.off_b = l.offs[3]; a.off_w = l.offs[4]; a.off_f = l.offs[5];
  a.erase_scale = (float)l.erase_scale;
  if (gdn2_layer_front(&a, p.dtype, st) != GDN2_OK || !attend(m)) return std::nullopt;
  Tensor normed = at::empty({p.B, p.S, l.H * l.DV}, opt);   // now, where the scan's workspace was
  const int rc = gdn2_layer_back(m.o, proj.data_ptr(), l.norm_w.data_ptr(), normed.data_ptr(), p.B * p.S, l.H, l.DV,
                                 proj.size(2), l.offs[6], (float)l.eps, p.dtype, st);
  if (rc != GDN2_OK) throw std::runtime_error(std::string("gdn2_layer_back: ") + gdn2_status_string(rc));
  // the front kernel writes the new convolution cache itself in its 16-bit forms, else a second one does
  bool fused = p.dtype != GDN2_F32 && l.DK == 128 && l.DV == 128 && l.K == 4 && a.NP % 4 == 0;
  for (int i = 0; i < 6; ++i) fused = fused && l.offs[i] % 4 == 0;
  return std::make_tuple(at::linear(normed, l.o_w), conv, int64_t(fused ? 2 : 3));
}

// GatedDeltaNet2.decode on x [B, n, hidden]: gdn2_layer_step where it applies, else stage by stage. The recurrent state is updated
// in place. Returns (out [B, n, hidden], new convolution cache, kernels launched) or None. `conv_in_place`: the convolution
// cache is updated in place too, or the call is not made.
std::optional<std::tuple<Tensor, Tensor, int64_t>> layer_decode(Tensor x, const Tensor& state, const std::optional<Tensor>& conv_state, const Tensor& w_cat,
                        const std::optional<Tensor>& conv_w, const std::optional<Tensor>& conv_b, const Tensor& A_log,
                        const Tensor& dt_bias, const Tensor& norm_w, const Tensor& o_w, const std::vector<int64_t>& offs, int64_t H,
                        int64_t HK, int64_t DK, int64_t DV, int64_t K, double erase_scale, double eps, double scale, bool conv_in_place) {
  const Layer l{state, w_cat, A_log, dt_bias, norm_w, o_w, conv_state, conv_w, conv_b, offs, H, HK, DK, DV, K, erase_scale, eps, scale};
  Problem p;
  at::NoGradGuard no_grad;
  if (!plain_layer(x, l, p)) return std::nullopt;
  const int64_t hidden = x.size(2);
  // (an autocast region or a dispatch mode would have seen the two linear layers)
  const size_t step_bytes = p.S == 1 && o_w.dim() == 2 && o_w.size(0) == hidden && o_w.size(1) == H * DV &&
                                    !at::autocast::is_autocast_enabled(at::kCUDA) && !c10::impl::TorchDispatchModeTLS::any_modes_set()
                                ? gdn2_layer_step_workspace_bytes(p.B, hidden, H, HK, DK, DV, K, p.dtype)
                                : 0;
  if (step_bytes > 0) {
    const auto opt = x.options().requires_grad(false);
    Tensor ws = at::empty({(int64_t)step_bytes}, opt.dtype(at::kByte)), out = at::empty({p.B, 1, hidden}, opt);
    Tensor conv = conv_in_place ? *conv_state : at::empty({p.B, l.CC(), K - 1}, opt);
    gdn2_layer_step_args s{};
    s.x = x.data_ptr(); s.w_cat = w_cat.data_ptr(); s.conv_state = conv_state->data_ptr(); s.conv_weight = conv_w->data_ptr();
    s.conv_bias = conv_b ? conv_b->data_ptr() : nullptr;
    s.A_log = A_log.data_ptr(); s.dt_bias = dt_bias.data_ptr(); s.norm_weight = norm_w.data_ptr(); s.o_weight = o_w.data_ptr();
    s.state = static_cast<float*>(state.data_ptr()); s.new_conv_state = conv.data_ptr(); s.out = out.data_ptr();
    s.workspace = ws.data_ptr(); s.workspace_bytes = step_bytes;
    s.B = p.B; s.hidden = hidden; s.H = H; s.HK = HK; s.DK = DK; s.DV = DV; s.K = K;
    s.off_q = offs[0]; s.off_k = offs[1]; s.off_v = offs[2]; s.off_b = offs[3]; s.off_w = offs[4]; s.off_f = offs[5]; s.off_gate = offs[6];
    s.erase_scale = (float)erase_scale; s.eps = (float)eps; s.scale = (float)scale;
    const int rc = gdn2_layer_step(&s, p.dtype, stream_of(p));
    if (rc == GDN2_OK) return std::make_tuple(out, conv, int64_t(3));
    // refused before anything ran; after a launch that failed part of the cache may have been written
    if (rc == GDN2_ERR_CUDA) throw std::runtime_error(std::string("gdn2_layer_step: ") + gdn2_status_string(rc));
  }
  if (conv_in_place) return std::nullopt;
  auto res = layer_stages(x, l, p, [&](const Stages& m) {
    return gdn2_decode(m.q, m.k, m.v, m.g, m.b, m.w, static_cast<float*>(state.data_ptr()), m.o, p.B, p.S, H, HK, DK, DV, p.S, p.S,
                       (float)scale, p.dtype, stream_of(p)) == GDN2_OK;
  });
  if (res) std::get<2>(*res) += 1;
  return res;
}

// GatedDeltaNet2.prefill on x [B, S, hidden], continuing from the cache. Returns (out [B, S, hidden], final recurrent state, new
// convolution cache, kernels launched) or None. A prompt shorter than a chunk is decoded and updates the recurrent state in
// place, as gdn2_prefill does.
std::optional<std::tuple<Tensor, Tensor, Tensor, int64_t>> layer_prefill(Tensor x, const Tensor& state, const std::optional<Tensor>& conv_state, const Tensor& w_cat,
                        const std::optional<Tensor>& conv_w, const std::optional<Tensor>& conv_b, const Tensor& A_log,
                        const Tensor& dt_bias, const Tensor& norm_w, const Tensor& o_w, const std::vector<int64_t>& offs, int64_t H,
                        int64_t HK, int64_t DK, int64_t DV, int64_t K, double erase_scale, double eps, double scale, int path, uint64_t side) {
  const Layer l{state, w_cat, A_log, dt_bias, norm_w, o_w, conv_state, conv_w, conv_b, offs, H, HK, DK, DV, K, erase_scale, eps, scale};
  Problem p;
  at::NoGradGuard no_grad;
  if (!plain_layer(x, l, p)) return std::nullopt;
  size_t bytes = 0;
  if (p.S >= 64 && !ragged_plan(p, path, bytes)) return std::nullopt;
  Tensor fin = state;
  const auto opt = x.options().requires_grad(false);
  int64_t launched = 1;
  auto res = layer_stages(x, l, p, [&](const Stages& m) {
    if (p.S < 64)
      return gdn2_decode_tail(m.q, m.k, m.v, m.g, m.b, m.w, static_cast<float*>(state.data_ptr()), m.o, p.B, p.S, H, HK, DK, DV, p.S, p.S,
                              (float)scale, p.dtype, stream_of(p)) == GDN2_OK;
    Tensor ws = at::empty({(int64_t)bytes}, opt.dtype(at::kByte));
    fin = at::empty({p.B, H, DK, DV}, opt.dtype(at::kFloat));
    launched = ragged_launches(p, path);
    return gdn2_prefill_ragged(m.q, m.k, m.v, m.g, m.b, m.w, static_cast<const float*>(state.data_ptr()), m.o, static_cast<float*>(fin.data_ptr()),
                               ws.data_ptr(), bytes, p.B, p.S, H, HK, DK, DV, p.S, p.S, (float)scale, p.dtype, path,
                               p.S % 64 ? reinterpret_cast<void*>(side) : nullptr, stream_of(p)) == GDN2_OK;
  });
  if (!res) return std::nullopt;
  return std::make_tuple(std::get<0>(*res), fin, std::get<1>(*res), std::get<2>(*res) + launched);
}

// ---------------------------------------------------------------- the differentiable operators

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

std::atomic<int64_t> g_gradient_launches{0};      // kernels launched by backward passes, which return to autograd and not to the caller

void check(int rc, const char* what) {
  if (rc != GDN2_OK)
    throw std::runtime_error(std::string(what) + ": " + gdn2_status_string(rc) +
                             (rc == GDN2_ERR_CUDA ? " (cudaError " + std::to_string(gdn2_last_cuda_error()) + ")" : "") + " [status " +
                             std::to_string(rc) + "]");
}
bool wants_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}
// An input with a forward-mode tangent: the operators have none, and the general path says so
bool has_tangent(std::initializer_list<const Tensor*> ts) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->_fw_grad(0).defined()) return true;
  return false;
}
// A tracer is at work, which would record the empty result of a kernel alone
bool traced() {
  using c10::impl::TorchDispatchModeTLS;
  using Key = c10::impl::TorchDispatchModeKey;
  if (at::tracer::impl::is_dispatch_enabled() || c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch)) return true;
  return TorchDispatchModeTLS::any_modes_set() &&
         (TorchDispatchModeTLS::get_mode(Key::PROXY) || TorchDispatchModeTLS::get_mode(Key::FAKE) || TorchDispatchModeTLS::get_mode(Key::FUNCTIONAL));
}
// A backward pass that is traced, or whose gradients carry tangents (forward mode over reverse mode)
void refuse_transforms(const variable_list& grads, const char* what) {
  TORCH_CHECK_NOT_IMPLEMENTED(!traced(), what, " cannot be traced: its gradient's kernels are not operators that a tracer sees");
  for (const Tensor& t : grads)
    TORCH_CHECK_NOT_IMPLEMENTED(!has_tangent({&t}), what, " has no forward-mode derivative (a gradient carries a tangent)");
}
// Gradients that were asked for with create_graph: there is no second derivative, and using one says so.
variable_list once(variable_list grads, const char* what) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list live;
  for (const Tensor& t : grads)
    if (t.defined()) live.push_back(t.set_requires_grad(true));      // new tensors of the pass's own, so that the error is attached
  auto error = std::make_shared<torch::autograd::DelayedError>(std::string(what) + " is differentiable once", (int64_t)live.size());
  live = (*error)(std::move(live));
  size_t i = 0;
  for (Tensor& t : grads)
    if (t.defined()) t = live[i++];
  return grads;
}
// A program's hooks may bring saved tensors back in another layout, which the backward passes lay out again; with another type, shape
// or device they are no longer what the kernels read.
bool saved_as(const Tensor& t, const Tensor& like, at::ScalarType type, at::IntArrayRef sizes) {
  return t.defined() && t.layout() == at::kStrided && t.device() == like.device() && t.scalar_type() == type && t.sizes() == sizes &&
         !t.is_conj() && !t.is_neg();
}
void check_saved(bool ok, const char* what) {
  TORCH_CHECK(ok, what, ": a saved tensor came back from a hook with another type, shape or device");
}
void* stream_on(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }
template <typename T> T* ptr(const Tensor& t) { return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr; }

// [B, S, ...] as rows [B, S, D] whose channels lie side by side, or an undefined tensor
Tensor as_rows(const Tensor& t) {
  if (t.dim() < 3) return Tensor();
  Tensor r = t.dim() == 3 ? t : t.is_contiguous() ? t.view({t.size(0), t.size(1), -1}) : Tensor();
  if (r.defined() && r.size(2) > 1 && r.stride(2) != 1) return Tensor();
  return r;
}
void set_rows(const Tensor& t, const void** p, int64_t* batch, int64_t* token) {
  *p = t.data_ptr();
  *batch = t.size(0) > 1 ? t.stride(0) : 0;
  *token = t.size(1) > 1 ? t.stride(1) : 0;
}
gdn2_recurrence_args recurrence_args(const Tensor& v, const Tensor& g, const Tensor& w, const std::vector<int64_t>& offsets) {
  gdn2_recurrence_args a{};
  const void* pg = nullptr;
  set_rows(v, &a.v, &a.v_batch_stride, &a.v_token_stride);
  set_rows(g, &pg, &a.g_batch_stride, &a.g_token_stride);
  a.g = static_cast<const float*>(pg);
  if (w.defined()) set_rows(w, &a.w, &a.w_batch_stride, &a.w_token_stride);
  a.B = v.size(0); a.S = v.size(1); a.D = v.size(2);
  a.sequences = offsets.empty() ? a.B : (int64_t)offsets.size() - 1;
  a.cu_seqlens = offsets.empty() ? nullptr : offsets.data();
  return a;
}
int64_t recurrence_launches(const gdn2_recurrence_args& a) { return a.cu_seqlens ? (a.sequences + 127) / 128 : 1; }

struct Recurrence : torch::autograd::Function<Recurrence> {
  static variable_list forward(AutogradContext* ctx, const Tensor& v, const Tensor& g, const std::optional<Tensor>& gate,
                               const std::optional<Tensor>& initial, const std::vector<int64_t>& offsets) {
    const Tensor w = gate.value_or(Tensor()), state = initial.value_or(Tensor());
    gdn2_recurrence_args a = recurrence_args(v, g, w, offsets);
    const auto opt = v.options().requires_grad(false);
    Tensor o = at::empty(v.sizes(), opt), final = at::empty({a.sequences, a.D}, opt.dtype(at::kFloat));
    Tensor marks = at::empty({(int64_t)gdn2_recurrence_marks(a.B, a.S, a.cu_seqlens, a.sequences), a.D}, opt.dtype(at::kFloat));
    a.state = ptr<float>(state); a.o = o.data_ptr(); a.final_state = ptr<float>(final); a.marks = ptr<float>(marks);
    check(gdn2_recurrence_forward(&a, dtype_code(v.scalar_type()), stream_on(v)), "gdn2_recurrence_forward");
    ctx->save_for_backward({v, g, w, marks});
    ctx->saved_data["offsets"] = offsets;
    ctx->saved_data["state"] = state.defined();
    ctx->set_materialize_grads(false);
    return {o, final};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined() && !grads[1].defined()) return variable_list(5);
    refuse_transforms(grads, "gated_recurrence");
    const auto saved = ctx->get_saved_variables();
    variable_list out(5);
    {
      at::NoGradGuard no_grad;
      const auto rows = [](const Tensor& t) { return t.defined() && t.dim() == 3 && t.size(2) > 1 && t.stride(2) != 1 ? t.contiguous() : t; };
      const Tensor v = rows(saved[0]), g = rows(saved[1]), w = rows(saved[2]), marks = saved[3].contiguous();
      const Tensor& given = grads[0].defined() ? grads[0] : grads[1];
      const std::vector<int64_t> offsets = ctx->saved_data["offsets"].toIntVector();
      check_saved(v.dim() == 3 && saved_as(v, given, v.scalar_type(), v.sizes()) && dtype_code(v.scalar_type()) >= 0 &&
                      (!grads[0].defined() || saved_as(v, given, grads[0].scalar_type(), grads[0].sizes())) &&
                      saved_as(g, given, at::kFloat, v.sizes()) && (!w.defined() || saved_as(w, given, v.scalar_type(), v.sizes())),
                  "gated_recurrence");
      const c10::cuda::CUDAGuard device(v.device());
      gdn2_recurrence_args a = recurrence_args(v, g, w, offsets);
      check_saved(saved_as(marks, given, at::kFloat, {(int64_t)gdn2_recurrence_marks(a.B, a.S, a.cu_seqlens, a.sequences), a.D}) &&
                      (!grads[1].defined() || (grads[1].dim() == 2 && grads[1].size(0) == a.sequences && grads[1].size(1) == a.D)),
                  "gated_recurrence");
      const auto opt = v.options().requires_grad(false);
      Tensor dout = grads[0].defined() ? grads[0] : at::zeros(v.sizes(), opt);
      if (dout.size(2) > 1 && dout.stride(2) != 1) dout = dout.contiguous();
      const Tensor dfinal = grads[1].defined() ? grads[1].contiguous() : Tensor();
      out[0] = at::empty(v.sizes(), opt);
      out[1] = at::empty(v.sizes(), opt.dtype(at::kFloat));
      if (w.defined()) out[2] = at::empty(v.sizes(), opt);
      if (ctx->saved_data["state"].toBool()) out[3] = at::empty({a.sequences, a.D}, opt.dtype(at::kFloat));
      set_rows(dout, &a.dout, &a.do_batch_stride, &a.do_token_stride);
      a.marks = ptr<float>(marks); a.dfinal_state = ptr<float>(dfinal);
      a.dv = out[0].data_ptr(); a.dg = ptr<float>(out[1]); a.dw = ptr<void>(out[2]); a.dstate = ptr<float>(out[3]);
      check(gdn2_recurrence_backward(&a, dtype_code(v.scalar_type()), stream_on(v)), "gdn2_recurrence_backward");
      g_gradient_launches += recurrence_launches(a);
    }
    return once(std::move(out), "gated_recurrence");
  }
};

// gated_recurrence on tensors of matching shapes and types (`offsets`: of packed sequences, or empty), and with `in_place`
// gated_recurrence_decode. Returns (o, final state, kernels launched) or None.
std::optional<std::tuple<Tensor, std::optional<Tensor>, int64_t>> recurrence(const Tensor& v, const Tensor& g, const std::optional<Tensor>& w,
                                                                             const std::optional<Tensor>& state, bool want_final,
                                                                             bool in_place, const std::vector<int64_t>& offsets) {
  const auto dev = c10::cuda::current_device();
  if (dtype_code(v.scalar_type()) < 0 || !unwrapped(v, v.scalar_type(), dev) || !unwrapped(g, at::kFloat, dev) || g.sizes() != v.sizes() ||
      v.numel() == 0 || (w && (!unwrapped(*w, v.scalar_type(), dev) || w->sizes() != v.sizes())))
    return std::nullopt;
  const Tensor vr = as_rows(v), gr = as_rows(g), wr = w ? as_rows(*w) : Tensor();
  if (!vr.defined() || !gr.defined() || (w && !wr.defined())) return std::nullopt;
  const int64_t sequences = offsets.empty() ? v.size(0) : (int64_t)offsets.size() - 1;
  std::vector<int64_t> state_shape(v.sizes().begin() + 1, v.sizes().end());
  state_shape[0] = sequences;
  if (state && (!unwrapped(*state, at::kFloat, dev) || !state->is_contiguous() || state->sizes() != at::IntArrayRef(state_shape)))
    return std::nullopt;
  const Tensor s = state ? state->view({sequences, -1}) : Tensor();
  if (has_tangent({&vr, &gr, &wr, &s}) || traced()) return std::nullopt;
  const bool grad = wants_grad({&vr, &gr, &wr, &s});
  if (in_place && (grad || !state)) return std::nullopt;
  if (grad) {
    const auto given = [](const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; };
    auto res = Recurrence::apply(vr, gr, given(wr), given(s), offsets);
    const int64_t launched = offsets.empty() ? 1 : (sequences + 127) / 128;
    return std::make_tuple(res[0].view(v.sizes()), want_final ? std::optional<Tensor>(res[1].view(state_shape)) : std::nullopt, launched);
  }
  gdn2_recurrence_args a = recurrence_args(vr, gr, wr, offsets);
  const auto opt = v.options().requires_grad(false);
  Tensor o = at::empty(v.sizes(), opt);
  std::optional<Tensor> final;
  if (in_place) final = *state;
  else if (want_final) final = at::empty(state_shape, opt.dtype(at::kFloat));
  a.state = ptr<float>(s); a.o = o.data_ptr(); a.final_state = final ? ptr<float>(*final) : nullptr;
  if (gdn2_recurrence_forward(&a, dtype_code(v.scalar_type()), stream_on(v)) != GDN2_OK) return std::nullopt;
  if (in_place && !state->is_inference()) state->unsafeGetTensorImpl()->bump_version();     // autograd sees that it was written
  return std::make_tuple(o, final, recurrence_launches(a));
}

// Matrices as the tensor-core kernels read them: rows that start on 16 bytes, elements side by side. Those that are not so are
// copied, all in one launch. Returns whether one was.
bool align_rows(std::vector<Tensor>& ms) {
  std::vector<gdn2_row_copy> copies;
  std::vector<Tensor> sources;                       // alive until the launch: a next operand's memory must not be one's source
  for (Tensor& t : ms) {
    if (t.size(1) > 1 && t.stride(1) != 1) t = t.contiguous();
    const bool one = t.size(0) == 1;
    if ((reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) || (!one && (t.stride(0) % 8 || t.stride(0) < t.size(1)))) {
      const int64_t pitch = (t.size(1) + 7) / 8 * 8;
      Tensor d = at::empty({t.size(0), pitch}, t.options().requires_grad(false)).narrow(1, 0, t.size(1));
      copies.push_back({t.data_ptr(), d.data_ptr(), t.size(0), t.size(1), one ? 0 : t.stride(0), pitch});
      sources.push_back(t);
      t = d;
    }
  }
  if (copies.empty()) return false;
  check(gdn2_align_rows(copies.data(), (int64_t)copies.size(), stream_on(ms[0])), "gdn2_align_rows");
  return true;
}
int64_t pitch_of(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : (t.size(1) + 7) / 8 * 8; }
gdn2_ffn_args ffn_args(const std::vector<Tensor>& in, int64_t activation) {
  gdn2_ffn_args a{};
  a.x = in[0].data_ptr(); a.w_gate = in[1].data_ptr(); a.w_up = in[2].data_ptr(); a.w_down = in[3].data_ptr();
  a.tokens = in[0].size(0); a.hidden = in[0].size(1); a.out = in[3].size(0); a.inner = in[3].size(1);
  a.x_stride = pitch_of(in[0]); a.w_gate_stride = pitch_of(in[1]); a.w_up_stride = pitch_of(in[2]); a.w_down_stride = pitch_of(in[3]);
  a.inner_stride = (a.inner + 15) / 16 * 16;
  a.activation = (int)activation;
  return a;
}
Tensor ffn_forward(const std::vector<Tensor>& in, int64_t activation, Tensor* kept) {
  gdn2_ffn_args a = ffn_args(in, activation);
  const auto opt = in[0].options().requires_grad(false);
  Tensor y = at::empty({a.tokens, a.out}, opt), h = at::empty({a.tokens, a.inner_stride}, opt);
  if (kept) *kept = at::empty({(int64_t)gdn2_ffn_kept_bytes(a.tokens, a.inner_stride)}, opt.dtype(at::kByte));
  a.h = h.data_ptr(); a.kept = kept ? kept->data_ptr() : nullptr; a.y = y.data_ptr(); a.y_stride = a.out;
  check(gdn2_ffn_forward(&a, dtype_code(in[0].scalar_type()), stream_on(in[0])), "gdn2_ffn_forward");
  return y;
}

struct FeedForward : torch::autograd::Function<FeedForward> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd, int64_t activation) {
    std::vector<Tensor> in{x, wg, wu, wd};
    align_rows(in);
    Tensor kept, y = ffn_forward(in, activation, &kept);
    ctx->save_for_backward({in[0], in[1], in[2], in[3], kept});
    ctx->saved_data["activation"] = activation;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    variable_list out(5);
    if (!grads[0].defined()) return out;
    refuse_transforms(grads, "gated_feed_forward");
    {
      at::NoGradGuard no_grad;
      std::vector<Tensor> in(saved.begin(), saved.begin() + 4);
      std::vector<Tensor> dy{grads[0]};
      bool ok = true;
      for (const Tensor& t : in) ok = ok && t.dim() == 2 && saved_as(t, dy[0], dy[0].scalar_type(), t.sizes());
      check_saved(ok && in[1].size(1) == in[0].size(1) && in[2].sizes() == in[1].sizes() && in[3].size(1) == in[1].size(0) &&
                      dy[0].sizes() == at::IntArrayRef({in[0].size(0), in[3].size(0)}),
                  "gated_feed_forward");
      const c10::cuda::CUDAGuard device(in[0].device());
      const int copied = (int)align_rows(dy) + (int)align_rows(in);
      gdn2_ffn_args a = ffn_args(in, ctx->saved_data["activation"].toInt());
      const Tensor kept = saved[4].contiguous();
      check_saved(saved_as(kept, dy[0], at::kByte, {(int64_t)gdn2_ffn_kept_bytes(a.tokens, a.inner_stride)}), "gated_feed_forward");
      const auto opt = in[0].options().requires_grad(false);
      const bool dx = ctx->needs_input_grad(0), dgate = ctx->needs_input_grad(1), dup = ctx->needs_input_grad(2), ddown = ctx->needs_input_grad(3);
      const Tensor h = at::empty({a.tokens, a.inner_stride}, opt), da = at::empty_like(h), du = at::empty_like(h);
      if (dx) out[0] = at::empty({a.tokens, a.hidden}, opt);
      if (dgate || dup) {
        out[1] = at::empty({a.inner, a.hidden}, opt);
        out[2] = at::empty({a.inner, a.hidden}, opt);
      }
      if (ddown) out[3] = at::empty({a.out, a.inner}, opt);
      a.h = h.data_ptr(); a.kept = kept.data_ptr(); a.dy = dy[0].data_ptr(); a.dy_stride = pitch_of(dy[0]);
      a.da = da.data_ptr(); a.du = du.data_ptr(); a.dx = ptr<void>(out[0]); a.dx_stride = a.hidden;
      a.dw_gate = ptr<void>(out[1]); a.dw_up = ptr<void>(out[2]); a.dw_down = ptr<void>(out[3]);
      check(gdn2_ffn_backward(&a, dtype_code(in[0].scalar_type()), stream_on(in[0])), "gdn2_ffn_backward");
      g_gradient_launches += 1 + copied + dx + (dgate || dup) + ddown;
      if (!dgate) out[1] = Tensor();
      if (!dup) out[2] = Tensor();
    }
    return once(std::move(out), "gated_feed_forward");
  }
};

// gated_feed_forward on tensors of matching shapes and types. Returns (y, kernels launched) or None.
std::optional<std::tuple<Tensor, int64_t>> feed_forward(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd, int64_t activation) {
  const auto dev = c10::cuda::current_device();
  const auto type = x.scalar_type();
  if ((type != at::kBFloat16 && type != at::kHalf) || !unwrapped(x, type, dev) || !unwrapped(wg, type, dev) || !unwrapped(wu, type, dev) ||
      !unwrapped(wd, type, dev) || x.dim() < 1 || wg.dim() != 2 || wd.dim() != 2 || wu.sizes() != wg.sizes() || wd.size(1) != wg.size(0) ||
      x.size(-1) != wg.size(1) || x.numel() == 0 || wg.numel() == 0 || wd.numel() == 0 || !(x.dim() == 2 || x.is_contiguous()))
    return std::nullopt;
  if (has_tangent({&x, &wg, &wu, &wd}) || traced()) return std::nullopt;
  const Tensor rows = x.dim() == 2 ? x : x.view({-1, x.size(-1)});
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = wd.size(0);
  if (wants_grad({&rows, &wg, &wu, &wd})) return std::make_tuple(FeedForward::apply(rows, wg, wu, wd, activation).view(shape), int64_t(2));
  std::vector<Tensor> in{rows, wg, wu, wd};
  const bool copied = align_rows(in);
  return std::make_tuple(ffn_forward(in, activation, nullptr).view(shape), int64_t(2) + copied);
}

// The state of a list of parameters: where each lies, its version and its type. Equal bytes = nothing was replaced,
// moved, converted or written to since.
py::bytes parameter_key(const std::vector<Tensor>& params) {
  std::string key;
  for (const Tensor& t : params) {
    const uint64_t rec[3] = {reinterpret_cast<uint64_t>(t.data_ptr()), (uint64_t)t._version(), (uint64_t)t.scalar_type()};
    key.append(reinterpret_cast<const char*>(rec), sizeof(rec));
  }
  return py::bytes(key);
}

}  // namespace

PYBIND11_MODULE(_gdn2_host, m) {
  // none of them touches Python objects: the lock is released meanwhile, as a foreign call does
  const auto unlocked = py::call_guard<py::gil_scoped_release>();
  m.def("decode", &decode, unlocked);
  m.def("prefill", &prefill, unlocked);
  m.def("prefill_short", &prefill_short, unlocked);
  m.def("layer_decode", &layer_decode, unlocked);
  m.def("layer_prefill", &layer_prefill, unlocked);
  m.def("recurrence", &recurrence, unlocked);
  m.def("feed_forward", &feed_forward, unlocked);
  m.def("gradient_launches", [] { return g_gradient_launches.load(); });
  m.def("parameter_key", &parameter_key);
}
