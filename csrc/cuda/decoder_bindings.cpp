// PyTorch bindings of the decoder-block kernels (decoder_api.h).
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <cmath>
#include <limits>
#include <string>

#include "decoder_api.h"

namespace nexar {

void count_launch(unsigned long long n);

namespace {
using OptTensor = c10::optional<at::Tensor>;

cudaStream_t stream_on(const at::Tensor& t) { return at::cuda::getCurrentCUDAStream(t.get_device()).stream(); }
void check(cudaError_t e, const char* what) {
  TORCH_CHECK(e == cudaSuccess, "nexar_b200: ", what, " failed: ", cudaGetErrorString(e));
}
const __nv_bfloat16* cbf(const at::Tensor& t) { return reinterpret_cast<const __nv_bfloat16*>(t.data_ptr()); }
__nv_bfloat16* mbf(const at::Tensor& t) { return reinterpret_cast<__nv_bfloat16*>(t.data_ptr()); }

// Numbers go into messages as text: formatting them through the message's own
// stream crashes where this module carries its own copy of the C++ library.
std::string num(long long v) { return std::to_string(v); }

int float_code(const at::Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return 0;
    case at::kHalf: return 1;
    case at::kFloat: return 2;
    default: TORCH_CHECK(false, "nexar_b200: ", name, " must be bf16, fp16 or fp32");
  }
  return -1;
}
void need_cuda(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), "nexar_b200: ", name, " must be a CUDA tensor");
}
void same_device(const at::Tensor& t, const at::Tensor& ref, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.get_device() == ref.get_device(), "nexar_b200: ", name,
              " must be on the same GPU as the input");
}

// ---------------------------------------------------------------- rotary
// x0 (and x1): [T, H, D] or [B, T, H, D]. Returns the rotated tensors, contiguous.
std::vector<at::Tensor> op_rotary(const at::Tensor& x0, const OptTensor& x1, const at::Tensor& table,
                                  const OptTensor& positions, int64_t start, int64_t heads, bool interleaved,
                                  bool inverse) {
  need_cuda(x0, "rotary input");
  const int code = float_code(x0, "rotary input");
  TORCH_CHECK(x0.dim() == 3 || x0.dim() == 4, "nexar_b200: rotary input must be [T, heads, D] or [B, T, heads, D]");
  same_device(table, x0, "rotary table");
  TORCH_CHECK(table.scalar_type() == at::kFloat && table.dim() == 2 && table.is_contiguous(),
              "nexar_b200: the rotary table must be a contiguous fp32 [rows, dim] tensor (rotary_table)");
  RotaryArgs a{};
  const bool batched = x0.dim() == 4;
  a.B = batched ? x0.size(0) : 1;
  a.T = x0.size(batched ? 1 : 0);
  a.D = (int)x0.size(-1);
  a.R = (int)table.size(1);
  a.rows = table.size(0);
  TORCH_CHECK(x0.size(-1) <= 65536 && a.R >= 2 && a.R % 2 == 0 && a.R <= a.D, "nexar_b200: the table turns ", num(a.R),
              " elements of heads of ", num(x0.size(-1)), "; it must be an even number of at most the head size");
  const uintptr_t tp = reinterpret_cast<uintptr_t>(table.data_ptr());
  TORCH_CHECK(tp % (a.R % 4 == 0 ? 16 : 8) == 0, "nexar_b200: the rotary table must be 16-byte aligned");
  a.interleaved = interleaved;
  a.sign = inverse ? -1.f : 1.f;
  a.table = table.data_ptr<float>();
  std::vector<at::Tensor> in{x0}, out;
  if (x1) in.push_back(*x1);
  for (at::Tensor& x : in) {
    same_device(x, x0, "rotary input");
    TORCH_CHECK(x.scalar_type() == x0.scalar_type() && x.dim() == x0.dim() && x.size(-1) == x0.size(-1) &&
                    x.size(-3) == x0.size(-3) && (!batched || x.size(0) == x0.size(0)),
                "nexar_b200: rotary inputs must agree in type, batch, tokens and head size");
    TORCH_CHECK(x.size(-2) <= 65536, "nexar_b200: rotary: at most 65536 heads");
    if (x.stride(-1) != 1) x = x.contiguous();
    out.push_back(at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous)));
    RotaryPart& p = a.part[a.nparts++];
    p.x = x.data_ptr();
    p.y = out.back().data_ptr();
    p.sb = batched && a.B > 1 ? x.stride(0) : 0;
    p.st = a.T > 1 ? x.stride(-3) : 0;
    p.sh = x.size(-2) > 1 ? x.stride(-2) : 0;
    p.heads = (int)x.size(-2);
    TORCH_CHECK(heads <= p.heads, "nexar_b200: rotary: ", num(heads), " heads to rotate, the input has ", num(p.heads));
    p.rotated = heads < 0 ? p.heads : (int)heads;
  }
  at::Tensor pos;
  if (positions) {
    pos = *positions;
    same_device(pos, x0, "positions");
    TORCH_CHECK(pos.scalar_type() == at::kLong || pos.scalar_type() == at::kInt,
                "nexar_b200: positions must be int64 or int32");
    TORCH_CHECK((pos.dim() == 1 && pos.size(0) == a.T) ||
                    (pos.dim() == 2 && batched && (pos.size(0) == a.B || pos.size(0) == 1) && pos.size(1) == a.T),
                "nexar_b200: positions must be [T] or [B, T]");
    a.positions = pos.data_ptr();
    a.positions_64 = pos.scalar_type() == at::kLong;
    a.pb = pos.dim() == 2 && pos.size(0) > 1 ? pos.stride(0) : 0;
    a.pt = pos.stride(-1);
  } else {
    TORCH_CHECK(start >= 0 && a.T <= a.rows && start <= a.rows - a.T, "nexar_b200: positions ", num(start),
                " to ", num(start + a.T - 1), " are past the table's ", num(a.rows), " rows");
    a.start = start;
  }
  bool any = false;
  for (const at::Tensor& x : in) any = any || x.numel() > 0;
  if (any) {
    c10::cuda::CUDAGuard g(x0.get_device());
    check(rotary(a, code == 2 ? 4 : 2, code == 1, stream_on(x0)), "rotary");
    count_launch(1);
  }
  return out;
}

void op_rotary_table(const at::Tensor& freq, const at::Tensor& table, double magnitude) {
  need_cuda(table, "table");
  same_device(freq, table, "freq");
  TORCH_CHECK(freq.scalar_type() == at::kDouble && freq.is_contiguous() && table.scalar_type() == at::kFloat &&
                  table.is_contiguous() && table.dim() == 2 && table.size(1) == 2 * freq.numel(),
              "nexar_b200: rotary_table: fp64 [R / 2] frequencies and an fp32 [rows, R] table");
  c10::cuda::CUDAGuard g(table.get_device());
  check(rotary_table(freq.data_ptr<double>(), table.data_ptr<float>(), table.size(0), (int)table.size(1), magnitude,
                     stream_on(table)),
        "rotary_table");
  count_launch(1);
}

// ---------------------------------------------------------------- dropout
struct Drop {
  uint32_t site, threshold;
  float scale;
};
Drop drop_of(double p, int64_t site) {
  TORCH_CHECK(p >= 0.0 && p <= 1.0, "nexar_b200: dropout probability must be in [0, 1], got ", std::to_string(p));
  TORCH_CHECK(site >= 0 && site <= 0xffffffffLL, "nexar_b200: dropout site must be in [0, 2^32)");
  const double t = std::nearbyint(p * 65536.0);
  return Drop{(uint32_t)site, (uint32_t)t, t < 65536.0 ? (float)(65536.0 / (65536.0 - t)) : 0.f};
}
const int64_t* drop_state(const at::Tensor& state, const at::Tensor& x) {
  same_device(state, x, "dropout state");
  TORCH_CHECK(state.scalar_type() == at::kLong && state.numel() == 2 && state.is_contiguous(),
              "nexar_b200: the dropout state must be two int64 values (seed, step)");
  return state.data_ptr<int64_t>();
}

// Returns y, and with `note` also the (seed, step) that was used.
std::tuple<at::Tensor, OptTensor> op_dropout(const at::Tensor& x_in, const at::Tensor& state, int64_t site, double p,
                                             bool note) {
  need_cuda(x_in, "dropout input");
  const int code = float_code(x_in, "dropout input");
  const Drop d = drop_of(p, site);
  const int64_t* st = drop_state(state, x_in);
  c10::cuda::CUDAGuard g(x_in.get_device());
  OptTensor snap;
  if (note) snap = at::empty({2}, state.options());
  if (d.threshold == 0) {  // nothing is dropped
    if (snap) snap->copy_(state.view({2}));
    return {x_in.clone(at::MemoryFormat::Contiguous), snap};
  }
  const at::Tensor x = x_in.contiguous();
  at::Tensor y = at::empty_like(x);
  if (x.numel() > 0) {
    check(dropout(x.data_ptr(), y.data_ptr(), x.numel(), code, st, d.site, d.threshold, d.scale,
                  snap ? snap->data_ptr<int64_t>() : nullptr, stream_on(x)),
          "dropout");
    count_launch(1);
  }
  return {y, snap};
}

void need_rows(const at::Tensor& t, const at::Tensor& x, int64_t n, const char* name) {
  same_device(t, x, name);
  TORCH_CHECK(t.scalar_type() == at::kBFloat16 && t.is_contiguous() && t.numel() == n &&
                  reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0,
              "nexar_b200: ", name, " must be a contiguous, 16-byte aligned bf16 tensor of ", num(n), " elements");
}

// Kernels read rows in 16-byte groups: a tensor at another address, or with other strides, is copied.
at::Tensor aligned_rows(const at::Tensor& t) {
  return t.is_contiguous() && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 ? t
                                                                                  : t.clone(at::MemoryFormat::Contiguous);
}
OptTensor aligned_rows(const OptTensor& t) { return t ? OptTensor(aligned_rows(*t)) : OptTensor(); }

// s = x + drop(r + rb), y = LayerNorm(s): returns s, y, mean, rstd, (seed, step).
std::vector<at::Tensor> op_dropout_ln_fwd(const at::Tensor& x_in, const at::Tensor& r_in, const OptTensor& rb_in,
                                          const at::Tensor& w_in, const at::Tensor& b_in, double eps,
                                          const at::Tensor& state, int64_t site, double p) {
  need_cuda(x_in, "x");
  c10::cuda::CUDAGuard g(x_in.get_device());
  const at::Tensor x = aligned_rows(x_in), r = aligned_rows(r_in), w = aligned_rows(w_in), b = aligned_rows(b_in);
  const OptTensor rb = aligned_rows(rb_in);
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) % 8 == 0 && x.size(-1) >= 8 && x.size(-1) <= 2048,
              "nexar_b200: residual_layer_norm with dropout needs rows of a multiple of 8, at most 2048");
  const int64_t C = x.size(-1), R = x.numel() / C;
  TORCH_CHECK(R <= std::numeric_limits<int>::max() - 65536, "nexar_b200: too many rows");
  need_rows(x, x, R * C, "x");
  need_rows(r, x, R * C, "r");
  need_rows(w, x, C, "weight");
  need_rows(b, x, C, "bias");
  if (rb) need_rows(*rb, x, C, "rbias");
  const Drop d = drop_of(p, site);
  TORCH_CHECK(d.threshold > 0, "nexar_b200: residual_layer_norm: a probability of ", std::to_string(p), " drops nothing");
  const int64_t* st = drop_state(state, x);
  at::Tensor s = at::empty_like(x), y = at::empty_like(x);
  at::Tensor mean = at::empty({R}, x.options().dtype(at::kFloat)), rstd = at::empty_like(mean);
  at::Tensor snap = at::empty({2}, state.options());
  if (R > 0) {
    check(dropout_ln_fwd(cbf(x), cbf(r), rb ? cbf(*rb) : nullptr, mbf(s), cbf(w), cbf(b), mbf(y),
                         mean.data_ptr<float>(), rstd.data_ptr<float>(), (int)R, (int)C, (float)eps, st, d.site,
                         d.threshold, d.scale, snap.data_ptr<int64_t>(), stream_on(x)),
          "dropout_ln_fwd");
    count_launch(1);
  }
  return {s, y, mean, rstd, snap};
}

// Returns dx, dr; writes dw, db (and drb).
std::vector<at::Tensor> op_dropout_ln_bwd(const at::Tensor& dy_in, const at::Tensor& s, const at::Tensor& mean,
                                          const at::Tensor& rstd, const at::Tensor& w_in, const OptTensor& dres_in,
                                          const at::Tensor& dw, const at::Tensor& db, const OptTensor& drb,
                                          const at::Tensor& snap, int64_t site, double p) {
  need_cuda(s, "s");
  c10::cuda::CUDAGuard g(s.get_device());
  const at::Tensor dy = aligned_rows(dy_in), w = aligned_rows(w_in);
  const OptTensor dres = aligned_rows(dres_in);
  const int64_t C = s.size(-1), R = s.numel() / C;
  need_rows(s, s, R * C, "s");
  need_rows(dy, s, R * C, "dy");
  if (dres) need_rows(*dres, s, R * C, "ds");
  need_rows(w, s, C, "weight");
  need_rows(dw, s, C, "dw");
  need_rows(db, s, C, "db");
  if (drb) need_rows(*drb, s, C, "drbias");
  const Drop d = drop_of(p, site);
  const int64_t* st = drop_state(snap, s);
  at::Tensor dx = at::empty_like(s), dr = at::empty_like(s);
  if (R == 0) {
    dw.zero_();
    db.zero_();
    if (drb) drb->zero_();
    return {dx, dr};
  }
  at::Tensor scratch = at::empty({(int64_t)dropout_ln_bwd_scratch_floats((int)R, (int)C)}, mean.options());
  check(dropout_ln_bwd(cbf(dy), cbf(s), mean.data_ptr<float>(), rstd.data_ptr<float>(), cbf(w),
                       dres ? cbf(*dres) : nullptr, mbf(dx), mbf(dr), mbf(dw), mbf(db), drb ? mbf(*drb) : nullptr,
                       scratch.data_ptr<float>(), (int)R, (int)C, st, d.site, d.threshold, d.scale, stream_on(s)),
        "dropout_ln_bwd");
  count_launch(2);
  return {dx, dr};
}

// ---------------------------------------------------------------- decay attention
// A [B, T, H, D] view whose rows the kernels can read in 16-byte groups, or a contiguous copy of it.
at::Tensor row_view(const at::Tensor& t) {
  bool ok = t.stride(-1) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  for (int64_t i = 0; i + 1 < t.dim(); ++i) ok = ok && (t.size(i) <= 1 || t.stride(i) % 8 == 0);
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);  // not contiguous(): it may be, at an odd address
}
void need_decay_input(const at::Tensor& t, const at::Tensor& q, const char* name) {
  same_device(t, q, name);
  TORCH_CHECK(t.scalar_type() == at::kBFloat16, "nexar_b200: decay attention: ", name, " must be bf16");
  TORCH_CHECK(t.sizes() == q.sizes(), "nexar_b200: decay attention: ", name, " must have the shape of q");
}
void need_state(const at::Tensor& st, const at::Tensor& q, int64_t B, int64_t H, int64_t D, const char* name) {
  same_device(st, q, name);
  TORCH_CHECK(st.scalar_type() == at::kFloat && st.is_contiguous() && st.dim() == 4 && st.size(0) == B &&
                  st.size(1) == H && st.size(2) == D && st.size(3) == D &&
                  reinterpret_cast<uintptr_t>(st.data_ptr()) % 16 == 0,
              "nexar_b200: decay attention: ", name, " must be a contiguous fp32 [B, H, D, D] tensor");
}
struct DecayShape {
  int64_t B, T, H, D;
};
DecayShape decay_shape(const at::Tensor& q, const at::Tensor& log_decay) {
  need_cuda(q, "q");
  TORCH_CHECK(q.scalar_type() == at::kBFloat16 && q.dim() == 4, "nexar_b200: decay attention: q must be bf16 [B, T, H, D]");
  const DecayShape s{q.size(0), q.size(1), q.size(2), q.size(3)};
  TORCH_CHECK(s.D == 64 || s.D == 128, "nexar_b200: decay attention takes heads of 64 or 128, got ", num(s.D));
  TORCH_CHECK(s.T < (1LL << 30) && s.B * s.H <= std::numeric_limits<int>::max(), "nexar_b200: decay attention: too large");
  same_device(log_decay, q, "log_decay");
  TORCH_CHECK(log_decay.scalar_type() == at::kFloat && log_decay.is_contiguous() && log_decay.numel() == s.H,
              "nexar_b200: decay attention: log_decay must be a contiguous fp32 tensor of one value per head");
  return s;
}
const int* decay_lengths(const OptTensor& lengths, const at::Tensor& q) {
  if (!lengths) return nullptr;
  same_device(*lengths, q, "lengths");
  TORCH_CHECK(lengths->scalar_type() == at::kInt && lengths->is_contiguous() && lengths->numel() == q.size(0),
              "nexar_b200: decay attention: lengths must be a contiguous int32 tensor of one value per sequence");
  return lengths->data_ptr<int>();
}
void set_in(const at::Tensor& t, const __nv_bfloat16*& p, long long& b, long long& tt, long long& h) {
  p = cbf(t);
  b = t.stride(0), tt = t.stride(1), h = t.stride(2);
}
void set_out(const at::Tensor& t, DecayRole& r) {
  r.out = mbf(t);
  r.ob = t.stride(0), r.ot = t.stride(1), r.oh = t.stride(2);
}
void set_tokens(DecayArgs& a, const DecayShape& s, const at::Tensor& log_decay, const OptTensor& lengths,
                const at::Tensor& q) {
  a.log_decay = log_decay.data_ptr<float>();
  a.lengths = decay_lengths(lengths, q);
  a.B = (int)s.B, a.T = (int)s.T, a.H = (int)s.H, a.D = (int)s.D;
}
void set_segments(DecayArgs& a, int chunks, int step) {
  a.seg_tokens = chunks * 64, a.step = step;
  a.nseg = (a.T + a.seg_tokens - 1) / a.seg_tokens;
}
// Memory for a role's own segment states.
at::Tensor own_segments(DecayArgs& a, DecayRole& r, const DecayShape& s, const at::Tensor& like) {
  at::Tensor t = at::empty({s.B * s.H * a.nseg, s.D, s.D}, like.options());
  r.segments = t.data_ptr<float>();
  r.seg_own = 1;
  return t;
}
void launch_decay(DecayArgs& a, const at::Tensor& q) {
  int launches = 0;
  check(decay_attention(a, stream_on(q), &launches), "decay_attention");
  count_launch(launches);
}

// Returns o [B, T, H, D], if asked for the final state, and where the tokens were split the states before the segments
// with the chunks of a segment.
std::tuple<at::Tensor, OptTensor, at::Tensor, int64_t> op_decay_fwd(const at::Tensor& q_in, const at::Tensor& k_in, const at::Tensor& v_in,
                                               const at::Tensor& log_decay, const OptTensor& state,
                                               const OptTensor& lengths, double scale, bool want_state) {
  const DecayShape s = decay_shape(q_in, log_decay);
  need_decay_input(k_in, q_in, "k");
  need_decay_input(v_in, q_in, "v");
  if (state) need_state(*state, q_in, s.B, s.H, s.D, "state");
  decay_lengths(lengths, q_in);
  c10::cuda::CUDAGuard g(q_in.get_device());
  const at::Tensor q = row_view(q_in), k = row_view(k_in), v = row_view(v_in);
  at::Tensor o = at::empty({s.B, s.T, s.H, s.D}, q.options());
  OptTensor fin;
  if (want_state) fin = at::empty({s.B, s.H, s.D, s.D}, log_decay.options());
  if (o.numel() == 0) {
    if (fin && fin->numel()) state ? fin->copy_(*state) : fin->zero_();
    return {o, fin, at::Tensor(), 0};
  }
  DecayArgs a{};
  a.nroles = 1;
  DecayRole& r = a.role[0];
  set_in(q, r.q, r.qb, r.qt, r.qh);
  set_in(k, r.k, r.kb, r.kt, r.kh);
  set_in(v, r.v, r.vb, r.vt, r.vh);
  set_out(o, r);
  r.intra = r.inter = (float)scale;
  r.kv = 1.f;
  r.init = state ? state->data_ptr<float>() : nullptr;
  r.final_state = fin ? fin->data_ptr<float>() : nullptr;
  set_tokens(a, s, log_decay, lengths, q);
  set_segments(a, decay_segment_chunks(a.B, a.T, a.H, a.D, a.lengths != nullptr), 1);
  at::Tensor seg;
  if (a.nseg > 1) seg = own_segments(a, r, s, log_decay);
  launch_decay(a, q);
  return {o, fin, seg, a.seg_tokens / 64};
}

// Writes dq, dk, dv ([B, T, H, D] views with unit inner stride); returns the gradient of the initial state if asked for.
OptTensor op_decay_bwd(const at::Tensor& q_in, const at::Tensor& k_in, const at::Tensor& v_in, const at::Tensor& do_in,
                       const at::Tensor& log_decay, const OptTensor& state, const OptTensor& dstate,
                       const OptTensor& lengths, double scale, const at::Tensor& dq, const at::Tensor& dk,
                       const at::Tensor& dv, bool want_dstate, const at::Tensor& fwd_segments, int64_t fwd_chunks) {
  const DecayShape s = decay_shape(q_in, log_decay);
  need_decay_input(k_in, q_in, "k");
  need_decay_input(v_in, q_in, "v");
  need_decay_input(do_in, q_in, "the output's gradient");
  if (state) need_state(*state, q_in, s.B, s.H, s.D, "state");
  if (dstate) need_state(*dstate, q_in, s.B, s.H, s.D, "the final state's gradient");
  for (const at::Tensor* t : {&dq, &dk, &dv}) {
    need_decay_input(*t, q_in, "gradient");
    TORCH_CHECK(row_view(*t).is_same(*t), "nexar_b200: decay attention: gradient rows must be 16-byte aligned");
  }
  decay_lengths(lengths, q_in);
  c10::cuda::CUDAGuard g(q_in.get_device());
  const at::Tensor q = row_view(q_in), k = row_view(k_in), v = row_view(v_in), dO = row_view(do_in);
  OptTensor ds0;
  if (want_dstate) ds0 = at::empty({s.B, s.H, s.D, s.D}, log_decay.options());
  if (q.numel() == 0) {
    if (ds0 && ds0->numel()) dstate ? ds0->copy_(*dstate) : ds0->zero_();
    return ds0;
  }
  DecayArgs a{};
  a.nroles = 3;
  const float sc = (float)scale;
  const float* ds = dstate ? dstate->data_ptr<float>() : nullptr;
  DecayRole& rv = a.role[0];  // dv: state dS [q dim, do dim], last token to first
  set_in(k, rv.q, rv.qb, rv.qt, rv.qh);
  set_in(q, rv.k, rv.kb, rv.kt, rv.kh);
  set_in(dO, rv.v, rv.vb, rv.vt, rv.vh);
  set_out(dv, rv);
  rv.reverse = 1, rv.intra = sc, rv.inter = 1.f, rv.kv = sc;
  rv.init = ds;
  rv.final_state = ds0 ? ds0->data_ptr<float>() : nullptr;
  DecayRole& rq = a.role[1];  // dq: state S transposed, first token to last
  set_in(dO, rq.q, rq.qb, rq.qt, rq.qh);
  set_in(v, rq.k, rq.kb, rq.kt, rq.kh);
  set_in(k, rq.v, rq.vb, rq.vt, rq.vh);
  set_out(dq, rq);
  rq.intra = rq.inter = sc, rq.kv = 1.f;
  rq.init = state ? state->data_ptr<float>() : nullptr;
  rq.init_transposed = 1;
  DecayRole& rk = a.role[2];  // dk: dS transposed, last token to first
  set_in(v, rk.q, rk.qb, rk.qt, rk.qh);
  set_in(dO, rk.k, rk.kb, rk.kt, rk.kh);
  set_in(q, rk.v, rk.vb, rk.vt, rk.vh);
  set_out(dk, rk);
  rk.reverse = 1, rk.intra = sc, rk.inter = 1.f, rk.kv = sc;
  rk.init = ds;
  rk.init_transposed = 1;
  set_tokens(a, s, log_decay, lengths, q);
  const int step = fwd_segments.defined() ? decay_backward_step(a.B, a.T, a.H, a.D, (int)fwd_chunks) : 0;
  at::Tensor seg;
  if (step == 0) {
    set_segments(a, (a.T + 63) / 64, 1);
  } else {
    set_segments(a, (int)fwd_chunks, step);
    seg = own_segments(a, rv, s, log_decay);
    rk.segments = rv.segments;
    rq.segments = fwd_segments.data_ptr<float>();
  }
  launch_decay(a, q);
  return ds0;
}

void no_tangents(std::initializer_list<const at::Tensor*> ts, const char* what);

// One token: q, k, v [B, H, D]; updates state [B, H, D, D] in place and returns o [B, H, D].
at::Tensor op_decay_step(const at::Tensor& q_in, const at::Tensor& k_in, const at::Tensor& v_in,
                         const at::Tensor& log_decay, const at::Tensor& state, double scale) {
  no_tangents({&q_in, &k_in, &v_in, &log_decay, &state}, "decay attention");
  need_cuda(q_in, "q");
  TORCH_CHECK(q_in.scalar_type() == at::kBFloat16 && q_in.dim() == 3,
              "nexar_b200: decay_attention_step: q must be bf16 [B, H, D]");
  const int64_t B = q_in.size(0), H = q_in.size(1), D = q_in.size(2);
  TORCH_CHECK(D == 64 || D == 128, "nexar_b200: decay attention takes heads of 64 or 128, got ", num(D));
  TORCH_CHECK(B * H <= std::numeric_limits<int>::max(), "nexar_b200: decay_attention_step: too large");
  need_decay_input(k_in, q_in, "k");
  need_decay_input(v_in, q_in, "v");
  same_device(log_decay, q_in, "log_decay");
  TORCH_CHECK(log_decay.scalar_type() == at::kFloat && log_decay.is_contiguous() && log_decay.numel() == H,
              "nexar_b200: decay attention: log_decay must be a contiguous fp32 tensor of one value per head");
  need_state(state, q_in, B, H, D, "state");
  c10::cuda::CUDAGuard g(q_in.get_device());
  const auto rows = [](const at::Tensor& t) { return t.stride(-1) == 1 ? t : t.contiguous(); };
  const at::Tensor q = rows(q_in), k = rows(k_in), v = rows(v_in);
  at::Tensor o = at::empty({B, H, D}, q.options().memory_format(at::MemoryFormat::Contiguous));
  if (o.numel() == 0) return o;
  DecayStepArgs a{};
  a.q = cbf(q), a.k = cbf(k), a.v = cbf(v), a.o = mbf(o);
  a.qb = q.stride(0), a.qh = q.stride(1), a.kb = k.stride(0), a.kh = k.stride(1), a.vb = v.stride(0), a.vh = v.stride(1);
  a.state = state.data_ptr<float>();
  a.log_decay = log_decay.data_ptr<float>();
  a.B = (int)B, a.H = (int)H, a.D = (int)D;
  a.scale = (float)scale;
  check(decay_step(a, stream_on(q)), "decay_attention_step");
  count_launch(1);
  if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();  // a graph that saved the old state notices
  return o;
}

// ---------------------------------------------------------------- autograd
// The graph nodes live here: a small call costs its kernel, not the interpreter.
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

bool any_grad(std::initializer_list<const at::Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const at::Tensor* t : ts)
    if (t && t->defined() && t->requires_grad()) return true;
  return false;
}
const at::Tensor* ptr(const OptTensor& t) { return t ? &*t : nullptr; }
// A tangent (forward-mode derivative) would be lost in the kernels, which torch reads as a derivative of zero.
void no_tangents(std::initializer_list<const at::Tensor*> ts, const char* what) {
  for (const at::Tensor* t : ts)
    TORCH_CHECK_NOT_IMPLEMENTED(!t || !t->defined() || !t->_fw_grad(0).defined(), "nexar_b200: ", what,
                                " has no forward-mode derivative");
}
at::Tensor or_none(const OptTensor& t) { return t ? *t : at::Tensor(); }
OptTensor opt(const at::Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }

// Gradients that come from kernels without a backward of their own: a second
// derivative raises instead of being silently absent.
variable_list once(variable_list grads, const char* what) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list given;
  for (at::Tensor& t : grads)
    if (t.defined()) given.push_back(t.detach().requires_grad_(true));
  auto node = std::make_shared<torch::autograd::DelayedError>(
      std::string("nexar_b200: ") + what + " has no second derivative", (int64_t)given.size());
  variable_list marked = (*node)(std::move(given));
  size_t i = 0;
  for (at::Tensor& t : grads)
    if (t.defined()) t = marked[i++];
  return grads;
}

std::vector<at::Tensor> rotate(const at::Tensor& x0, const OptTensor& x1, const at::Tensor& table,
                               const OptTensor& positions, int64_t start, int64_t heads, bool interleaved,
                               bool inverse);

// The turn is orthogonal up to the table's magnitude: its adjoint is the turn by
// the opposite angles with the same magnitude.
struct RotaryFn : public torch::autograd::Function<RotaryFn> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x0, const OptTensor& x1,
                               const at::Tensor& table, const OptTensor& positions, int64_t start, int64_t heads,
                               bool interleaved, bool inverse) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({table, or_none(positions)});
    ctx->saved_data["start"] = start;
    ctx->saved_data["heads"] = heads;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["inverse"] = inverse;
    return op_rotary(x0, x1, table, positions, start, heads, interleaved, inverse);
  }
  static variable_list backward(AutogradContext* ctx, variable_list dy) {
    const auto saved = ctx->get_saved_variables();
    variable_list out(8);
    std::vector<at::Tensor> given;
    for (const at::Tensor& d : dy)
      if (d.defined()) given.push_back(d);
    if (given.empty()) return out;
    const auto got = rotate(given[0], given.size() > 1 ? OptTensor(given[1]) : OptTensor(), saved[0], opt(saved[1]),
                            ctx->saved_data["start"].toInt(), ctx->saved_data["heads"].toInt(),
                            ctx->saved_data["interleaved"].toBool(), !ctx->saved_data["inverse"].toBool());
    size_t i = 0;
    for (size_t k = 0; k < dy.size(); ++k)
      if (dy[k].defined()) out[k] = got[i++];
    return out;
  }
};
std::vector<at::Tensor> rotate(const at::Tensor& x0, const OptTensor& x1, const at::Tensor& table,
                               const OptTensor& positions, int64_t start, int64_t heads, bool interleaved,
                               bool inverse) {
  TORCH_CHECK_VALUE(!table.requires_grad(), "nexar_b200: the rotary table takes no gradient");
  no_tangents({&x0, ptr(x1), &table}, "rotary");
  if (any_grad({&x0, ptr(x1)})) return RotaryFn::apply(x0, x1, table, positions, start, heads, interleaved, inverse);
  return op_rotary(x0, x1, table, positions, start, heads, interleaved, inverse);
}

at::Tensor drop(const at::Tensor& x, const at::Tensor& state, int64_t site, double p);

struct DropoutFn : public torch::autograd::Function<DropoutFn> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& state, int64_t site,
                            double p) {
    auto [y, used] = op_dropout(x, state, site, p, true);
    ctx->save_for_backward({*used});
    ctx->saved_data["site"] = site;
    ctx->saved_data["p"] = p;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list dy) {
    return {drop(dy[0], ctx->get_saved_variables()[0], ctx->saved_data["site"].toInt(), ctx->saved_data["p"].toDouble()),
            at::Tensor(), at::Tensor(), at::Tensor()};
  }
};
at::Tensor drop(const at::Tensor& x, const at::Tensor& state, int64_t site, double p) {
  no_tangents({&x}, "dropout");
  if (any_grad({&x})) return DropoutFn::apply(x, state, site, p);
  return std::get<0>(op_dropout(x, state, site, p, false));
}

// s = x + drop(r + rb), y = LayerNorm(s) for parameters with ordinary gradients.
struct DropoutLayerNormFn : public torch::autograd::Function<DropoutLayerNormFn> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& r, const OptTensor& rb,
                               const at::Tensor& w, const at::Tensor& b, double eps, const at::Tensor& state,
                               int64_t site, double p) {
    ctx->set_materialize_grads(false);
    auto out = op_dropout_ln_fwd(x, r, rb, w, b, eps, state, site, p);
    ctx->save_for_backward({out[0], w, out[2], out[3], out[4], or_none(rb)});
    ctx->saved_data["site"] = site;
    ctx->saved_data["p"] = p;
    ctx->saved_data["r"] = r.sizes().vec();
    return {out[0], out[1]};
  }
  static variable_list backward(AutogradContext* ctx, variable_list d) {
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &s = saved[0], &w = saved[1], &rb = saved[5];
    const at::Tensor dy = d[1].defined() ? d[1] : at::zeros_like(s);
    const OptTensor ds = opt(d[0]);
    OptTensor drb;
    if (rb.defined()) drb = at::empty_like(rb);
    at::Tensor dw = at::empty_like(w), db = at::empty_like(w);
    auto g = op_dropout_ln_bwd(dy, s, saved[2], saved[3], w, ds, dw, db, drb, saved[4],
                               ctx->saved_data["site"].toInt(), ctx->saved_data["p"].toDouble());
    return once({g[0], g[1].view(ctx->saved_data["r"].toIntVector()), or_none(drb), dw, db, at::Tensor(), at::Tensor(),
                 at::Tensor(), at::Tensor()},
                "residual_layer_norm with dropout");
  }
};
variable_list dropout_layer_norm(const at::Tensor& x, const at::Tensor& r, const OptTensor& rb, const at::Tensor& w,
                                 const at::Tensor& b, double eps, const at::Tensor& state, int64_t site, double p) {
  no_tangents({&x, &r, ptr(rb), &w, &b}, "residual_layer_norm with dropout");
  return DropoutLayerNormFn::apply(x, r, rb, w, b, eps, state, site, p);
}

// q, k, v [B, T, H, D], or (k and v absent) one packed qkv [B, T, 3, H, D].
struct DecayFn : public torch::autograd::Function<DecayFn> {
  static std::vector<at::Tensor> parts(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v) {
    return k.defined() ? std::vector<at::Tensor>{q, k, v} : q.unbind(2);
  }
  static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const OptTensor& k, const OptTensor& v,
                               const at::Tensor& log_decay, const OptTensor& state, const OptTensor& lengths,
                               double scale, bool want_state) {
    ctx->set_materialize_grads(false);
    const auto a = parts(q, or_none(k), or_none(v));
    auto [o, fin, segments, chunks] = op_decay_fwd(a[0], a[1], a[2], log_decay, state, lengths, scale, want_state);
    ctx->save_for_backward({q, or_none(k), or_none(v), log_decay, or_none(state), or_none(lengths), segments});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["chunks"] = chunks;
    if (!want_state) return {o};
    return {o, *fin};
  }
  static variable_list backward(AutogradContext* ctx, variable_list d) {
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &q = saved[0], &k = saved[1];
    const auto a = parts(q, k, saved[2]);
    variable_list out(8);
    at::Tensor packed;
    std::vector<at::Tensor> g;
    if (k.defined()) {
      for (int i = 0; i < 3; ++i) g.push_back(at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous)));
    } else {
      packed = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
      g = packed.unbind(2);
    }
    const at::Tensor dO = d[0].defined() ? d[0] : at::zeros(a[0].sizes(), q.options());
    OptTensor ds;
    if (d.size() > 1 && d[1].defined()) ds = aligned_rows(d[1]);
    const OptTensor ds0 = op_decay_bwd(a[0], a[1], a[2], dO, saved[3], opt(saved[4]), ds, opt(saved[5]),
                                       ctx->saved_data["scale"].toDouble(), g[0], g[1], g[2],
                                       saved[4].defined() && ctx->needs_input_grad(k.defined() ? 4 : 2), saved[6],
                                       ctx->saved_data["chunks"].toInt());
    out[0] = k.defined() ? g[0] : packed;
    if (k.defined()) out[1] = g[1], out[2] = g[2];
    out[4] = or_none(ds0);
    return once(out, "decay attention");
  }
};
variable_list decay(const at::Tensor& q, const OptTensor& k, const OptTensor& v, const at::Tensor& log_decay,
                    const OptTensor& state, const OptTensor& lengths, double scale, bool want_state) {
  TORCH_CHECK_VALUE(k || q.dim() == 5, "nexar_b200: decay_attention_qkv takes qkv [B, T, 3, H, D]");
  TORCH_CHECK_VALUE(k || q.size(2) == 3, "nexar_b200: decay_attention_qkv takes qkv [B, T, 3, H, D]");
  TORCH_CHECK_VALUE(!log_decay.requires_grad(),
                    "nexar_b200: decay attention: the decays are fixed; log_decay takes no gradient (detach it)");
  no_tangents({&q, ptr(k), ptr(v), &log_decay, ptr(state)}, "decay attention");
  if (any_grad({&q, ptr(k), ptr(v), ptr(state)}))
    return DecayFn::apply(q, k, v, log_decay, state, lengths, scale, want_state);
  const auto a = DecayFn::parts(q, or_none(k), or_none(v));
  const auto out = op_decay_fwd(a[0], a[1], a[2], log_decay, state, lengths, scale, want_state);
  if (!want_state) return {std::get<0>(out)};
  return {std::get<0>(out), *std::get<1>(out)};
}
}  // namespace

void register_decoder_ops(py::module& m) {
  m.def("rotary", &rotate);
  m.def("rotary_table", &op_rotary_table);
  m.def("dropout", &drop);
  m.def("dropout_ln", &dropout_layer_norm);
  m.def("dropout_ln_fwd", &op_dropout_ln_fwd);
  m.def("dropout_ln_bwd", &op_dropout_ln_bwd);
  m.def("decay_attention", &decay);
  m.def("decay_step", &op_decay_step);
  m.def("decay_error_flag", &decay_error_flag);
}

}  // namespace nexar
