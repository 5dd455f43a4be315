// Host path of the floating-point operators: the selective scan with gradients, its single-token form, token log probabilities.
#include "binding.h"

namespace qbn {
namespace {

int type_code(const Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat: return 0;
    case at::kHalf: return 1;
    case at::kBFloat16: return 2;
    default: throw std::runtime_error(std::string(name) + " must be float32, float16 or bfloat16");
  }
}
std::string said(const char* name, const char* what) { return std::string(name) + what; }

// of x's type, on x's device, with unit stride in the last dim
void like(const Tensor& t, const Tensor& x, const char* name) {
  need(t.is_cuda() && t.device() == x.device(), said(name, " must be a CUDA tensor on x's device"));
  need(t.scalar_type() == x.scalar_type(), said(name, " must have x's type"));
  need(t.size(-1) <= 1 || t.stride(-1) == 1, said(name, " must be contiguous in its last dim"));
}
Tensor param(const Tensor& t, const Tensor& x, at::IntArrayRef shape, const char* name, const char* form) {
  if (!t.defined()) return t;
  need(t.is_cuda() && t.device() == x.device() && t.scalar_type() == at::kFloat, said(name, " must be a float32 CUDA tensor on x's device"));
  need(t.sizes() == shape, said(name, form));
  return contiguous(t);
}
bool same_rows(const Tensor& t, const Tensor& x) { return !t.defined() || t.sizes() == x.sizes(); }

struct ScanIn {
  Tensor x, dt, A, B, C, D, z, bias, init, lengths;
  int64_t batch = 0, len = 0, dim = 0, n = 0, groups = 0;
  bool softplus = false;

  // (x, dt, A, B, C, D, z, dt_bias, dt_softplus, initial_state, lengths, ...); B and C as (batch, seqlen, groups, dstate)
  explicit ScanIn(const Args& a)
      : x(a.tensor(0)), dt(a.tensor(1)), A(a.tensor(2)), B(a.tensor(3)), C(a.tensor(4)), D(a.opt_tensor(5)), z(a.opt_tensor(6)), bias(a.opt_tensor(7)),
        init(a.opt_tensor(9)), lengths(a.opt_tensor(10)) {
    need(x.is_cuda(), "x must be a CUDA tensor");
    type_code(x, "x");
    need(x.dim() == 3, "x must be (batch, seqlen, dim)");
    batch = x.size(0); len = x.size(1); dim = x.size(2);
    need(dim > 0, "x must have channels");
    need(same_rows(dt, x), "dt must have the shape of x");
    need(same_rows(z, x), "z must have the shape of x");
    like(x, x, "x"); like(dt, x, "dt");
    if (z.defined()) like(z, x, "z");
    need(A.dim() == 2 && A.size(0) == dim && A.size(1) >= 1 && A.size(1) <= 64, "A must be (dim, dstate) with dstate 1 to 64");
    n = A.size(1);
    for (Tensor* t : {&B, &C}) {
      const char* name = t == &B ? "B" : "C";
      need(t->dim() == 3 || t->dim() == 4, said(name, " must be (batch, seqlen, dstate) or (batch, seqlen, groups, dstate)"));
      if (t->dim() == 3) *t = t->unsqueeze(2);
      need(t->size(0) == batch && t->size(1) == len && t->size(3) == n, said(name, " must be (batch, seqlen, dstate) or (batch, seqlen, groups, dstate)"));
      like(*t, x, name);
    }
    groups = B.size(2);
    need(C.size(2) == groups && groups > 0 && dim % groups == 0, "B and C must have the same groups, and dim be divisible by them");
    A = param(A, x, {dim, n}, "A", " must be (dim, dstate)");
    D = param(D, x, {dim}, "D", " must be (dim,)");
    bias = param(bias, x, {dim}, "dt_bias", " must be (dim,)");
    init = param(init, x, {batch, dim, n}, "initial_state", " must be (batch, dim, dstate)");
    if (lengths.defined()) {
      need(lengths.is_cuda() && lengths.device() == x.device() && lengths.scalar_type() == at::kInt && lengths.dim() == 1 && lengths.size(0) == batch,
           "lengths must be an int32 CUDA tensor (batch,) on x's device");
      lengths = contiguous(lengths);
    }
    softplus = a.flag(8);
    need(std::max(batch, dim) < (1ll << 31) && len <= (1ll << 30), "the tensors are too large");
  }
  qb_float_scan_args args() const {
    qb_float_scan_args s{};
    s.x = x.data_ptr(); s.dt = dt.data_ptr(); s.z = ptr(z); s.Bm = B.data_ptr(); s.Cm = C.data_ptr();
    s.A = f32(A); s.D = f32(D); s.dt_bias = f32(bias); s.initial_state = f32(init); s.lengths = i32(lengths);
    s.x_sb = x.stride(0); s.x_sl = x.stride(1); s.dt_sb = dt.stride(0); s.dt_sl = dt.stride(1);
    if (z.defined()) { s.z_sb = z.stride(0); s.z_sl = z.stride(1); }
    s.B_sb = B.stride(0); s.B_sl = B.stride(1); s.B_sg = B.stride(2);
    s.C_sb = C.stride(0); s.C_sl = C.stride(1); s.C_sg = C.stride(2);
    s.batch = batch; s.seqlen = len; s.dim = dim; s.dstate = n; s.groups = groups; s.dtype = type_code(x, "x"); s.dt_softplus = softplus;
    return s;
  }
};

// Whether float32 tensors of n consecutive values a row are the same rows or share none (rows that interleave some other way than
// with equal strides count as shared).
bool same_or_apart(const Tensor& a, const Tensor& b, int64_t n) {
  if (a.numel() == 0) return true;
  std::vector<int64_t> steps;
  int64_t reach_a = n, reach_b = n;
  bool alike = true;
  for (int i = 0; i < 2; ++i) {
    if (a.size(i) == 1) continue;
    alike = alike && a.stride(i) == b.stride(i);
    reach_a += (a.size(i) - 1) * a.stride(i);
    reach_b += (b.size(i) - 1) * b.stride(i);
    steps.push_back(a.stride(i));
  }
  const float *pa = static_cast<const float*>(a.data_ptr()), *pb = static_cast<const float*>(b.data_ptr());
  if (pa + reach_a <= pb || pb + reach_b <= pa || (alike && pa == pb)) return true;
  if (!alike || steps.empty()) return false;
  std::sort(steps.begin(), steps.end());
  const int64_t small = steps.front(), big = steps.back(), off = std::abs(pb - pa) % big;
  for (const int64_t r : {off, big - off})
    if (r % small < n || small - r % small < n) return false;
  return true;
}

// A workspace or the kept states; the stand-in for an empty tensor's address (which may be null) is never read.
Tensor bytes_of(const Device& dev, int64_t bytes) { return dev.empty({std::max<int64_t>(bytes, 16)}, at::kByte); }
const void* some(const Tensor& t, const Tensor& other) { return t.numel() > 0 ? t.data_ptr() : ptr(other); }

}  // namespace

// (..., want_final, want_checkpoints) -> (y, final_state | None, checkpoints | None)
PyObject* float_scan_fwd(const Args& a) {
  ScanIn in(a);
  const bool final = a.flag(11), keep = a.flag(12);
  Device dev(in.x);
  Tensor y = dev.empty({in.batch, in.len, in.dim}, in.x.scalar_type()), last, ck;
  if (final) last = dev.empty({in.batch, in.dim, in.n}, at::kFloat);
  const int64_t ck_bytes = qb_float_scan_checkpoint_bytes(in.batch, in.len, in.dim, in.groups, in.n);
  if (keep) ck = bytes_of(dev, ck_bytes);
  if (in.batch > 0) {
    const int64_t ws_bytes = qb_float_scan_workspace_bytes(in.batch, in.len, in.dim, in.groups, in.n, 0);
    Tensor ws;
    if (ws_bytes > 0) ws = bytes_of(dev, ws_bytes);
    qb_float_scan_args s = in.args();
    s.x = some(in.x, in.A); s.dt = some(in.dt, in.A); s.Bm = some(in.B, in.A); s.Cm = some(in.C, in.A);
    s.y = ptr(y); s.final_state = f32(last); s.checkpoints = static_cast<float*>(ptr(ck)); s.workspace = ptr(ws); s.workspace_bytes = ws_bytes;
    QBN_CALL(qb_float_scan_fwd, s, dev.stream);
  }
  return wrap_tuple({y, last, ck});
}

// (..., checkpoints, dy, d_final | None) -> gradients of x, dt, A, B, C, D, z, dt_bias, initial_state, None for what was not given
PyObject* float_scan_bwd(const Args& a) {
  ScanIn in(a);
  const Tensor ck = a.tensor(11);
  Tensor dy = a.tensor(12), dlast = a.opt_tensor(13);
  need(dy.sizes() == in.x.sizes() && dy.scalar_type() == in.x.scalar_type() && dy.device() == in.x.device(), "the gradient of y must be like y");
  if (dy.stride(-1) != 1) dy = contiguous(dy);
  dlast = param(dlast, in.x, {in.batch, in.dim, in.n}, "the gradient of the final state", " must be (batch, dim, dstate)");
  Device dev(in.x);
  const auto type = in.x.scalar_type();
  Tensor dx = dev.empty({in.batch, in.len, in.dim}, type), ddt = dev.empty({in.batch, in.len, in.dim}, type), dA = dev.empty({in.dim, in.n}, at::kFloat);
  Tensor dB = dev.empty(a.tensor(3).sizes(), type), dC = dev.empty(a.tensor(4).sizes(), type);     // with or without groups, as they came
  Tensor dD, dz, dbias, dinit;
  if (in.D.defined()) dD = dev.empty({in.dim}, at::kFloat);
  if (in.z.defined()) dz = dev.empty({in.batch, in.len, in.dim}, type);
  if (in.bias.defined()) dbias = dev.empty({in.dim}, at::kFloat);
  if (in.init.defined()) dinit = dev.empty({in.batch, in.dim, in.n}, at::kFloat);
  const int64_t ws_bytes = qb_float_scan_workspace_bytes(in.batch, in.len, in.dim, in.groups, in.n, 1);
  const Tensor ws = bytes_of(dev, ws_bytes);
  qb_float_scan_args s = in.args();
  s.x = some(in.x, in.A); s.dt = some(in.dt, in.A); s.Bm = some(in.B, in.A); s.Cm = some(in.C, in.A);
  s.dy = dy.numel() > 0 ? dy.data_ptr() : nullptr; s.dy_sb = dy.stride(0); s.dy_sl = dy.stride(1); s.d_final = f32(dlast);
  s.checkpoints = static_cast<float*>(ptr(ck));
  s.d_x = ptr(dx); s.d_dt = ptr(ddt); s.d_z = ptr(dz); s.d_B = ptr(dB); s.d_C = ptr(dC);
  s.d_A = f32(dA); s.d_D = f32(dD); s.d_bias = f32(dbias); s.d_initial = f32(dinit);
  s.workspace = ptr(ws); s.workspace_bytes = ws_bytes;
  QBN_CALL(qb_float_scan_bwd, s, dev.stream);
  return wrap_tuple({dx, ddt, dA, dB, dC, dD, dz, dbias, dinit});
}

// (state, x, dt, A, B, C, D, z, dt_bias, dt_softplus, state_out | None) -> y
PyObject* float_scan_update(const Args& a) {
  const Tensor st = a.tensor(0), x = a.tensor(1), dt = a.tensor(2), z = a.opt_tensor(7);
  Tensor A = a.tensor(3), B = a.tensor(4), C = a.tensor(5), D = a.opt_tensor(6), bias = a.opt_tensor(8);
  const Tensor so = a.is_none(10) ? st : a.tensor(10);
  need(x.is_cuda(), "x must be a CUDA tensor");
  const int code = type_code(x, "x");
  need(x.dim() == 2, "x must be (batch, dim)");
  const int64_t batch = x.size(0), dim = x.size(1);
  need(dim > 0, "x must have channels");
  need(same_rows(dt, x), "dt must have the shape of x");
  need(same_rows(z, x), "z must have the shape of x");
  like(x, x, "x"); like(dt, x, "dt");
  if (z.defined()) like(z, x, "z");
  need(A.dim() == 2 && A.size(0) == dim && A.size(1) >= 1 && A.size(1) <= 64, "A must be (dim, dstate) with dstate 1 to 64");
  const int64_t n = A.size(1);
  for (const Tensor* t : {&st, &so}) {
    const char* name = t == &st ? "state" : "state_out";
    need(t->is_cuda() && t->device() == x.device() && t->scalar_type() == at::kFloat, said(name, " must be a float32 CUDA tensor on x's device"));
    need(t->dim() == 3 && t->size(0) == batch && t->size(1) == dim && t->size(2) == n, said(name, " must be (batch, dim, dstate)"));
    need(n == 1 || t->stride(2) == 1, said(name, " must be contiguous in its last dim"));
  }
  // one state per (sequence, channel): rows written twice would race
  need(batch * dim == 0 || ((batch == 1 || so.stride(0) >= n) && (dim == 1 || so.stride(1) >= n) &&
                            (batch == 1 || dim == 1 || so.stride(0) >= (dim - 1) * so.stride(1) + n || so.stride(1) >= (batch - 1) * so.stride(0) + n)),
       "the rows of state_out must not overlap");
  need(same_or_apart(st, so, n), "state_out must be state itself or share no memory with it");
  for (Tensor* t : {&B, &C}) {
    const char* name = t == &B ? "B" : "C";
    need(t->dim() == 2 || t->dim() == 3, said(name, " must be (batch, dstate) or (batch, groups, dstate)"));
    if (t->dim() == 2) *t = t->unsqueeze(1);
    need(t->size(0) == batch && t->size(2) == n, said(name, " must be (batch, dstate) or (batch, groups, dstate)"));
    like(*t, x, name);
  }
  const int64_t groups = B.size(1);
  need(C.size(1) == groups && groups > 0 && dim % groups == 0, "B and C must have the same groups, and dim be divisible by them");
  A = param(A, x, {dim, n}, "A", " must be (dim, dstate)");
  D = param(D, x, {dim}, "D", " must be (dim,)");
  bias = param(bias, x, {dim}, "dt_bias", " must be (dim,)");
  Device dev(x);
  Tensor y = dev.empty({batch, dim}, x.scalar_type());
  if (batch > 0) {
    qb_float_update_args s{};
    s.state = f32(st); s.state_out = f32(so); s.x = x.data_ptr(); s.dt = dt.data_ptr(); s.z = ptr(z); s.Bm = B.data_ptr(); s.Cm = C.data_ptr();
    s.A = f32(A); s.D = f32(D); s.dt_bias = f32(bias); s.y = y.data_ptr();
    s.state_sb = st.stride(0); s.state_sd = st.stride(1); s.state_out_sb = so.stride(0); s.state_out_sd = so.stride(1);
    s.x_sb = x.stride(0); s.dt_sb = dt.stride(0); s.z_sb = z.defined() ? z.stride(0) : 0;
    s.B_sb = B.stride(0); s.B_sg = B.stride(1); s.C_sb = C.stride(0); s.C_sg = C.stride(1);
    s.batch = batch; s.dim = dim; s.dstate = n; s.groups = groups; s.dtype = code; s.dt_softplus = a.flag(9);
    QBN_CALL(qb_float_scan_update, s, dev.stream);
  }
  return wrap(y);
}

namespace {

struct LogitsIn {
  Tensor logits, targets;
  int64_t rows = 0, inner = 1, outer_stride = 0, row_stride = 0, vocab = 0;
  int code;
  LogitsIn(const Tensor& l, const Tensor& t) : logits(l), targets(t) {
    need(l.is_cuda(), "logits must be a CUDA tensor");
    code = type_code(l, "logits");
    need(l.dim() == 2 || l.dim() == 3, "logits must be (rows, vocab) or (batch, seqlen, vocab)");
    vocab = l.size(-1);
    need(vocab > 0 && vocab <= (1ll << 30), "logits must have a vocabulary of 1 to 2^30 columns");
    need(vocab == 1 || l.stride(-1) == 1, "logits must be contiguous in their last dim");
    need(t.is_cuda() && t.device() == l.device() && t.scalar_type() == at::kLong, "targets must be an int64 CUDA tensor on the logits' device");
    need(t.sizes() == l.sizes().slice(0, l.dim() - 1), "targets must have the shape of the logits without the vocabulary");
    targets = contiguous(t);
    inner = l.size(-2);
    rows = l.dim() == 3 ? l.size(0) * inner : inner;
    row_stride = l.stride(-2);
    outer_stride = l.dim() == 3 ? l.stride(0) : 0;
  }
  qb_logprobs_args args(int64_t ignore) const {
    qb_logprobs_args s{};
    s.logits = logits.data_ptr(); s.targets = static_cast<const int64_t*>(targets.data_ptr());
    s.outer_stride = outer_stride; s.row_stride = row_stride; s.ignore_index = ignore; s.rows = rows; s.inner_rows = inner; s.vocab = vocab; s.dtype = code;
    return s;
  }
};

}  // namespace

// (logits, targets, top_k, want_entropy, ignore_index) -> (logprobs, entropy | None, lse, top_logprobs | None, top_ids | None)
PyObject* logprobs_fwd(const Args& a) {
  const LogitsIn in(a.tensor(0), a.tensor(1));
  const long top = a.integer(2), ignore = a.integer(4);
  need(top >= 0 && top <= QB_LOGPROBS_MAX_TOP && top <= in.vocab, "top_k must be 0 to 32 and at most the vocabulary");
  Device dev(in.logits);
  const at::IntArrayRef shape = in.targets.sizes();
  Tensor lp = dev.empty(shape, at::kFloat), lse = dev.empty(shape, at::kFloat), ent, tl, ti;
  if (a.flag(3)) ent = dev.empty(shape, at::kFloat);
  if (top > 0) {
    std::vector<int64_t> wide(shape.begin(), shape.end());
    wide.push_back(top);
    tl = dev.empty(wide, at::kFloat);
    ti = dev.empty(wide, at::kLong);
  }
  if (in.rows > 0) {
    qb_logprobs_args s = in.args(ignore);
    s.logprobs = f32(lp); s.entropy = f32(ent); s.lse = f32(lse); s.top_logprobs = f32(tl); s.top_ids = static_cast<int64_t*>(ptr(ti)); s.top_k = top;
    QBN_CALL(qb_logprobs_fwd, s, dev.stream);
  }
  return wrap_tuple({lp, ent, lse, tl, ti});
}

// (logits, targets, lse, entropy | None, ignore_index, d_logprobs | None, d_entropy | None) -> d_logits
PyObject* logprobs_bwd(const Args& a) {
  const LogitsIn in(a.tensor(0), a.tensor(1));
  const Tensor lse = a.tensor(2), ent = a.opt_tensor(3);
  Tensor g = a.opt_tensor(5), h = a.opt_tensor(6);
  for (Tensor* t : {&g, &h}) {
    if (!t->defined()) continue;
    need(t->is_cuda() && t->device() == in.logits.device() && t->scalar_type() == at::kFloat && t->sizes() == in.targets.sizes(),
         "the gradients of log probabilities and entropy must be float32, one per row");
    *t = contiguous(*t);
  }
  Device dev(in.logits);
  // Rows of the gradient begin at the same offset from a 16-byte boundary as those of the logits, so that both move in 16-byte pieces.
  const int64_t size = in.logits.element_size(), per = 16 / size;
  const auto up = [&](int64_t v, int64_t as) { return v + ((as - v) % per + per) % per; };       // the next value congruent to `as`
  const int64_t shift = (reinterpret_cast<uintptr_t>(in.logits.data_ptr()) & 15) / size;
  const int64_t row = up(in.vocab, in.row_stride), outer = up(in.inner * row, in.outer_stride), outers = in.logits.dim() == 3 ? in.logits.size(0) : 1;
  const Tensor all = dev.empty({shift + outers * outer}, in.logits.scalar_type());
  const Tensor d = in.logits.dim() == 3 ? all.as_strided(in.logits.sizes(), {outer, row, 1}, shift) : all.as_strided(in.logits.sizes(), {row, 1}, shift);
  if (in.rows > 0) {
    qb_logprobs_args s = in.args(a.integer(4));
    s.lse = f32(lse); s.entropy = f32(ent); s.d_logprobs = f32(g); s.d_entropy = f32(h); s.d_logits = d.data_ptr();
    s.d_outer_stride = outer; s.d_row_stride = row;
    QBN_CALL(qb_logprobs_bwd, s, dev.stream);
  }
  return wrap(d);
}

}  // namespace qbn
