// Registrations of the decoder's operators for the native imperative path:
// RMSNorm, _contrib_rms_norm_int8, _contrib_encdec_attention and
// _contrib_sample_tokens.  GPU: the launchers of rmsnorm.hip,
// encdec_attention.hip and sample.hip with scratch from the engine's arena;
// CPU: plain loops in 64 bits (oracles, fp32 data).
#include <algorithm>
#include <cmath>
#include <limits>

#include "ew_common.h"
#include "ops_api.h"

namespace mxcore {
namespace {

using V = const std::vector<TBlob>&;

LaunchCtx LC(const OpCtx& o) {
  LaunchCtx lc;
  lc.stream = o.rc.stream;
  lc.dev = o.rc.ctx.dev_id;
  lc.workspace = o.workspace;
  return lc;
}

Arr Scratch(const OpCtx& o, int64_t n, int dtype) {
  if (n == 0) return Arr();
  return Arr(o.workspace(n * dtype_size(dtype)), {n}, dtype);
}

void CheckCpu(const TBlob& b, const char* name) {
  MX_CHECK(b.dtype == kFloat32, name << ": CPU path is fp32 (oracle)");
}

bool IsFloat(int dt) {
  return dt == kFloat32 || dt == kFloat16 || dt == kBFloat16;
}

std::vector<NDArray> RunOp(const char* name, const NodeAttrs& attrs,
                           const std::vector<NDArray>& ins) {
  OpEntry* e = OpRegistry::Get()->Find(name);
  MX_CHECK(e, "op not registered: " << name);
  return Imperative::Run(e, attrs, ins);
}

// ---------------------------------------------------------------------------
// RMSNorm: (data, gamma[, residual])
// ---------------------------------------------------------------------------
// outputs: y or int8, the sum (a placeholder without a residual), 1 / rms or
// the scale of each row
FInferShape RmsInfer(bool int8) {
  return [int8](const NodeAttrs&, const std::vector<TShape>& is,
                const std::vector<int>& it, std::vector<TShape>* os,
                std::vector<int>* ot) {
    MX_CHECK(is.size() == 2 || is.size() == 3,
             "RMSNorm: data, gamma and perhaps a residual");
    MX_CHECK(is[0].size() >= 1 && is[0].back() >= 1 && IsFloat(it[0]),
             "RMSNorm: floating data with a last axis to norm");
    MX_CHECK(is[1] == TShape{is[0].back()} && it[1] == kFloat32,
             "RMSNorm: gamma must hold one float32 for each column");
    MX_CHECK(is.size() == 2 || (is[2] == is[0] && it[2] == it[0]),
             "RMSNorm: the residual must be like the data");
    TShape stat = is[0];
    stat.back() = 1;
    *os = {is[0], is.size() == 3 ? is[0] : TShape{1}, stat};
    *ot = {int8 ? (int)kInt8 : it[0], it[0], kFloat32};
  };
}

void RmsGpu(const NodeAttrs& a, const OpCtx& o, V in, V out) {
  const bool res = in.size() == 3, int8 = out[0].dtype == kInt8;
  rms_norm_fwd_raw(LC(o), in[0], in[1], res ? Arr(in[2]) : Arr(),
                   a.GetFloat("eps", 1e-6), out[0],
                   int8 ? Arr(out[2]) : Arr(), res ? Arr(out[1]) : Arr(),
                   int8 ? Arr() : Arr(out[2]));
}

void RmsCpu(const NodeAttrs& a, const OpCtx&, V in, V out) {
  CheckCpu(in[0], "RMSNorm");
  const double eps = a.GetFloat("eps", 1e-6);
  const long C = in[0].shape.back(), rows = in[0].size() / C;
  const bool res = in.size() == 3, int8 = out[0].dtype == kInt8;
  const float* g = (const float*)in[1].dptr;
  std::vector<float> h(C);
  for (long r = 0; r < rows; ++r) {
    double sq = 0;
    for (long c = 0; c < C; ++c) {
      h[c] = ((const float*)in[0].dptr)[r * C + c];
      if (res) {
        h[c] += ((const float*)in[2].dptr)[r * C + c];
        ((float*)out[1].dptr)[r * C + c] = h[c];
      }
      sq += (double)h[c] * h[c];
    }
    const float inv = (float)(1.0 / std::sqrt(sq / C + eps));
    float* stat = (float*)out[2].dptr + r;
    if (!int8) {
      *stat = inv;
      for (long c = 0; c < C; ++c)
        ((float*)out[0].dptr)[r * C + c] = h[c] * inv * g[c];
      continue;
    }
    float top = 0.f;
    bool bad = false;
    for (long c = 0; c < C; ++c) {
      const float y = std::fabs(h[c] * inv * g[c]);
      bad |= !std::isfinite(y);
      top = std::max(top, y);
    }
    float f = 127.0f * (1.0f / top);
    *stat = top * (1.0f / 127.0f);
    if (!(top > 0.f) || std::isinf(f)) {
      *stat = 1.f;
      f = 0.f;
    }
    if (bad) *stat = std::numeric_limits<float>::quiet_NaN();
    for (long c = 0; c < C; ++c) {
      const float q = bad ? 0.f : std::nearbyint(h[c] * inv * g[c] * f);
      ((signed char*)out[0].dptr)[r * C + c] =
          (signed char)std::min(127.f, std::max(-127.f, q));
    }
  }
}

// inputs: [dy,] [dsum,] h, gamma, 1 / rms
std::vector<NDArray> RmsBwd(const TapeNode& n,
                            const std::vector<NDArray>& og) {
  const bool res = n.inputs.size() == 3;
  std::vector<NDArray> r(n.inputs.size());
  const NDArray& dy = og[0];
  NDArray dsum;
  if (res) dsum = og[1];
  if (dy.is_none()) {  // only the sum was used
    r[0] = dsum;
    r[2] = dsum;
    return r;
  }
  std::vector<NDArray> ins = {dy};
  if (!dsum.is_none()) ins.push_back(dsum);
  ins.push_back(res ? n.outputs[1] : n.inputs[0]);
  ins.push_back(n.inputs[1]);
  ins.push_back(n.outputs[2]);
  auto outs = RunOp("_rms_norm_bwd", {}, ins);
  r[0] = outs[0];
  r[1] = outs[1];
  if (res) r[2] = outs[0];
  return r;
}

// ---------------------------------------------------------------------------
// attention: (queries, keys_values[, values][, valid_length][, mask])
// ---------------------------------------------------------------------------
struct EncDec {
  Arr q, kv, values, len, mask;
  int heads, kv_heads;
  bool apart, tnc;  // apart: values, also of no keys and without memory
  int64_t B, sq, sk, D;
};

EncDec ReadEncDec(const NodeAttrs& a, const Arr* in, size_t n_in) {
  EncDec e;
  size_t i = 0;
  auto next = [&]() -> Arr {
    MX_CHECK(i < n_in, "encdec_attention: too few inputs");
    return in[i++];
  };
  e.q = next();
  e.kv = next();
  e.apart = a.GetBool("has_values", false);
  if (e.apart) e.values = next();
  if (a.GetBool("has_length", false)) e.len = next();
  if (a.GetBool("has_mask", false)) e.mask = next();
  e.heads = (int)a.GetInt("heads", 1);
  e.kv_heads = (int)a.GetInt("kv_heads", e.heads);
  e.tnc = a.GetBool("tnc", false);
  MX_CHECK(e.q.dim() == 3 && e.kv.dim() == 3 && e.heads > 0 &&
               e.kv_heads > 0 && e.heads % e.kv_heads == 0 &&
               e.q.size(2) % e.heads == 0 && e.q.size(2) > 0,
           "encdec_attention: bad heads");
  e.B = e.q.size(e.tnc ? 1 : 0);
  e.sq = e.q.size(e.tnc ? 0 : 1);
  e.sk = e.kv.size(e.tnc ? 0 : 1);
  e.D = e.q.size(2) / e.heads;
  return e;
}

std::vector<Arr> Arrs(V in, size_t from = 0) {
  return std::vector<Arr>(in.begin() + from, in.end());
}

void EncDecInfer(const NodeAttrs& a, const std::vector<TShape>& is,
                 const std::vector<int>& it, std::vector<TShape>* os,
                 std::vector<int>* ot) {
  std::vector<Arr> in;
  for (size_t i = 0; i < is.size(); ++i) in.emplace_back(nullptr, is[i], it[i]);
  const EncDec e = ReadEncDec(a, in.data(), in.size());
  const bool apart = e.apart;
  MX_CHECK(IsFloat(e.q.dtype) && e.kv.dtype == e.q.dtype &&
               e.kv.size(2) == e.kv_heads * e.D * (apart ? 1 : 2) &&
               e.kv.size(e.tnc ? 1 : 0) == e.B,
           "encdec_attention: the keys do not fit the queries and heads");
  MX_CHECK(!apart || (e.values.shape == e.kv.shape &&
                      e.values.dtype == e.kv.dtype),
           "encdec_attention: the values must be like the keys");
  MX_CHECK(!a.GetBool("has_length", false) ||
               (e.len.shape == TShape{e.B} &&
                (e.len.dtype == kInt32 || e.len.dtype == kInt64)),
           "encdec_attention: valid_length must hold one int32 or int64 for "
           "each sequence");
  MX_CHECK(!a.GetBool("has_mask", false) ||
               (e.mask.shape == TShape{e.B, e.sk} &&
                (e.mask.dtype == kUint8 || e.mask.dtype == kBool)),
           "encdec_attention: the mask must hold one byte for each key");
  *os = {e.q.shape, TShape{e.B, e.heads, e.sq}};
  *ot = {e.q.dtype, kFloat32};
}

// the CPU's loops over [B, S, heads, D] in either layout
struct Walk {
  const EncDec& e;
  int64_t row(const Arr& x, int64_t b, int64_t s) const {
    return (e.tnc ? s * e.B + b : b * x.size(1) + s) * x.size(2);
  }
  int64_t q(int64_t b, int64_t h, int64_t s) const {
    return row(e.q, b, s) + h * e.D;
  }
  int64_t k(int64_t b, int64_t h, int64_t s) const {
    return row(e.kv, b, s) + h * e.D * (e.apart ? 1 : 2);
  }
  bool keep(int64_t b, int64_t s) const {
    if (e.len.defined() &&
        s >= (e.len.dtype == kInt64 ? e.len.data<int64_t>()[b]
                                    : e.len.data<int>()[b]))
      return false;
    return !e.mask.defined() || e.mask.data<uint8_t>()[b * e.sk + s];
  }
  // weights of one row; false if it has no key
  bool weights(int64_t b, int64_t h, int64_t s, std::vector<double>* p) const {
    const float* qr = e.q.data<float>() + q(b, h, s);
    double top = -INFINITY, sum = 0;
    for (int64_t j = 0; j < e.sk; ++j) {
      (*p)[j] = -INFINITY;
      if (!keep(b, j)) continue;
      const float* kr =
          e.kv.data<float>() + k(b, h / (e.heads / e.kv_heads), j);
      double v = 0;
      for (int64_t d = 0; d < e.D; ++d) v += (double)qr[d] * kr[d];
      (*p)[j] = v / std::sqrt((double)e.D);
      top = std::max(top, (*p)[j]);
    }
    if (top == -INFINITY) return false;
    for (auto& v : *p) sum += v = std::exp(v - top);
    for (auto& v : *p) v /= sum;
    return true;
  }
};

void EncDecCpu(const NodeAttrs& a, const OpCtx&, V in, V out) {
  CheckCpu(in[0], "encdec_attention");
  const auto ins = Arrs(in);
  const EncDec e = ReadEncDec(a, ins.data(), ins.size());
  const Walk w{e};
  const float* vals = e.apart ? e.values.data<float>()
                              : e.kv.data<float>() + e.D;
  std::vector<double> p(e.sk);
  for (int64_t b = 0; b < e.B; ++b)
    for (int64_t h = 0; h < e.heads; ++h)
      for (int64_t s = 0; s < e.sq; ++s) {
        float* o = (float*)out[0].dptr + w.q(b, h, s);
        std::fill(o, o + e.D, 0.f);
        if (!w.weights(b, h, s, &p)) continue;
        for (int64_t d = 0; d < e.D; ++d) {
          double v = 0;
          for (int64_t j = 0; j < e.sk; ++j)
            if (p[j] > 0)
              v += p[j] * vals[w.k(b, h / (e.heads / e.kv_heads), j) + d];
          o[d] = (float)v;
        }
      }
}

// inputs: dout, out, lse, then the forward's; outputs like the first of those
void EncDecBwdCpu(const NodeAttrs& a, const OpCtx&, V in, V out) {
  CheckCpu(in[0], "encdec_attention");
  const auto ins = Arrs(in, 3);
  const EncDec e = ReadEncDec(a, ins.data(), ins.size());
  const Walk w{e};
  const bool apart = e.apart;
  const float* vals = apart ? e.values.data<float>()
                            : e.kv.data<float>() + e.D;
  const double c = 1 / std::sqrt((double)e.D);
  std::vector<double> p(e.sk), dk(e.kv.numel()),
      dv(apart ? e.kv.numel() : 0);
  double* dvp = apart ? dv.data() : dk.data() + e.D;
  for (int64_t b = 0; b < e.B; ++b)
    for (int64_t h = 0; h < e.heads; ++h)
      for (int64_t s = 0; s < e.sq; ++s) {
        const int64_t qa = w.q(b, h, s);
        const float* g = (const float*)in[0].dptr + qa;
        const float* q = e.q.data<float>() + qa;
        std::vector<double> dq(e.D), dp(e.sk);
        double delta = 0;
        if (w.weights(b, h, s, &p)) {
          for (int64_t j = 0; j < e.sk; ++j) {
            if (p[j] == 0) continue;
            const int64_t ka = w.k(b, h / (e.heads / e.kv_heads), j);
            for (int64_t d = 0; d < e.D; ++d) dp[j] += g[d] * (double)vals[ka + d];
            delta += p[j] * dp[j];
          }
          for (int64_t j = 0; j < e.sk; ++j) {
            if (p[j] == 0) continue;
            const int64_t ka = w.k(b, h / (e.heads / e.kv_heads), j);
            const double ds = p[j] * (dp[j] - delta) * c;
            for (int64_t d = 0; d < e.D; ++d) {
              dq[d] += ds * e.kv.data<float>()[ka + d];
              dk[ka + d] += ds * q[d];
              dvp[ka + d] += p[j] * g[d];
            }
          }
        }
        for (int64_t d = 0; d < e.D; ++d)
          ((float*)out[0].dptr)[qa + d] = (float)dq[d];
      }
  for (size_t i = 0; i < dk.size(); ++i) ((float*)out[1].dptr)[i] = (float)dk[i];
  for (size_t i = 0; i < dv.size(); ++i) ((float*)out[2].dptr)[i] = (float)dv[i];
}

// ---------------------------------------------------------------------------
// sampling: (logits, uniform[, temperature][, top_k][, top_p][, min_p])
// ---------------------------------------------------------------------------
struct SampleIn {
  Arr x, u, t, k, p, m;
};

SampleIn ReadSample(const NodeAttrs& a, const std::vector<Arr>& in) {
  SampleIn s;
  size_t i = 2;
  s.x = in.at(0);
  s.u = in.at(1);
  if (a.GetBool("has_temperature", false)) s.t = in.at(i++);
  if (a.GetBool("has_top_k", false)) s.k = in.at(i++);
  if (a.GetBool("has_top_p", false)) s.p = in.at(i++);
  if (a.GetBool("has_min_p", false)) s.m = in.at(i++);
  return s;
}

void SampleCpu(const NodeAttrs& a, const OpCtx&, V in, V out) {
  CheckCpu(in[0], "sample_tokens");
  const SampleIn s = ReadSample(a, Arrs(in));
  const int64_t N = s.x.size(0), V_ = s.x.size(1);
  for (int64_t n = 0; n < N; ++n) {
    const float* row = s.x.data<float>() + n * V_;
    std::vector<std::pair<float, int>> o(V_);
    for (int64_t i = 0; i < V_; ++i)
      o[i] = {row[i] == row[i] ? row[i] : -INFINITY, (int)i};
    std::stable_sort(o.begin(), o.end(),
                     [](auto& l, auto& r) { return l.first > r.first; });
    int* token = (int*)out[0].dptr + n;
    float* logp = (float*)out[1].dptr + n;
    const float top = o[0].first;
    if (top == -INFINITY) {
      *token = -1;
      *logp = std::numeric_limits<float>::quiet_NaN();
      continue;
    }
    const double t = s.t.defined()
                         ? std::min<double>(s.t.data<float>()[n], 1e30)
                         : a.GetFloat("temperature", 1);
    int64_t k = !s.k.defined()        ? a.GetInt("top_k", 0)
                : s.k.dtype == kInt64 ? s.k.data<int64_t>()[n]
                                      : s.k.data<int>()[n];
    const double p = s.p.defined() ? s.p.data<float>()[n]
                                   : a.GetFloat("top_p", 1);
    const double m = s.m.defined() ? std::min<double>(s.m.data<float>()[n], 1)
                                   : a.GetFloat("min_p", 0);
    if (!(t > 0)) k = 1;
    int64_t keep = k > 0 && k < V_ ? k : V_;
    std::vector<double> w(keep);
    double sum = 0, run = 0;
    for (int64_t i = 0; i < keep; ++i) {
      w[i] = o[i].first == top ? 1.0 : std::exp(((double)o[i].first - top) / t);
      sum += w[i];
    }
    if (p < 1)
      for (int64_t i = 0; i < keep; ++i) {
        run += w[i];
        if (run >= p * sum) keep = i + 1;
      }
    if (m > 0)
      while (keep > 1 && w[keep - 1] < m) --keep;
    sum = 0;
    for (int64_t i = 0; i < keep; ++i) sum += w[i];
    const float raw = s.u.data<float>()[n], most = 1.f - 0x1p-24f;
    const double u = std::isnan(raw) ? most : std::max(std::min(raw, most), 0.f);
    int64_t at = 0;
    for (run = w[0]; at + 1 < keep && run <= u * sum; run += w[at]) ++at;
    *token = o[at].second;
    *logp = (float)std::log(w[at] / sum);
  }
}

bool _registered = [] {
  for (bool int8 : {false, true}) {
    OpEntry& e = OpRegistry::Get()->Register(
        int8 ? "_contrib_rms_norm_int8" : "RMSNorm");
    e.n_out = 3;
    e.infer = RmsInfer(int8);
    e.fcompute_gpu = RmsGpu;
    e.fcompute_cpu = RmsCpu;
    if (!int8) e.fbackward = RmsBwd;
  }
  {
    OpEntry& e = OpRegistry::Get()->Register("_rms_norm_bwd");
    e.n_out = 2;
    e.infer = [](const NodeAttrs&, const std::vector<TShape>& is,
                 const std::vector<int>& it, std::vector<TShape>* os,
                 std::vector<int>* ot) {
      *os = {is[0], TShape{is[0].back()}};
      *ot = {it[0], kFloat32};
    };
    e.fcompute_gpu = [](const NodeAttrs&, const OpCtx& o, V in, V out) {
      const size_t n = in.size();
      const int64_t C = in[0].shape.back(), rows = in[0].size() / C;
      rms_norm_bwd_raw(LC(o), in[0], n == 5 ? Arr(in[1]) : Arr(), in[n - 3],
                       in[n - 2], in[n - 1], out[0], out[1],
                       Scratch(o, rms_norm_bwd_blocks(rows) * C, kFloat32));
    };
    e.fcompute_cpu = [](const NodeAttrs&, const OpCtx&, V in, V out) {
      CheckCpu(in[0], "RMSNorm");
      const size_t n = in.size();
      const long C = in[0].shape.back(), rows = in[0].size() / C;
      const float* dy = (const float*)in[0].dptr;
      const float* dsum = n == 5 ? (const float*)in[1].dptr : nullptr;
      const float* h = (const float*)in[n - 3].dptr;
      const float* g = (const float*)in[n - 2].dptr;
      const float* inv = (const float*)in[n - 1].dptr;
      std::vector<double> dg(C);
      for (long r = 0; r < rows; ++r) {
        double m = 0;
        for (long c = 0; c < C; ++c) {
          const double nn = (double)h[r * C + c] * inv[r];
          m += (double)dy[r * C + c] * g[c] * nn;
          dg[c] += dy[r * C + c] * nn;
        }
        m /= C;
        for (long c = 0; c < C; ++c)
          ((float*)out[0].dptr)[r * C + c] = (float)(
              inv[r] * ((double)dy[r * C + c] * g[c] -
                        (double)h[r * C + c] * inv[r] * m) +
              (dsum ? dsum[r * C + c] : 0.0));
      }
      for (long c = 0; c < C; ++c) ((float*)out[1].dptr)[c] = (float)dg[c];
    };
  }
  {
    OpEntry& e = OpRegistry::Get()->Register("_contrib_encdec_attention");
    e.n_out = 2;
    e.infer = EncDecInfer;
    e.fcompute_gpu = [](const NodeAttrs& a, const OpCtx& o, V in, V out) {
      const auto ins = Arrs(in);
      const EncDec e = ReadEncDec(a, ins.data(), ins.size());
      const int64_t n = encdec_attention_workspace(e.B, e.heads, e.kv_heads,
                                                   e.sq, e.sk, e.D,
                                                   e.q.dtype)[0];
      encdec_attention_fwd_raw(LC(o), e.q, e.kv, e.values, e.heads,
                               e.kv_heads, e.len, e.mask, e.tnc, out[0],
                               out[1], Scratch(o, n, kFloat32));
    };
    e.fcompute_cpu = EncDecCpu;
    e.fbackward = [](const TapeNode& n, const std::vector<NDArray>& og) {
      std::vector<NDArray> ins = {og[0], n.outputs[0], n.outputs[1]};
      ins.insert(ins.end(), n.inputs.begin(), n.inputs.end());
      auto outs = RunOp("_contrib_encdec_attention_bwd", n.attrs, ins);
      std::vector<NDArray> r(n.inputs.size());
      std::copy(outs.begin(), outs.end(), r.begin());
      return r;
    };
  }
  {
    OpEntry& e = OpRegistry::Get()->Register("_contrib_encdec_attention_bwd");
    e.infer = [](const NodeAttrs& a, const std::vector<TShape>& is,
                 const std::vector<int>& it, std::vector<TShape>* os,
                 std::vector<int>* ot) {
      const int n = a.GetBool("has_values", false) ? 3 : 2;
      os->assign(is.begin() + 3, is.begin() + 3 + n);
      ot->assign(it.begin() + 3, it.begin() + 3 + n);
    };
    e.fcompute_gpu = [](const NodeAttrs& a, const OpCtx& o, V in, V out) {
      const auto ins = Arrs(in, 3);
      const EncDec e = ReadEncDec(a, ins.data(), ins.size());
      const int64_t n = encdec_attention_workspace(e.B, e.heads, e.kv_heads,
                                                   e.sq, e.sk, e.D,
                                                   e.q.dtype)[1];
      encdec_attention_bwd_raw(LC(o), in[0], e.q, e.kv, e.values, e.heads,
                               e.kv_heads, e.len, e.mask, e.tnc, in[1], in[2],
                               out[0], out[1],
                               out.size() == 3 ? Arr(out[2]) : Arr(),
                               Scratch(o, n, kFloat32));
    };
    e.fcompute_cpu = EncDecBwdCpu;
  }
  {
    OpEntry& e = OpRegistry::Get()->Register("_contrib_sample_tokens");
    e.n_out = 2;
    e.infer = [](const NodeAttrs& a, const std::vector<TShape>& is,
                 const std::vector<int>& it, std::vector<TShape>* os,
                 std::vector<int>* ot) {
      MX_CHECK(is.size() >= 2 && is[0].size() == 2 && IsFloat(it[0]) &&
                   is[0][1] >= 1 && is[0][1] <= (1 << 19),
               "sample_tokens: rows of 1 to 2^19 logits");
      const TShape n = {is[0][0]};
      MX_CHECK(is[1] == n && it[1] == kFloat32,
               "sample_tokens: uniform must hold one float32 a row");
      size_t i = 2;
      for (const char* p : {"temperature", "top_k", "top_p", "min_p"})
        if (a.GetBool(std::string("has_") + p, false)) {
          MX_CHECK(i < is.size() && is[i] == n &&
                       (p[4] == 'k' ? it[i] == kInt32 || it[i] == kInt64
                                    : it[i] == kFloat32),
                   "sample_tokens: " << p << " must hold one value a row");
          ++i;
        }
      os->assign(2, n);
      *ot = {kInt32, kFloat32};
    };
    e.fcompute_gpu = [](const NodeAttrs& a, const OpCtx& o, V in, V out) {
      const SampleIn s = ReadSample(a, Arrs(in));
      sample_tokens_raw(
          LC(o), s.x, s.u, s.t, s.k, s.p, s.m, a.GetFloat("temperature", 1),
          a.GetInt("top_k", 0), a.GetFloat("top_p", 1),
          a.GetFloat("min_p", 0), out[0], out[1],
          Scratch(o, sample_tokens_workspace(s.x.size(0), s.x.size(1)),
                  kUint8));
    };
    e.fcompute_cpu = SampleCpu;
  }
  return true;
}();

}  // namespace
}  // namespace mxcore
