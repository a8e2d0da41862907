// Native elementwise / broadcast / reduce / fill / random operator family.
//
// Reference parity: src/operator/tensor/elemwise_binary_op.h:852 (RTC
// elementwise), broadcast_reduce-inl, init_op, sample_op.  The reference
// JIT-compiles these with NVRTC; here they are AOT-templated CDNA4 kernels
// (guide: vectorize 8-16 B/lane — hipcc does not auto-vectorize fp16 — and
// cap the grid, grid-striding the rest).  CPU variants are plain loops
// (the CPU implementation is the test oracle, reference test strategy).
#include "ew_common.h"

namespace mxcore {
namespace {

// ---------------------------------------------------------------------------
// functors (compute in fp32)
// ---------------------------------------------------------------------------
#define HD __host__ __device__ __forceinline__
struct FAdd { static HD float f(float a, float b) { return a + b; } };
struct FSub { static HD float f(float a, float b) { return a - b; } };
struct FMul { static HD float f(float a, float b) { return a * b; } };
struct FDiv { static HD float f(float a, float b) { return a / b; } };
struct FMax { static HD float f(float a, float b) { return a > b ? a : b; } };
struct FMin { static HD float f(float a, float b) { return a < b ? a : b; } };
struct FPow { static HD float f(float a, float b) { return powf(a, b); } };
struct FGe  { static HD float f(float a, float b) { return a >= b ? 1.f : 0.f; } };
struct FGt  { static HD float f(float a, float b) { return a > b ? 1.f : 0.f; } };
struct FLe  { static HD float f(float a, float b) { return a <= b ? 1.f : 0.f; } };
struct FLt  { static HD float f(float a, float b) { return a < b ? 1.f : 0.f; } };
struct FEq  { static HD float f(float a, float b) { return a == b ? 1.f : 0.f; } };
struct FNe  { static HD float f(float a, float b) { return a != b ? 1.f : 0.f; } };
// fused backward binaries: f(dy, saved)
struct FBwdRelu    { static HD float f(float dy, float y) { return y > 0.f ? dy : 0.f; } };
struct FBwdSigmoid { static HD float f(float dy, float y) { return dy * y * (1.f - y); } };
struct FBwdTanh    { static HD float f(float dy, float y) { return dy * (1.f - y * y); } };
struct FBwdSqrt    { static HD float f(float dy, float y) { return 0.5f * dy / y; } };
struct FBwdExp     { static HD float f(float dy, float y) { return dy * y; } };
struct FBwdLog     { static HD float f(float dy, float x) { return dy / x; } };
struct FBwdSquare  { static HD float f(float dy, float x) { return 2.f * dy * x; } };
struct FBwdAbs     { static HD float f(float dy, float x) { return x >= 0.f ? dy : -dy; } };
struct FBwdGelu {
  static HD float f(float dy, float x) {
    // d/dx [x * Phi(x)] with tanh approximation (matches forward)
    const float c = 0.7978845608f, a = 0.044715f;
    float x3 = x * x * x;
    float t = tanhf(c * (x + a * x3));
    float dt = (1.f - t * t) * c * (1.f + 3.f * a * x * x);
    return dy * (0.5f * (1.f + t) + 0.5f * x * dt);
  }
};

// unary functors: f(x, alpha, beta)
struct FRelu { static HD float f(float x, float, float) { return x > 0.f ? x : 0.f; } };
struct FSigmoid { static HD float f(float x, float, float) { return 1.f / (1.f + expf(-x)); } };
struct FTanh { static HD float f(float x, float, float) { return tanhf(x); } };
struct FExp { static HD float f(float x, float, float) { return expf(x); } };
struct FLog { static HD float f(float x, float, float) { return logf(x); } };
struct FSqrt { static HD float f(float x, float, float) { return sqrtf(x); } };
struct FSquare { static HD float f(float x, float, float) { return x * x; } };
struct FNeg { static HD float f(float x, float, float) { return -x; } };
struct FAbs { static HD float f(float x, float, float) { return fabsf(x); } };
struct FCopy { static HD float f(float x, float, float) { return x; } };
struct FGelu {
  static HD float f(float x, float, float) {
    const float c = 0.7978845608f, a = 0.044715f;
    return 0.5f * x * (1.f + tanhf(c * (x + a * x * x * x)));
  }
};
struct FAddS { static HD float f(float x, float a, float) { return x + a; } };
struct FRSubS { static HD float f(float x, float a, float) { return a - x; } };
struct FMulS { static HD float f(float x, float a, float) { return x * a; } };
struct FRDivS { static HD float f(float x, float a, float) { return a / x; } };
struct FPowS { static HD float f(float x, float a, float) { return powf(x, a); } };
struct FClip {
  static HD float f(float x, float lo, float hi) {
    return x < lo ? lo : (x > hi ? hi : x);
  }
};
struct FBwdClip {
  static HD float f(float dy, float x, float lo, float hi) {
    return (x > lo && x < hi) ? dy : 0.f;
  }
};
struct FLeaky { static HD float f(float x, float a, float) { return x > 0.f ? x : a * x; } };
struct FBwdLeaky { static HD float f(float dy, float x, float a, float) { return x > 0.f ? dy : a * dy; } };

template <typename T>
HD float ldf(const T& v) { return (float)v; }
template <typename T>
HD T stf(float v) { return (T)v; }

// ---------------------------------------------------------------------------
// GPU kernels
// ---------------------------------------------------------------------------
template <typename T, typename OP>
__global__ void bin_kernel(const T* __restrict__ a, const T* __restrict__ b,
                           T* __restrict__ y, long n) {
  // 16B/lane vectorized main body + scalar tail
  constexpr int V = 16 / sizeof(T);
  typedef T vec_t __attribute__((ext_vector_type(V)));
  long nv = n / V;
  for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < nv;
       i += (long)gridDim.x * blockDim.x) {
    vec_t va = ((const vec_t*)a)[i], vb = ((const vec_t*)b)[i], vy;
#pragma unroll
    for (int k = 0; k < V; ++k) vy[k] = stf<T>(OP::f(ldf(va[k]), ldf(vb[k])));
    ((vec_t*)y)[i] = vy;
  }
  for (long i = nv * V + (long)blockIdx.x * blockDim.x + threadIdx.x; i < n;
       i += (long)gridDim.x * blockDim.x)
    y[i] = stf<T>(OP::f(ldf(a[i]), ldf(b[i])));
}

template <typename T, typename OP>
__global__ void bin_strided_kernel(const T* __restrict__ a,
                                   const T* __restrict__ b, T* __restrict__ y,
                                   long n, Strides8 st) {
  for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < n;
       i += (long)gridDim.x * blockDim.x) {
    long rem = i, oa = 0, ob = 0;
#pragma unroll 4
    for (int d = st.ndim - 1; d >= 0; --d) {
      long idx = rem % st.shape[d];
      rem /= st.shape[d];
      oa += idx * st.s0[d];
      ob += idx * st.s1[d];
    }
    y[i] = stf<T>(OP::f(ldf(a[oa]), ldf(b[ob])));
  }
}

template <typename T, typename OP>
__global__ void unary_kernel(const T* __restrict__ x, T* __restrict__ y,
                             long n, float alpha, float beta) {
  constexpr int V = 16 / sizeof(T);
  typedef T vec_t __attribute__((ext_vector_type(V)));
  long nv = n / V;
  for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < nv;
       i += (long)gridDim.x * blockDim.x) {
    vec_t vx = ((const vec_t*)x)[i], vy;
#pragma unroll
    for (int k = 0; k < V; ++k) vy[k] = stf<T>(OP::f(ldf(vx[k]), alpha, beta));
    ((vec_t*)y)[i] = vy;
  }
  for (long i = nv * V + (long)blockIdx.x * blockDim.x + threadIdx.x; i < n;
       i += (long)gridDim.x * blockDim.x)
    y[i] = stf<T>(OP::f(ldf(x[i]), alpha, beta));
}

// ternary pointwise for clip-style backward: f(a, b, alpha, beta)
template <typename T, typename OP>
__global__ void bin_param_kernel(const T* __restrict__ a,
                                 const T* __restrict__ b, T* __restrict__ y,
                                 long n, float alpha, float beta) {
  for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < n;
       i += (long)gridDim.x * blockDim.x)
    y[i] = stf<T>(OP::f(ldf(a[i]), ldf(b[i]), alpha, beta));
}

// Only the 16-bit types go through float32: whole numbers, and float64, it
// does not hold.
template <typename TD, typename TS>
HD TD cast_value(TS v) {
  constexpr bool half = (std::is_same<TS, _Float16>::value ||
                         std::is_same<TS, __bf16>::value ||
                         std::is_same<TD, _Float16>::value ||
                         std::is_same<TD, __bf16>::value);
  if constexpr (half) return (TD)(float)v;
  else return (TD)v;
}

// MXC_DISPATCH_ALL, and the types that only a cast reads and writes
#define DISPATCH_CAST(DTYPE, NAME, ...)   \
  if ((DTYPE) == kFloat64) {              \
    using scalar_t = double;              \
    __VA_ARGS__                           \
  } else if ((DTYPE) == kInt8) {          \
    using scalar_t = signed char;         \
    __VA_ARGS__                           \
  } else {                                \
    MXC_DISPATCH_ALL(DTYPE, NAME, __VA_ARGS__) \
  }

template <typename TS, typename TD>
__global__ void cast_kernel(const TS* __restrict__ x, TD* __restrict__ y,
                            long n) {
  for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < n;
       i += (long)gridDim.x * blockDim.x)
    y[i] = cast_value<TD>(x[i]);
}

template <typename T>
__global__ void fill_kernel(T* __restrict__ y, long n, float v) {
  constexpr int V = 16 / sizeof(T);
  typedef T vec_t __attribute__((ext_vector_type(V)));
  long nv = n / V;
  T tv = stf<T>(v);
  vec_t vv;
#pragma unroll
  for (int k = 0; k < V; ++k) vv[k] = tv;
  for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < nv;
       i += (long)gridDim.x * blockDim.x)
    ((vec_t*)y)[i] = vv;
  for (long i = nv * V + (long)blockIdx.x * blockDim.x + threadIdx.x; i < n;
       i += (long)gridDim.x * blockDim.x)
    y[i] = tv;
}

// ---- philox4x32-10 counter-based RNG --------------------------------------
HD void philox_round(unsigned int& c0, unsigned int& c1, unsigned int& c2,
                     unsigned int& c3, unsigned int k0, unsigned int k1) {
  unsigned long long p0 = (unsigned long long)0xD2511F53u * c0;
  unsigned long long p1 = (unsigned long long)0xCD9E8D57u * c2;
  unsigned int h0 = (unsigned int)(p0 >> 32), l0 = (unsigned int)p0;
  unsigned int h1 = (unsigned int)(p1 >> 32), l1 = (unsigned int)p1;
  c0 = h1 ^ c1 ^ k0;
  c1 = l1;
  c2 = h0 ^ c3 ^ k1;
  c3 = l0;
}

HD void philox4(unsigned long long seed, unsigned long long idx,
                unsigned int out[4]) {
  unsigned int k0 = (unsigned int)seed, k1 = (unsigned int)(seed >> 32);
  unsigned int c0 = (unsigned int)idx, c1 = (unsigned int)(idx >> 32), c2 = 0xCAFEF00Du,
               c3 = 0xBAADF00Du;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    philox_round(c0, c1, c2, c3, k0, k1);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  out[0] = c0; out[1] = c1; out[2] = c2; out[3] = c3;
}

HD float u32_to_uniform(unsigned int v) {
  return (v >> 8) * (1.0f / 16777216.0f);  // [0,1)
}

template <typename T, bool NORMAL>
__global__ void random_kernel(T* __restrict__ y, long n,
                              unsigned long long seed, float p0, float p1) {
  for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i * 4 < n;
       i += (long)gridDim.x * blockDim.x) {
    unsigned int r[4];
    philox4(seed, (unsigned long long)i, r);
    float v[4];
    if (NORMAL) {
      // Box-Muller on pairs
      float u1 = u32_to_uniform(r[0]) + 1e-12f, u2 = u32_to_uniform(r[1]);
      float u3 = u32_to_uniform(r[2]) + 1e-12f, u4 = u32_to_uniform(r[3]);
      float m1 = sqrtf(-2.f * logf(u1)), m2 = sqrtf(-2.f * logf(u3));
      v[0] = p0 + p1 * m1 * __cosf(6.2831853f * u2);
      v[1] = p0 + p1 * m1 * __sinf(6.2831853f * u2);
      v[2] = p0 + p1 * m2 * __cosf(6.2831853f * u4);
      v[3] = p0 + p1 * m2 * __sinf(6.2831853f * u4);
    } else {
      for (int k = 0; k < 4; ++k)
        v[k] = p0 + (p1 - p0) * u32_to_uniform(r[k]);
    }
    long base = i * 4;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (base + k < n) y[base + k] = stf<T>(v[k]);
  }
}

// ---------------------------------------------------------------------------
// host wrappers
// ---------------------------------------------------------------------------
template <typename OP>
void BinGPU(const NodeAttrs&, const OpCtx& o, const std::vector<TBlob>& in,
            const std::vector<TBlob>& out) {
  long n = out[0].size();
  if (n == 0) return;
  bool same = in[0].shape == in[1].shape;
  MXC_DISPATCH_FLOAT(out[0].dtype, "binary", {
    if (same) {
      bin_kernel<scalar_t, OP><<<grid_for(n, 16 / sizeof(scalar_t)), kBlock, 0,
                                 o.rc.stream>>>(
          (const scalar_t*)in[0].dptr, (const scalar_t*)in[1].dptr,
          (scalar_t*)out[0].dptr, n);
    } else {
      Strides8 st = make_strides(out[0].shape, in[0].shape, in[1].shape);
      bin_strided_kernel<scalar_t, OP><<<grid_for(n), kBlock, 0,
                                         o.rc.stream>>>(
          (const scalar_t*)in[0].dptr, (const scalar_t*)in[1].dptr,
          (scalar_t*)out[0].dptr, n, st);
    }
  });
  HIP_CHECK_LAST();
}

template <typename OP>
void BinCPU(const NodeAttrs&, const OpCtx&, const std::vector<TBlob>& in,
            const std::vector<TBlob>& out) {
  long n = out[0].size();
  bool same = in[0].shape == in[1].shape;
  MXC_DISPATCH_FLOAT(out[0].dtype, "binary", {
    auto* a = (const scalar_t*)in[0].dptr;
    auto* b = (const scalar_t*)in[1].dptr;
    auto* y = (scalar_t*)out[0].dptr;
    if (same) {
      for (long i = 0; i < n; ++i) y[i] = stf<scalar_t>(OP::f(ldf(a[i]), ldf(b[i])));
    } else {
      Strides8 st = make_strides(out[0].shape, in[0].shape, in[1].shape);
      for (long i = 0; i < n; ++i) {
        long rem = i, oa = 0, ob = 0;
        for (int d = st.ndim - 1; d >= 0; --d) {
          long idx = rem % st.shape[d];
          rem /= st.shape[d];
          oa += idx * st.s0[d];
          ob += idx * st.s1[d];
        }
        y[i] = stf<scalar_t>(OP::f(ldf(a[oa]), ldf(b[ob])));
      }
    }
  });
}

template <typename OP>
void UnaryGPU(const NodeAttrs& at, const OpCtx& o, const std::vector<TBlob>& in,
              const std::vector<TBlob>& out) {
  long n = out[0].size();
  if (n == 0) return;
  float alpha = (float)at.GetFloat("alpha", 0.0);
  float beta = (float)at.GetFloat("beta", 0.0);
  MXC_DISPATCH_FLOAT(out[0].dtype, "unary", {
    unary_kernel<scalar_t, OP><<<grid_for(n, 16 / sizeof(scalar_t)), kBlock, 0,
                                 o.rc.stream>>>(
        (const scalar_t*)in[0].dptr, (scalar_t*)out[0].dptr, n, alpha, beta);
  });
  HIP_CHECK_LAST();
}

template <typename OP>
void UnaryCPU(const NodeAttrs& at, const OpCtx&, const std::vector<TBlob>& in,
              const std::vector<TBlob>& out) {
  long n = out[0].size();
  float alpha = (float)at.GetFloat("alpha", 0.0);
  float beta = (float)at.GetFloat("beta", 0.0);
  MXC_DISPATCH_FLOAT(out[0].dtype, "unary", {
    auto* x = (const scalar_t*)in[0].dptr;
    auto* y = (scalar_t*)out[0].dptr;
    for (long i = 0; i < n; ++i) y[i] = stf<scalar_t>(OP::f(ldf(x[i]), alpha, beta));
  });
}

template <typename OP>
void BinParamGPU(const NodeAttrs& at, const OpCtx& o,
                 const std::vector<TBlob>& in, const std::vector<TBlob>& out) {
  long n = out[0].size();
  float alpha = (float)at.GetFloat("alpha", 0.0);
  float beta = (float)at.GetFloat("beta", 0.0);
  MXC_DISPATCH_FLOAT(out[0].dtype, "binparam", {
    bin_param_kernel<scalar_t, OP><<<grid_for(n), kBlock, 0, o.rc.stream>>>(
        (const scalar_t*)in[0].dptr, (const scalar_t*)in[1].dptr,
        (scalar_t*)out[0].dptr, n, alpha, beta);
  });
  HIP_CHECK_LAST();
}

template <typename OP>
void BinParamCPU(const NodeAttrs& at, const OpCtx&,
                 const std::vector<TBlob>& in, const std::vector<TBlob>& out) {
  long n = out[0].size();
  float alpha = (float)at.GetFloat("alpha", 0.0);
  float beta = (float)at.GetFloat("beta", 0.0);
  MXC_DISPATCH_FLOAT(out[0].dtype, "binparam", {
    auto* a = (const scalar_t*)in[0].dptr;
    auto* b = (const scalar_t*)in[1].dptr;
    auto* y = (scalar_t*)out[0].dptr;
    for (long i = 0; i < n; ++i)
      y[i] = stf<scalar_t>(OP::f(ldf(a[i]), ldf(b[i]), alpha, beta));
  });
}

// ---------------------------------------------------------------------------
// registration helpers
// ---------------------------------------------------------------------------
NDArray RunOp(const char* name, const NodeAttrs& attrs,
              const std::vector<NDArray>& ins) {
  OpEntry* e = OpRegistry::Get()->Find(name);
  MX_CHECK(e, "op not registered: " << name);
  return Imperative::Run(e, attrs, ins)[0];
}

NDArray ReduceTo(const NDArray& dy, const TShape& target) {
  if (dy.shape() == target) return dy;
  NodeAttrs a;
  std::string s = "(";
  for (auto d : target) s += std::to_string(d) + ",";
  s += ")";
  a.d["shape"] = s;
  return RunOp("_reduce_to", a, {dy});
}

FBackward BwdPair(const char* da_op, const char* db_op) {
  // generic binary backward where da = da_op(dy, other), db = db_op(dy, other)
  std::string dao = da_op ? da_op : "", dbo = db_op ? db_op : "";
  return [dao, dbo](const TapeNode& n, const std::vector<NDArray>& og)
             -> std::vector<NDArray> {
    std::vector<NDArray> r(2);
    if (!dao.empty())
      r[0] = ReduceTo(RunOp(dao.c_str(), {}, {og[0], n.inputs[1]}),
                      n.inputs[0].shape());
    if (!dbo.empty())
      r[1] = ReduceTo(RunOp(dbo.c_str(), {}, {og[0], n.inputs[0]}),
                      n.inputs[1].shape());
    return r;
  };
}

struct Reg {
  OpEntry* e;
  explicit Reg(const char* name) {
    e = &OpRegistry::Get()->Register(name);
    e->n_out = 1;
  }
  Reg& in(int n) { e->n_in = n; return *this; }
  Reg& infer(FInferShape f) { e->infer = std::move(f); return *this; }
  Reg& gpu(FCompute f) { e->fcompute_gpu = std::move(f); return *this; }
  Reg& cpu(FCompute f) { e->fcompute_cpu = std::move(f); return *this; }
  Reg& bwd(FBackward f) { e->fbackward = std::move(f); return *this; }
};

// no-grad source / non-diff marker
FBackward NoGrad() {
  return [](const TapeNode& n, const std::vector<NDArray>&) {
    return std::vector<NDArray>(n.inputs.size());
  };
}

// ---------------------------------------------------------------------------
// op registrations
// ---------------------------------------------------------------------------
#define REG_BINARY(NAME, OP, ...)                                    \
  Reg(#NAME).in(2).infer(InferBroadcast())                            \
      .gpu(BinGPU<OP>).cpu(BinCPU<OP>).bwd(__VA_ARGS__)

#define REG_UNARY(NAME, OP, ...)                                      \
  Reg(#NAME).in(1).infer(InferSame())                                 \
      .gpu(UnaryGPU<OP>).cpu(UnaryCPU<OP>).bwd(__VA_ARGS__)

// unary backward via fused f(dy, saved) binary, saved = output
FBackward BwdFromOut(const char* op) {
  std::string o = op;
  return [o](const TapeNode& n, const std::vector<NDArray>& og)
             -> std::vector<NDArray> {
    return {RunOp(o.c_str(), {}, {og[0], n.outputs[0]})};
  };
}
FBackward BwdFromIn(const char* op) {
  std::string o = op;
  return [o](const TapeNode& n, const std::vector<NDArray>& og)
             -> std::vector<NDArray> {
    return {RunOp(o.c_str(), {}, {og[0], n.inputs[0]})};
  };
}

bool _registered = [] {
  // ---- binary (broadcasting) ----
  REG_BINARY(elemwise_add, FAdd, [](const TapeNode& n,
                                    const std::vector<NDArray>& og)
                                     -> std::vector<NDArray> {
    return {ReduceTo(og[0], n.inputs[0].shape()),
            ReduceTo(og[0], n.inputs[1].shape())};
  });
  REG_BINARY(elemwise_sub, FSub, [](const TapeNode& n,
                                    const std::vector<NDArray>& og)
                                     -> std::vector<NDArray> {
    return {ReduceTo(og[0], n.inputs[0].shape()),
            ReduceTo(RunOp("negative", {}, {og[0]}), n.inputs[1].shape())};
  });
  REG_BINARY(elemwise_mul, FMul, BwdPair("elemwise_mul", "elemwise_mul"));
  REG_BINARY(elemwise_div, FDiv, [](const TapeNode& n,
                                    const std::vector<NDArray>& og)
                                     -> std::vector<NDArray> {
    NDArray da = ReduceTo(RunOp("elemwise_div", {}, {og[0], n.inputs[1]}),
                          n.inputs[0].shape());
    NDArray t = RunOp("elemwise_mul", {}, {og[0], n.outputs[0]});
    t = RunOp("elemwise_div", {}, {t, n.inputs[1]});
    NDArray db = ReduceTo(RunOp("negative", {}, {t}), n.inputs[1].shape());
    return {da, db};
  });
  REG_BINARY(maximum, FMax, [](const TapeNode& n,
                               const std::vector<NDArray>& og)
                                -> std::vector<NDArray> {
    NDArray m = RunOp("greater_equal", {}, {n.inputs[0], n.inputs[1]});
    NDArray da = ReduceTo(RunOp("elemwise_mul", {}, {og[0], m}),
                          n.inputs[0].shape());
    NDArray one_minus = RunOp("_rminus_scalar",
                              [] { NodeAttrs a; a.d["alpha"] = "1"; return a; }(),
                              {m});
    NDArray db = ReduceTo(RunOp("elemwise_mul", {}, {og[0], one_minus}),
                          n.inputs[1].shape());
    return {da, db};
  });
  REG_BINARY(minimum, FMin, [](const TapeNode& n,
                               const std::vector<NDArray>& og)
                                -> std::vector<NDArray> {
    NDArray m = RunOp("less_equal", {}, {n.inputs[0], n.inputs[1]});
    NDArray da = ReduceTo(RunOp("elemwise_mul", {}, {og[0], m}),
                          n.inputs[0].shape());
    NDArray one_minus = RunOp("_rminus_scalar",
                              [] { NodeAttrs a; a.d["alpha"] = "1"; return a; }(),
                              {m});
    NDArray db = ReduceTo(RunOp("elemwise_mul", {}, {og[0], one_minus}),
                          n.inputs[1].shape());
    return {da, db};
  });
  REG_BINARY(greater_equal, FGe, NoGrad());
  REG_BINARY(greater, FGt, NoGrad());
  REG_BINARY(less_equal, FLe, NoGrad());
  REG_BINARY(less, FLt, NoGrad());
  REG_BINARY(equal, FEq, NoGrad());
  REG_BINARY(not_equal, FNe, NoGrad());
  REG_BINARY(power, FPow, [](const TapeNode& n, const std::vector<NDArray>& og)
                              -> std::vector<NDArray> {
    // da = dy * b * a^(b-1) = dy * b * y / a ; db = dy * y * ln a
    NDArray t = RunOp("elemwise_div", {}, {n.outputs[0], n.inputs[0]});
    t = RunOp("elemwise_mul", {}, {t, n.inputs[1]});
    NDArray da = ReduceTo(RunOp("elemwise_mul", {}, {og[0], t}),
                          n.inputs[0].shape());
    NDArray la = RunOp("log", {}, {n.inputs[0]});
    NDArray u = RunOp("elemwise_mul", {}, {n.outputs[0], la});
    NDArray db = ReduceTo(RunOp("elemwise_mul", {}, {og[0], u}),
                          n.inputs[1].shape());
    return {da, db};
  });

  // fused backward binaries (not recorded: used only inside backward)
  REG_BINARY(_backward_relu, FBwdRelu, NoGrad());
  REG_BINARY(_backward_sigmoid, FBwdSigmoid, NoGrad());
  REG_BINARY(_backward_tanh, FBwdTanh, NoGrad());
  REG_BINARY(_backward_sqrt, FBwdSqrt, NoGrad());
  REG_BINARY(_backward_exp, FBwdExp, NoGrad());
  REG_BINARY(_backward_log, FBwdLog, NoGrad());
  REG_BINARY(_backward_square, FBwdSquare, NoGrad());
  REG_BINARY(_backward_abs, FBwdAbs, NoGrad());
  REG_BINARY(_backward_gelu, FBwdGelu, NoGrad());

  // ---- unary ----
  REG_UNARY(relu, FRelu, BwdFromOut("_backward_relu"));
  REG_UNARY(sigmoid, FSigmoid, BwdFromOut("_backward_sigmoid"));
  REG_UNARY(tanh, FTanh, BwdFromOut("_backward_tanh"));
  REG_UNARY(exp, FExp, BwdFromOut("_backward_exp"));
  REG_UNARY(log, FLog, BwdFromIn("_backward_log"));
  REG_UNARY(sqrt, FSqrt, BwdFromOut("_backward_sqrt"));
  REG_UNARY(square, FSquare, BwdFromIn("_backward_square"));
  REG_UNARY(abs, FAbs, BwdFromIn("_backward_abs"));
  REG_UNARY(gelu, FGelu, BwdFromIn("_backward_gelu"));
  REG_UNARY(negative, FNeg, [](const TapeNode&, const std::vector<NDArray>& og)
                                -> std::vector<NDArray> {
    return {RunOp("negative", {}, {og[0]})};
  });
  REG_UNARY(_copy, FCopy, [](const TapeNode&, const std::vector<NDArray>& og)
                              -> std::vector<NDArray> { return {og[0]}; });
  REG_UNARY(leaky_relu, FLeaky, [](const TapeNode& n,
                                   const std::vector<NDArray>& og)
                                    -> std::vector<NDArray> {
    return {RunOp("_backward_leaky", n.attrs, {og[0], n.inputs[0]})};
  });
  Reg("_backward_leaky").in(2).infer(InferSame())
      .gpu(BinParamGPU<FBwdLeaky>).cpu(BinParamCPU<FBwdLeaky>).bwd(NoGrad());

  // scalar ops: alpha attr
  REG_UNARY(_plus_scalar, FAddS, [](const TapeNode&,
                                    const std::vector<NDArray>& og)
                                     -> std::vector<NDArray> { return {og[0]}; });
  REG_UNARY(_rminus_scalar, FRSubS, [](const TapeNode&,
                                       const std::vector<NDArray>& og)
                                        -> std::vector<NDArray> {
    return {RunOp("negative", {}, {og[0]})};
  });
  REG_UNARY(_mul_scalar, FMulS, [](const TapeNode& n,
                                   const std::vector<NDArray>& og)
                                    -> std::vector<NDArray> {
    return {RunOp("_mul_scalar", n.attrs, {og[0]})};
  });
  REG_UNARY(_rdiv_scalar, FRDivS, [](const TapeNode& n,
                                     const std::vector<NDArray>& og)
                                      -> std::vector<NDArray> {
    // y = a/x -> dx = -dy * y / x
    NDArray t = RunOp("elemwise_mul", {}, {og[0], n.outputs[0]});
    t = RunOp("elemwise_div", {}, {t, n.inputs[0]});
    return {RunOp("negative", {}, {t})};
  });
  REG_UNARY(_power_scalar, FPowS, [](const TapeNode& n,
                                     const std::vector<NDArray>& og)
                                      -> std::vector<NDArray> {
    double a = n.attrs.GetFloat("alpha", 1.0);
    NDArray t = RunOp("elemwise_div", {}, {n.outputs[0], n.inputs[0]});
    NodeAttrs m;
    m.d["alpha"] = std::to_string(a);
    t = RunOp("_mul_scalar", m, {t});
    return {RunOp("elemwise_mul", {}, {og[0], t})};
  });
  REG_UNARY(clip, FClip, [](const TapeNode& n, const std::vector<NDArray>& og)
                             -> std::vector<NDArray> {
    return {RunOp("_backward_clip", n.attrs, {og[0], n.inputs[0]})};
  });
  Reg("_backward_clip").in(2).infer(InferSame())
      .gpu(BinParamGPU<FBwdClip>).cpu(BinParamCPU<FBwdClip>).bwd(NoGrad());

  // in-place accumulate / copy (InvokeInto only)
  Reg("_grad_add").in(1).infer(InferSame())
      .gpu([](const NodeAttrs&, const OpCtx& o, const std::vector<TBlob>& in,
              const std::vector<TBlob>& out) {
        long n = out[0].size();
        MXC_DISPATCH_FLOAT(out[0].dtype, "_grad_add", {
          bin_kernel<scalar_t, FAdd><<<grid_for(n, 16 / sizeof(scalar_t)),
                                       kBlock, 0, o.rc.stream>>>(
              (const scalar_t*)in[0].dptr, (const scalar_t*)out[0].dptr,
              (scalar_t*)out[0].dptr, n);
        });
        HIP_CHECK_LAST();
      })
      .cpu([](const NodeAttrs&, const OpCtx&, const std::vector<TBlob>& in,
              const std::vector<TBlob>& out) {
        long n = out[0].size();
        MXC_DISPATCH_FLOAT(out[0].dtype, "_grad_add", {
          auto* a = (const scalar_t*)in[0].dptr;
          auto* y = (scalar_t*)out[0].dptr;
          for (long i = 0; i < n; ++i)
            y[i] = stf<scalar_t>(ldf(a[i]) + ldf(y[i]));
        });
      });
  Reg("_copy_into").in(1).infer(InferSame())
      .gpu([](const NodeAttrs&, const OpCtx& o, const std::vector<TBlob>& in,
              const std::vector<TBlob>& out) {
        size_t nb = (size_t)out[0].size() * dtype_size(out[0].dtype);
        MX_HIP_CALL(hipMemcpyAsync(out[0].dptr, in[0].dptr, nb,
                                   hipMemcpyDeviceToDevice, o.rc.stream));
      })
      .cpu([](const NodeAttrs&, const OpCtx&, const std::vector<TBlob>& in,
              const std::vector<TBlob>& out) {
        memcpy(out[0].dptr, in[0].dptr,
               (size_t)out[0].size() * dtype_size(out[0].dtype));
      });

  // ---- fills / sources ----
  auto infer_from_attrs = [](const NodeAttrs& a,
                             const std::vector<TShape>&,
                             const std::vector<int>&, std::vector<TShape>* os,
                             std::vector<int>* ot) {
    NodeAttrs at = a;
    std::vector<int64_t> s = at.GetTuple("shape", {});
    os->assign(1, TShape(s.begin(), s.end()));
    ot->assign(1, (int)at.GetInt("dtype", kFloat32));
  };
  auto fill_gpu = [](const NodeAttrs& a, const OpCtx& o,
                     const std::vector<TBlob>&, const std::vector<TBlob>& out) {
    long n = out[0].size();
    if (n == 0) return;
    float v = (float)a.GetFloat("value", 0.0);
    MXC_DISPATCH_ALL(out[0].dtype, "fill", {
      fill_kernel<scalar_t><<<grid_for(n, 16 / sizeof(scalar_t)), kBlock, 0,
                              o.rc.stream>>>((scalar_t*)out[0].dptr, n, v);
    });
    HIP_CHECK_LAST();
  };
  auto fill_cpu = [](const NodeAttrs& a, const OpCtx&,
                     const std::vector<TBlob>&, const std::vector<TBlob>& out) {
    long n = out[0].size();
    float v = (float)a.GetFloat("value", 0.0);
    MXC_DISPATCH_ALL(out[0].dtype, "fill", {
      auto* y = (scalar_t*)out[0].dptr;
      for (long i = 0; i < n; ++i) y[i] = (scalar_t)v;
    });
  };
  Reg("_full").in(0).infer(infer_from_attrs).gpu(fill_gpu).cpu(fill_cpu)
      .bwd(NoGrad());
  Reg("zeros_like").in(1).infer(InferSame())
      .gpu([fill_gpu](const NodeAttrs&, const OpCtx& o,
                      const std::vector<TBlob>& in,
                      const std::vector<TBlob>& out) {
        NodeAttrs a;
        a.d["value"] = "0";
        fill_gpu(a, o, in, out);
      })
      .cpu([fill_cpu](const NodeAttrs&, const OpCtx& o,
                      const std::vector<TBlob>& in,
                      const std::vector<TBlob>& out) {
        NodeAttrs a;
        a.d["value"] = "0";
        fill_cpu(a, o, in, out);
      })
      .bwd(NoGrad());
  Reg("ones_like").in(1).infer(InferSame())
      .gpu([fill_gpu](const NodeAttrs&, const OpCtx& o,
                      const std::vector<TBlob>& in,
                      const std::vector<TBlob>& out) {
        NodeAttrs a;
        a.d["value"] = "1";
        fill_gpu(a, o, in, out);
      })
      .cpu([fill_cpu](const NodeAttrs&, const OpCtx& o,
                      const std::vector<TBlob>& in,
                      const std::vector<TBlob>& out) {
        NodeAttrs a;
        a.d["value"] = "1";
        fill_cpu(a, o, in, out);
      })
      .bwd(NoGrad());

  // ---- random (philox4x32-10, reference sample_op via curand philox) ----
  auto rand_op = [](bool normal) {
    return [normal](const NodeAttrs& a, const OpCtx& o,
                    const std::vector<TBlob>&, const std::vector<TBlob>& out) {
      long n = out[0].size();
      if (n == 0) return;
      unsigned long long seed = (unsigned long long)a.GetInt("seed", 0);
      float p0 = (float)a.GetFloat(normal ? "loc" : "low", normal ? 0.0 : 0.0);
      float p1 = (float)a.GetFloat(normal ? "scale" : "high", 1.0);
      MXC_DISPATCH_FLOAT(out[0].dtype, "random", {
        if (normal)
          random_kernel<scalar_t, true><<<grid_for(n, 4), kBlock, 0,
                                          o.rc.stream>>>(
              (scalar_t*)out[0].dptr, n, seed, p0, p1);
        else
          random_kernel<scalar_t, false><<<grid_for(n, 4), kBlock, 0,
                                           o.rc.stream>>>(
              (scalar_t*)out[0].dptr, n, seed, p0, p1);
      });
      HIP_CHECK_LAST();
    };
  };
  auto rand_cpu = [](bool normal) {
    return [normal](const NodeAttrs& a, const OpCtx&,
                    const std::vector<TBlob>&, const std::vector<TBlob>& out) {
      long n = out[0].size();
      unsigned long long seed = (unsigned long long)a.GetInt("seed", 0);
      float p0 = (float)a.GetFloat(normal ? "loc" : "low", 0.0);
      float p1 = (float)a.GetFloat(normal ? "scale" : "high", 1.0);
      MXC_DISPATCH_FLOAT(out[0].dtype, "random", {
        auto* y = (scalar_t*)out[0].dptr;
        for (long i = 0; i * 4 < n; ++i) {
          unsigned int r[4];
          philox4(seed, (unsigned long long)i, r);
          float v[4];
          if (normal) {
            float u1 = u32_to_uniform(r[0]) + 1e-12f, u2 = u32_to_uniform(r[1]);
            float u3 = u32_to_uniform(r[2]) + 1e-12f, u4 = u32_to_uniform(r[3]);
            float m1 = sqrtf(-2.f * logf(u1)), m2 = sqrtf(-2.f * logf(u3));
            v[0] = p0 + p1 * m1 * cosf(6.2831853f * u2);
            v[1] = p0 + p1 * m1 * sinf(6.2831853f * u2);
            v[2] = p0 + p1 * m2 * cosf(6.2831853f * u4);
            v[3] = p0 + p1 * m2 * sinf(6.2831853f * u4);
          } else {
            for (int k = 0; k < 4; ++k)
              v[k] = p0 + (p1 - p0) * u32_to_uniform(r[k]);
          }
          for (int k = 0; k < 4 && i * 4 + k < n; ++k)
            y[i * 4 + k] = stf<scalar_t>(v[k]);
        }
      });
    };
  };
  Reg("_random_uniform").in(0).infer(infer_from_attrs)
      .gpu(rand_op(false)).cpu(rand_cpu(false)).bwd(NoGrad());
  Reg("_random_normal").in(0).infer(infer_from_attrs)
      .gpu(rand_op(true)).cpu(rand_cpu(true)).bwd(NoGrad());

  // ---- cast ----
  Reg("cast").in(1)
      .infer([](const NodeAttrs& a, const std::vector<TShape>& is,
                const std::vector<int>&, std::vector<TShape>* os,
                std::vector<int>* ot) {
        os->assign(1, is[0]);
        ot->assign(1, (int)a.GetInt("dtype", kFloat32));
      })
      .gpu([](const NodeAttrs&, const OpCtx& o, const std::vector<TBlob>& in,
              const std::vector<TBlob>& out) {
        long n = out[0].size();
        if (n == 0) return;
        DISPATCH_CAST(in[0].dtype, "cast_src", {
          using src_t = scalar_t;
          DISPATCH_CAST(out[0].dtype, "cast_dst", {
            cast_kernel<src_t, scalar_t><<<grid_for(n), kBlock, 0,
                                           o.rc.stream>>>(
                (const src_t*)in[0].dptr, (scalar_t*)out[0].dptr, n);
          });
        });
        HIP_CHECK_LAST();
      })
      .cpu([](const NodeAttrs&, const OpCtx&, const std::vector<TBlob>& in,
              const std::vector<TBlob>& out) {
        long n = out[0].size();
        DISPATCH_CAST(in[0].dtype, "cast_src", {
          using src_t = scalar_t;
          auto* x = (const src_t*)in[0].dptr;
          DISPATCH_CAST(out[0].dtype, "cast_dst", {
            auto* y = (scalar_t*)out[0].dptr;
            for (long i = 0; i < n; ++i) y[i] = cast_value<scalar_t>(x[i]);
          });
        });
      })
      .bwd([](const TapeNode& n, const std::vector<NDArray>& og)
               -> std::vector<NDArray> {
        NodeAttrs a;
        a.d["dtype"] = std::to_string(n.inputs[0].dtype());
        return {RunOp("cast", a, {og[0]})};
      });

  return true;
}();

}  // namespace

// comm-stream helper (rccl_comm.cc): in-place scale without at:: / registry
void ScaleInPlace(void* p, int64_t n, int dtype, float alpha,
                  hipStream_t s) {
  MXC_DISPATCH_FLOAT(dtype, "scale_inplace", {
    unary_kernel<scalar_t, FMulS><<<grid_for(n, 16 / sizeof(scalar_t)),
                                    kBlock, 0, s>>>(
        (const scalar_t*)p, (scalar_t*)p, n, alpha, 0.f);
  });
  HIP_CHECK_LAST();
}

}  // namespace mxcore
