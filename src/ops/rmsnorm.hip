// Root-mean-square norm over the last axis, with the residual's addition in
// front and an int8 output with one scale a row.
//
//   h = data + residual                (rounded to the data's type: it is
//                                       stored, and the norm is of what is)
//   r = 1 / sqrt(mean(h^2) + eps)
//   y = h * r * gamma
//   int8: a = max|y|, scale = a * (1 / 127), q = rint(y * (127 * (1 / a))),
//         each factor rounded to 32 bits
//
//   backward, from dy and the sum's own gradient dsum:
//   g = dy * gamma, n = h * r
//   dh = r * (g - n * mean(g * n)) + dsum      (for data and residual alike)
//   dgamma = sum over rows of dy * n
//
// Both directions are bound by HBM: about ten operations for eight bytes
// moved.  So a row is read once and stays in registers between its sum and
// its output: a wave a row where it fits (no barrier at all), else a block.
// Measured with the residual and both gradients: 16384x4096 in bf16, forward
// 95 us (5.6 TB/s of reads and writes), backward 104 us (5.2 TB/s) and 5 for
// dgamma's partials; 4096x768 in fp16, 6.8 us, 8.4 and 3.2 (out of the caches,
// where launches and the rows' latency count); a large copy moves 5.1 TB/s.
// The sum of squares is held in 64 bits.  It costs no time here (64-bit FMAs
// run at the rate of 32-bit ones, far under the memory's time) and makes r
// the correctly rounded value, so that an int8 step does not depend on the
// order in which a row's squares were added.
#include "ops_api.h"

namespace mxcore {
namespace {

DEV_INLINE double wave_sum_f64(double v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

// sum over the TPR threads of a row; `red` holds one value a wave.  The two
// barriers keep a second call from overwriting what a slow wave still reads.
template <int TPR>
DEV_INLINE double row_sum(double v, double* red) {
  v = wave_sum_f64(v);
  if constexpr (TPR > 64) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int i = 0; i < TPR / 64; ++i) v += red[i];
    __syncthreads();
  }
  return v;
}

template <int TPR>
DEV_INLINE float row_sum_f32(float v, float* red) {
  v = wave_reduce_sum(v);
  if constexpr (TPR > 64) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int i = 0; i < TPR / 64; ++i) v += red[i];
    __syncthreads();
  }
  return v;
}

template <int TPR>
DEV_INLINE unsigned row_max(unsigned v, unsigned* red) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = max(v, __shfl_xor(v, off, 64));
  if constexpr (TPR > 64) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < TPR / 64; ++i) v = max(v, red[i]);
    __syncthreads();
  }
  return v;
}

DEV_INLINE float inv_rms(double sumsq, int C, double eps) {
  return (float)(1.0 / sqrt(sumsq / C + eps));
}

// The largest magnitude is taken of the values' bits, which order infinities
// and NaN (of the row, or that gamma made) above all numbers.
constexpr unsigned kInfBits = 0x7f800000u;
DEV_INLINE unsigned magnitude(float v) {
  return __float_as_uint(v) & 0x7fffffffu;
}

// a row's scale and its reciprocal.  A row of zeros (or so small that
// 127 / a overflows) quantises to zeros under a scale of 1; a row whose norm
// is not finite everywhere, to zeros under a scale of NaN.
DEV_INLINE void int8_scale(unsigned bits, float* scale, float* inv) {
  const float a = __uint_as_float(bits);
  *scale = a * (1.0f / 127.0f);
  *inv = 127.0f * (1.0f / a);
  if (bits == 0 || isinf(*inv)) {
    *scale = 1.f;
    *inv = 0.f;
  }
  if (bits >= kInfBits) {
    *scale = __builtin_nanf("");
    *inv = 0.f;
  }
}

DEV_INLINE signed char to_int8(float v) {
  float q = rintf(v);
  q = q > 127.f ? 127.f : q < -127.f ? -127.f : q;
  return q == q ? (signed char)q : (signed char)0;
}

// VEC elements of a row, of which `left` are there: aligned to 16 bytes and
// all there, or (LOOSE) neither.  The hardware reads and writes vectors at any
// element's address; a row's last ones go one by one, and zeros fill them up
// (4096 rows of 4097 in bf16, forward and backward: 24 us and 46, where all
// elements one by one take 50 and 92, and 4096 columns 19 and 32).
template <typename T, int VEC>
using Vec = T __attribute__((ext_vector_type(VEC)));

template <int VEC, bool LOOSE, bool ONCE = false, typename T>
DEV_INLINE Vec<T, VEC> load_vec(const T* p, int left) {
  using V = Vec<T, VEC>;
  typedef V U __attribute__((aligned(sizeof(T))));
  if constexpr (!LOOSE)
    return ONCE ? __builtin_nontemporal_load((const V*)p) : *(const V*)p;
  if (left >= VEC) return *(const U*)p;
  V v = {};
#pragma unroll
  for (int j = 0; j < VEC; ++j)
    if (j < left) v[j] = p[j];
  return v;
}

template <int VEC, bool LOOSE, typename T>
DEV_INLINE void store_vec(T* p, int left, Vec<T, VEC> v) {
  typedef Vec<T, VEC> U __attribute__((aligned(sizeof(T))));
  if constexpr (!LOOSE) {
    *(Vec<T, VEC>*)p = v;
    return;
  }
  if (left >= VEC) {
    *(U*)p = v;
    return;
  }
#pragma unroll
  for (int j = 0; j < VEC; ++j)
    if (j < left) p[j] = v[j];
}

// ---------------------------------------------------------------------------
// forward, the row in registers: TPR threads a row, NV vectors a thread.
// 32x1024 in fp16 (a step of decoding) takes 3.2 us, a launch's own time;
// 8192x1024 in bf16 to int8, 15.5 us (3.8 TB/s: 59 MB, partly from the cache).
// ---------------------------------------------------------------------------
template <typename T, int VEC, int TPR, int NV, bool LOOSE, bool RES, bool INT8>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void rms_fwd_kernel(
    const T* __restrict__ x, const T* __restrict__ res,
    const float* __restrict__ gamma, T* __restrict__ y,
    signed char* __restrict__ q, float* __restrict__ scale,
    T* __restrict__ sum, float* __restrict__ rstd, long rows, int C,
    double eps) {
  using VecT = Vec<T, VEC>;
  using VecG = Vec<float, VEC>;
  using VecQ = Vec<signed char, VEC>;
  constexpr int RPB = TPR < 256 ? 256 / TPR : 1;
  __shared__ double red[TPR > 64 ? TPR / 64 : 1];
  const int lane = threadIdx.x % TPR;
  const long row = (long)blockIdx.x * RPB + threadIdx.x / TPR;
  if (row >= rows) return;  // whole waves, and only where no barrier follows
  const long base = row * C;
  VecT h[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * TPR + lane) * VEC;
    if (c < C) h[i] = load_vec<VEC, LOOSE>(x + base + c, C - c);
  }
  double s = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * TPR + lane) * VEC;
    if (c < C) {
      if constexpr (RES) {
        const VecT r = load_vec<VEC, LOOSE>(res + base + c, C - c);
#pragma unroll
        for (int j = 0; j < VEC; ++j) h[i][j] = (T)((float)h[i][j] + (float)r[j]);
        store_vec<VEC, LOOSE>(sum + base + c, C - c, h[i]);
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const double f = (double)(float)h[i][j];
        s += f * f;
      }
    }
  }
  s = row_sum<TPR>(s, red);
  const float r = inv_rms(s, C, eps);
  if (!INT8 && rstd && lane == 0) rstd[row] = r;
  if constexpr (!INT8) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * VEC;
      if (c < C) {
        const VecG g = load_vec<VEC, LOOSE>(gamma + c, C - c);
        VecT o;
#pragma unroll
        for (int j = 0; j < VEC; ++j) o[j] = (T)((float)h[i][j] * r * g[j]);
        store_vec<VEC, LOOSE>(y + base + c, C - c, o);
      }
    }
  } else {
    float v[NV][VEC];
    unsigned a = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * VEC;
      if (c < C) {
        const VecG g = load_vec<VEC, LOOSE>(gamma + c, C - c);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          v[i][j] = (float)h[i][j] * r * g[j];
          a = max(a, magnitude(v[i][j]));
        }
      }
    }
    a = row_max<TPR>(a, (unsigned*)red);
    float sc, inv;
    int8_scale(a, &sc, &inv);
    if (lane == 0) scale[row] = sc;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * VEC;
      if (c < C) {
        VecQ o;
#pragma unroll
        for (int j = 0; j < VEC; ++j) o[j] = to_int8(v[i][j] * inv);
        store_vec<VEC, LOOSE>(q + base + c, C - c, o);
      }
    }
  }
}

// forward of rows that no register variant holds (over 32768 columns of 16
// bits, 16384 of 32): the row is read again, from the cache, an element at a
// time.  1024 rows of 65536 in bf16: forward 178 us (3.0 TB/s of what has to
// be moved), backward 314 (1.7); in fp32 317 and 465.
template <typename T, bool RES, bool INT8>
__global__ __launch_bounds__(1024) void rms_fwd_long_kernel(
    const T* __restrict__ x, const T* __restrict__ res,
    const float* __restrict__ gamma, T* __restrict__ y,
    signed char* __restrict__ q, float* __restrict__ scale,
    T* __restrict__ sum, float* __restrict__ rstd, long rows, int C,
    double eps) {
  __shared__ double red[16];
  for (long row = blockIdx.x; row < rows; row += gridDim.x) {
    const long base = row * C;
    auto value = [&](int c) {
      const float f = (float)x[base + c];
      return RES ? (float)(T)(f + (float)res[base + c]) : f;
    };
    double s = 0;
    for (int c = threadIdx.x; c < C; c += 1024) {
      const double f = value(c);
      s += f * f;
    }
    s = row_sum<1024>(s, red);
    const float r = inv_rms(s, C, eps);
    if (!INT8 && rstd && threadIdx.x == 0) rstd[row] = r;
    float sc = 0.f, inv = 0.f;
    if constexpr (INT8) {
      unsigned a = 0;
      for (int c = threadIdx.x; c < C; c += 1024)
        a = max(a, magnitude(value(c) * r * gamma[c]));
      a = row_max<1024>(a, (unsigned*)red);
      int8_scale(a, &sc, &inv);
      if (threadIdx.x == 0) scale[row] = sc;
    }
    for (int c = threadIdx.x; c < C; c += 1024) {
      const float f = value(c);
      if constexpr (RES) sum[base + c] = (T)f;
      if constexpr (INT8)
        q[base + c] = to_int8(f * r * gamma[c] * inv);
      else
        y[base + c] = (T)(f * r * gamma[c]);
    }
  }
}

// ---------------------------------------------------------------------------
// backward, one pass over dy, h (and dsum): a thread keeps its columns for
// all rows of its block, so dgamma's partial sums stay in registers; the
// blocks' partials are added by rms_dgamma_kernel in a fixed order.
// ---------------------------------------------------------------------------
template <typename T, int VEC, int TPR, int NV, bool LOOSE, bool DSUM>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void rms_bwd_kernel(
    const T* __restrict__ dy, const T* __restrict__ dsum,
    const T* __restrict__ h, const float* __restrict__ gamma,
    const float* __restrict__ rstd, T* __restrict__ dx,
    float* __restrict__ partial, long rows, int C) {
  using VecT = Vec<T, VEC>;
  using VecG = Vec<float, VEC>;
  constexpr int RPB = TPR < 256 ? 256 / TPR : 1;
  __shared__ float red[TPR > 64 ? TPR / 64 : 1];
  const int lane = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  float dg[NV][VEC] = {};
  // a row is on its way while the one before is reduced (16384x4096 bf16:
  // 112 us, 127 without), where the registers hold two.  Elsewhere they do not
  // hold dsum beside the row either: it is read where it is added
  constexpr bool AHEAD = TPR < 1024 || NV <= 2;
  VecT a[NV], b[NV], e[NV], na[NV], nb[NV], ne[NV];
  float r = 0.f, nr = 0.f;
  const long step = (long)gridDim.x * RPB;
  auto fetch = [&](long row) __attribute__((always_inline)) {
    const long base = row * C;
    nr = rstd[row];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * VEC;
      if (c < C) {
        na[i] = load_vec<VEC, LOOSE, true>(dy + base + c, C - c);
        nb[i] = load_vec<VEC, LOOSE>(h + base + c, C - c);
        if constexpr (DSUM && AHEAD)
          ne[i] = load_vec<VEC, LOOSE, true>(dsum + base + c, C - c);
      }
    }
  };
  long row = (long)blockIdx.x * RPB + sub;
  if (AHEAD && row < rows) fetch(row);
  for (; row < rows; row += step) {
    const long base = row * C;
    if (!AHEAD) fetch(row);
    r = nr;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      a[i] = na[i];
      b[i] = nb[i];
      if constexpr (DSUM && AHEAD) e[i] = ne[i];
    }
    if (AHEAD && row + step < rows) fetch(row + step);
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * VEC;
      if (c < C) {
        const VecG g = load_vec<VEC, LOOSE>(gamma + c, C - c);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float d = (float)a[i][j], n = (float)b[i][j] * r;
          m += d * g[j] * n;
          dg[i][j] += d * n;
        }
      }
    }
    m = row_sum_f32<TPR>(m, red) / C;
    // (without this the compiler keeps the row's products for the loop below,
    // in scratch memory where the registers do not hold them: 32768 columns.
    // Of four vectors of 16 bits, 5 to 9 registers still lie there.)
    if constexpr (!AHEAD) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        asm volatile("" : "+v"(*(int4_t*)&a[i]), "+v"(*(int4_t*)&b[i]));
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * VEC;
      if (c < C) {
        const VecG g = load_vec<VEC, LOOSE>(gamma + c, C - c);
        if constexpr (DSUM && !AHEAD)
          e[i] = load_vec<VEC, LOOSE, true>(dsum + base + c, C - c);
        VecT o;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          float v = r * ((float)a[i][j] * g[j] - (float)b[i][j] * r * m);
          if constexpr (DSUM) v += (float)e[i][j];
          o[j] = (T)v;
        }
        store_vec<VEC, LOOSE>(dx + base + c, C - c, o);
      }
    }
  }
  if constexpr (RPB == 1) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + lane) * VEC;
      if (c < C)
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          if (!LOOSE || c + j < C)
            partial[(long)blockIdx.x * C + c + j] = dg[i][j];
    }
  } else {
    __shared__ float part[RPB][TPR * NV * VEC];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        part[sub][(i * TPR + lane) * VEC + j] = dg[i][j];
    __syncthreads();
    for (int c = threadIdx.x; c < C; c += 256) {
      float v = 0.f;
#pragma unroll
      for (int k = 0; k < RPB; ++k) v += part[k][c];
      partial[(long)blockIdx.x * C + c] = v;
    }
  }
}

template <typename T, bool DSUM>
__global__ __launch_bounds__(1024) void rms_bwd_long_kernel(
    const T* __restrict__ dy, const T* __restrict__ dsum,
    const T* __restrict__ h, const float* __restrict__ gamma,
    const float* __restrict__ rstd, T* __restrict__ dx, long rows, int C) {
  __shared__ float red[16];
  for (long row = blockIdx.x; row < rows; row += gridDim.x) {
    const long base = row * C;
    const float r = rstd[row];
    float m = 0.f;
    for (int c = threadIdx.x; c < C; c += 1024)
      m += (float)dy[base + c] * gamma[c] * ((float)h[base + c] * r);
    m = row_sum_f32<1024>(m, red) / C;
    for (int c = threadIdx.x; c < C; c += 1024) {
      float v = r * ((float)dy[base + c] * gamma[c] -
                     (float)h[base + c] * r * m);
      if constexpr (DSUM) v += (float)dsum[base + c];
      dx[base + c] = (T)v;
    }
  }
}

// a thread a column over one block row's share of the rows
template <typename T>
__global__ __launch_bounds__(256) void rms_dgamma_long_kernel(
    const T* __restrict__ dy, const T* __restrict__ h,
    const float* __restrict__ rstd, float* __restrict__ partial, long rows,
    int C) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= C) return;
  float v = 0.f;
  for (long row = blockIdx.y; row < rows; row += gridDim.y)
    v += (float)dy[row * C + c] * ((float)h[row * C + c] * rstd[row]);
  partial[(long)blockIdx.y * C + c] = v;
}

// dgamma[c] = sum of the partials' column c (rows of them lie `stride` apart):
// 32 columns a block, 32 threads a column, eight reads of each on their way,
// always in the same order (512 partials of 768 columns: 3.2 us, bound by two
// rounds of latency)
__global__ __launch_bounds__(1024) void rms_dgamma_kernel(
    const float* __restrict__ partial, float* __restrict__ dgamma, int nblk,
    int C, long stride) {
  __shared__ float part[32][33];
  const int col = threadIdx.x & 31, k = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + col;
  float v = 0.f;
  if (c < C) {
#pragma unroll 8
    for (int b = k; b < nblk; b += 32) v += partial[b * stride + c];
  }
  part[k][col] = v;
  __syncthreads();
  // a wave takes two columns: 32 lanes add one
  const int mine = threadIdx.x >> 5, from = threadIdx.x & 31;
  v = part[from][mine];
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  if (from == 0 && blockIdx.x * 32 + mine < C) dgamma[blockIdx.x * 32 + mine] = v;
}

// ---------------------------------------------------------------------------
// Which variant: the smallest number of threads whose registers hold the row.
// A wave a row needs no barrier, but a launch of few rows wants a whole block
// on each, or most of the chip idles.  In bf16, forward and backward in us,
// a wave a row against a block:
//   512 rows of 768  3.3, 6.8 against 3.1, 6.3     of 2048  4.5, 9.2, 3.7, 7.9
//   1024 rows        3.4, 6.9 against 3.5, 7.4              5.0, 9.4, 4.3, 9.4
//   4096 rows        5.3, 10.0 against 7.4, 16.0            11, 18.5, 12, 22
// ---------------------------------------------------------------------------
struct RowPlan {
  int tpr = 0, nv = 0;  // 0: the kernel that reads the row again
  bool loose = false;   // rows that are not whole, aligned vectors
};

RowPlan plan_rows(long rows, int C, size_t size, bool aligned) {
  RowPlan p;
  const int vec = (int)(16 / size);
  p.loose = !aligned || C % vec;
  auto fits = [&](int tpr, int nv) {
    if (p.tpr == 0 && C <= (long)tpr * nv * vec) {
      p.tpr = tpr;
      p.nv = nv;
    }
  };
  if (rows >= 1024 || C <= 64 * vec) {
    fits(64, 1);
    fits(64, 2);
    fits(64, 4);
  }
  fits(256, 1);
  fits(256, 2);
  fits(256, 4);
  fits(1024, 2);
  fits(1024, 4);
  return p;
}

#define RMS_CASE(TPR_, NV_) \
  if (p.tpr == TPR_ && p.nv == NV_) { \
    constexpr int TPR = TPR_, NV = NV_; \
    if (p.loose) { \
      constexpr bool LOOSE = true; \
      LAUNCH(); \
    } else { \
      constexpr bool LOOSE = false; \
      LAUNCH(); \
    } \
    RETURN; \
  }

// LAUNCH sees VEC, TPR, NV and LOOSE as constants, RETURN follows it
#define RMS_DISPATCH() \
  RMS_CASE(64, 1) \
  RMS_CASE(64, 2) \
  RMS_CASE(64, 4) \
  RMS_CASE(256, 1) \
  RMS_CASE(256, 2) \
  RMS_CASE(256, 4) \
  RMS_CASE(1024, 2) \
  RMS_CASE(1024, 4)

bool aligned16(std::initializer_list<const void*> ps) {
  for (auto p : ps)
    if ((uintptr_t)p & 15) return false;
  return true;
}

void check_rows(const Arr& x, const Arr& gamma, const char* name) {
  MX_CHECK(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) < (1 << 30),
           name << ": the last axis must have 1 to 2^30 - 1 elements");
  MX_CHECK(gamma.dtype == kFloat32 && gamma.numel() == x.size(-1),
           name << ": gamma must be float32, one value a column");
  MX_CHECK(x.numel() / x.size(-1) < (1L << 31),
           name << ": 2^31 rows or more");
}

template <typename T, bool RES, bool INT8>
void fwd_launch(const LaunchCtx& lc, const Arr& x, const Arr& gamma,
                const Arr& res, double eps, const Arr& y, const Arr& scale,
                const Arr& sum, const Arr& rstd) {
  const int C = (int)x.size(-1);
  const long rows = x.numel() / C;
  RowPlan p = plan_rows(rows, C, sizeof(T),
                        aligned16({x.ptr, gamma.ptr, y.ptr, res.ptr,
                                   sum.ptr}));
  T* yp = INT8 ? nullptr : (T*)y.ptr;
  signed char* qp = INT8 ? (signed char*)y.ptr : nullptr;
  // a launch has fewer than 2^32 threads: 2^21 blocks of 1024 at most
  constexpr int VEC = 16 / sizeof(T);
#define RETURN return
#define LAUNCH()                                                            \
  constexpr int RPB = TPR < 256 ? 256 / TPR : 1;                            \
  for (long r0 = 0; r0 < rows; r0 += (1L << 21) * RPB) {                    \
    const long n = std::min(rows - r0, (1L << 21) * RPB), at = r0 * C;      \
    rms_fwd_kernel<T, VEC, TPR, NV, LOOSE, RES, INT8>                       \
        <<<(unsigned)((n + RPB - 1) / RPB), TPR < 256 ? 256 : TPR, 0,       \
           lc.stream>>>(                                                    \
            x.data<T>() + at, RES ? res.data<T>() + at : nullptr,           \
            gamma.data<float>(), INT8 ? nullptr : yp + at,                  \
            INT8 ? qp + at : nullptr,                                       \
            INT8 ? scale.data<float>() + r0 : nullptr,                      \
            RES ? sum.data<T>() + at : nullptr,                             \
            rstd.defined() ? rstd.data<float>() + r0 : nullptr, n, C, eps); \
  }
  RMS_DISPATCH()
#undef LAUNCH
#undef RETURN
  rms_fwd_long_kernel<T, RES, INT8>
      <<<(unsigned)std::min<long>(rows, 4096), 1024, 0, lc.stream>>>(
          x.data<T>(), res.data<T>(), gamma.data<float>(), yp, qp,
          scale.data<float>(), sum.data<T>(), rstd.data<float>(), rows, C,
          eps);
}

// returns the number of dgamma's partials, at most nblk
template <typename T, bool DSUM>
int bwd_launch(const LaunchCtx& lc, const Arr& dy, const Arr& dsum,
               const Arr& h, const Arr& gamma, const Arr& rstd, const Arr& dx,
               float* partial, int nblk) {
  const int C = (int)h.size(-1);
  const long rows = h.numel() / C;
  RowPlan p = plan_rows(rows, C, sizeof(T),
                        aligned16({dy.ptr, dsum.ptr, h.ptr, gamma.ptr,
                                   dx.ptr}));
  constexpr int VEC = 16 / sizeof(T);
#define RETURN return nblk
#define LAUNCH()                                                          \
  rms_bwd_kernel<T, VEC, TPR, NV, LOOSE, DSUM>                            \
      <<<(unsigned)nblk, TPR < 256 ? 256 : TPR, 0, lc.stream>>>(          \
          dy.data<T>(), dsum.data<T>(), h.data<T>(), gamma.data<float>(), \
          rstd.data<float>(), dx.data<T>(), partial, rows, C)
  RMS_DISPATCH()
#undef LAUNCH
#undef RETURN
  rms_bwd_long_kernel<T, DSUM>
      <<<(unsigned)std::min<long>(rows, 4096), 1024, 0, lc.stream>>>(
          dy.data<T>(), dsum.data<T>(), h.data<T>(), gamma.data<float>(),
          rstd.data<float>(), dx.data<T>(), rows, C);
  // (fewer than 2^32 threads: 2^23 blocks, or one for each 256 columns)
  const int columns = (C + 255) / 256;
  nblk = std::min(nblk, std::max(1, (1 << 23) / columns));
  rms_dgamma_long_kernel<T>
      <<<dim3((unsigned)columns, (unsigned)nblk), 256, 0, lc.stream>>>(
          dy.data<T>(), h.data<T>(), rstd.data<float>(), partial, rows, C);
  return nblk;
}

}  // namespace

void rms_norm_fwd_raw(const LaunchCtx& lc, const Arr& x, const Arr& gamma,
                      const Arr& residual, double eps, const Arr& y,
                      const Arr& scale, const Arr& sum, const Arr& rstd) {
  check_rows(x, gamma, "RMSNorm");
  const bool res = residual.defined(), int8 = y.dtype == kInt8;
  const long rows = x.numel() / x.size(-1);
  if (rows == 0) return;
  MX_CHECK(y.numel() == x.numel() && (int8 || y.dtype == x.dtype),
           "RMSNorm: the output must have the data's size, and its type or "
           "int8");
  MX_CHECK(!res || (residual.numel() == x.numel() &&
                    residual.dtype == x.dtype && sum.defined() &&
                    sum.numel() == x.numel() && sum.dtype == x.dtype),
           "RMSNorm: the residual and the sum must be like the data");
  const Arr& stat = int8 ? scale : rstd;
  MX_CHECK(stat.defined() ? stat.dtype == kFloat32 && stat.numel() == rows
                          : !int8,
           "RMSNorm: one float32 value a row is needed beside the output");
  DISPATCH_FLOAT_NATIVE(x.dtype, "RMSNorm", [&] {
    auto go = [&](auto r, auto q) {
      fwd_launch<scalar_t, decltype(r)::value, decltype(q)::value>(
          lc, x, gamma, residual, eps, y, scale, sum, rstd);
    };
    if (res && int8) go(std::true_type{}, std::true_type{});
    else if (res) go(std::true_type{}, std::false_type{});
    else if (int8) go(std::false_type{}, std::true_type{});
    else go(std::false_type{}, std::false_type{});
  });
  HIP_CHECK_LAST();
}

// Two blocks for each of 256 CUs, and no more than there are rows; four from
// 16384 rows on, of which a block then has 16 or more (768 columns: 25 us
// against 29 with two, 4096: 99 against 105, 2048: 53 against 52), since the
// partials are a row a block to write and to read again (4096 rows of 768:
// 10.7 us with four, 10.0 with two).
int64_t rms_norm_bwd_blocks(int64_t rows) {
  return std::max<int64_t>(1,
                           std::min<int64_t>(rows, rows < 16384 ? 512 : 1024));
}

void rms_norm_bwd_raw(const LaunchCtx& lc, const Arr& dy, const Arr& dsum,
                      const Arr& h, const Arr& gamma, const Arr& rstd,
                      const Arr& dx, const Arr& dgamma, const Arr& partial) {
  check_rows(h, gamma, "RMSNorm backward");
  const int64_t C = h.size(-1), rows = h.numel() / C;
  const int64_t nblk = rms_norm_bwd_blocks(rows);
  MX_CHECK(dy.numel() == h.numel() && dy.dtype == h.dtype &&
               dx.numel() == h.numel() && dx.dtype == h.dtype &&
               (!dsum.defined() ||
                (dsum.numel() == h.numel() && dsum.dtype == h.dtype)),
           "RMSNorm backward: the gradients must be like the data");
  MX_CHECK(rstd.dtype == kFloat32 && rstd.numel() == rows &&
               dgamma.dtype == kFloat32 && dgamma.numel() == C &&
               partial.dtype == kFloat32 && partial.numel() >= nblk * C,
           "RMSNorm backward: statistics, dgamma or workspace too small");
  int partials = 0;
  DISPATCH_FLOAT_NATIVE(h.dtype, "RMSNorm backward", [&] {
    if (rows == 0) return;
    partials = dsum.defined()
                   ? bwd_launch<scalar_t, true>(lc, dy, dsum, h, gamma, rstd,
                                                dx, partial.data<float>(),
                                                (int)nblk)
                   : bwd_launch<scalar_t, false>(lc, dy, dsum, h, gamma, rstd,
                                                 dx, partial.data<float>(),
                                                 (int)nblk);
  });
  // (fewer than 2^32 threads a launch: 2^26 columns)
  for (int64_t c = 0; c < C; c += 1 << 26) {
    const int64_t n = std::min<int64_t>(C - c, 1 << 26);
    rms_dgamma_kernel<<<(unsigned)((n + 31) / 32), 1024, 0, lc.stream>>>(
        partial.data<float>() + c, dgamma.data<float>() + c, partials, (int)n,
        C);
  }
  HIP_CHECK_LAST();
}

}  // namespace mxcore
