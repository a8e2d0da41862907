// The next token of each row of logits, from given random numbers.
//
//   order: by logit, the largest first; the lower index first among equals
//   w_i = exp((x_i - max) / T)
//   kept: the first top_k of the order; of those the shortest prefix that
//         holds top_p of their sum; of those the ones with w_i >= min_p
//   token: the first in the order whose running sum exceeds u * (kept sum)
//
// Every step asks for a prefix of one order, so the row is never sorted: it is
// counted into 2048 buckets of (max - x) / T, 1/64 wide (the weight of each,
// and for top_k the number), which answers every question up to one bucket;
// only that bucket's few entries are gathered, sorted and looked at one by one.
//
// Weights are 64-bit: whether a token is kept or drawn lies next to a border.
// They are counted as whole numbers of 2^-s (s = 62 - ceil(log2 V), at most
// 51), so that sums cannot overflow and do not depend on the order in which
// lanes and blocks add.
//
// Bound by latency for few rows and by the 64-bit exponentials for many.  The
// logits are read from memory once and scanned again from the cache.  Rows
// that fill the chip, and short ones, take one launch with a block a row; else
// two launches cut each row into parts for the maximum and the counts, and a
// third answers.
#include "ops_api.h"

namespace mxcore {
namespace {

constexpr int NB = 2048;      // buckets
constexpr float STEP = 64.f;  // buckets for each unit of (max - x) / T
constexpr int LIST = 2048;    // entries that are sorted in LDS
constexpr int NT = 1024;      // threads of the block that answers for a row
constexpr float kInf = __builtin_huge_valf();
typedef unsigned long long u64;

struct Sample {
  const void* x;
  long V;
  int N, parts;
  const float* u;
  // one a row where the pointer is given, else the value
  const float *tp, *pp, *mp;
  const int* kp;
  double t, p, m;
  int k;
  int sbits;
  int* token;
  float* logp;
  // workspace, where a row is cut into parts
  u64* mass;        // [N, NB]
  unsigned* count;  // [N, NB]
  float* pmax;      // [N, parts]
};

struct Row {
  double inv;    // 1 / T
  float finv;    // buckets for each unit of logit
  float top;
  bool greedy;
};

// NaN counts as -inf: it is never drawn
template <typename T>
DEV_INLINE float logit(T x) {
  const float v = (float)x;
  return v == v ? v : -kInf;
}

// f(index, logit) over [i0, i1) by the block's threads, 16 bytes at a time
// where the memory is aligned
template <typename T, int THREADS, typename F>
DEV_INLINE void scan(const T* x, long i0, long i1, F f) {
  constexpr int N = 16 / sizeof(T);
  using VecT = T __attribute__((ext_vector_type(N)));
  long a = i0 + ((-(uintptr_t)(x + i0) & 15) / sizeof(T));
  if (a > i1) a = i1;
  const long nv = (i1 - a) / N;
  for (long i = i0 + threadIdx.x; i < a; i += THREADS) f(i, logit(x[i]));
  for (long k = threadIdx.x; k < nv; k += THREADS) {
    const VecT v = *(const VecT*)(x + a + k * N);
#pragma unroll
    for (int j = 0; j < N; ++j) f(a + k * N + j, logit(v[j]));
  }
  for (long i = a + nv * N + threadIdx.x; i < i1; i += THREADS)
    f(i, logit(x[i]));
}

// non-increasing in v, so buckets follow the order
DEV_INLINE int bucket(float v, const Row& r) {
  if (v == r.top) return 0;
  const float b = (r.top - v) * r.finv;
  return b < (float)(NB - 1) ? (int)b : NB - 1;  // NaN (inf * 0): the last
}

// (max - x) / T; 0 for an infinite maximum itself
DEV_INLINE double depth(float v, const Row& r) {
  if (v == r.top) return 0.0;
  return r.greedy ? (double)kInf : ((double)r.top - (double)v) * r.inv;
}

// 2^s exp(-d), rounded to a whole number: exp(-d) = 2^-n e^r with |r| <=
// ln(2) / 2, e^r by its Taylor series to the 11th power (off by 7e-15, a
// quarter of 2^-s at 10^5 logits).  Adding 2^52 (1.5 * 2^52 where the number
// may be negative) rounds a double to a whole number in its lowest bits.
DEV_INLINE u64 weight(double d, int sbits) {
  if (!(d < 45.0)) return 0;  // under 2^-64
  const double t = fma(d, 1.4426950408889634, 0x1.8p52), n = t - 0x1.8p52;
  // ln 2 to 107 bits, as two doubles
  double r = fma(n, 0.6931471805599453, -d);
  r = fma(n, 2.3190468138462996e-17, r);
  double e = 1.0 / 39916800.0;
  e = fma(e, r, 1.0 / 3628800.0);
  e = fma(e, r, 1.0 / 362880.0);
  e = fma(e, r, 1.0 / 40320.0);
  e = fma(e, r, 1.0 / 5040.0);
  e = fma(e, r, 1.0 / 720.0);
  e = fma(e, r, 1.0 / 120.0);
  e = fma(e, r, 1.0 / 24.0);
  e = fma(e, r, 1.0 / 6.0);
  e = fma(e, r, 0.5);
  e = fma(e, r, 1.0);
  e = fma(e, r, 1.0);
  // 2^(s - n); n is t's lowest bits
  const int x = 1023 + sbits - (int)__double2loint(t);
  const double f = __hiloint2double(x << 20, 0);
  return (u64)__double_as_longlong(fma(e, f, 0x1p52)) - 0x4330000000000000ull;
}

// the order as ascending numbers: larger logits first, then lower indices
DEV_INLINE u64 entry(float v, long i) {
  if (v == 0.f) v = 0.f;  // -0 and 0 are equal
  unsigned k = __float_as_uint(v);
  k = k & 0x80000000u ? k : ~k & 0x7fffffffu;
  return (u64)k << 32 | (unsigned)i;
}
DEV_INLINE float entry_logit(u64 e) {
  unsigned k = (unsigned)(e >> 32);
  k = k & 0x80000000u ? k : ~k & 0x7fffffffu;
  return __uint_as_float(k);
}

DEV_INLINE double temperature(const Sample& a, int n) {
  return a.tp ? (double)a.tp[n] : a.t;
}

DEV_INLINE Row make_row(double temp, float top) {
  Row r;
  r.greedy = !(temp > 0.0);
  r.inv = r.greedy ? 0.0 : 1.0 / temp;
  r.finv = r.greedy ? kInf : (float)(r.inv * STEP);
  r.top = top;
  return r;
}

// ---------------------------------------------------------------------------
// rows cut into parts: 1. each part's maximum; the row's counts are cleared
// ---------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void sample_max_kernel(Sample a) {
  __shared__ float red[4];
  const int n = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
  float top = -kInf;
  scan<T, 256>((const T*)a.x + n * a.V, a.V * part / a.parts,
               a.V * (part + 1) / a.parts,
               [&](long, float v) { top = fmaxf(top, v); });
  top = wave_reduce_max(top);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
  __syncthreads();
  if (threadIdx.x == 0)
    a.pmax[(long)n * a.parts + part] =
        fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  for (int b = part * 256 + threadIdx.x; b < NB; b += a.parts * 256) {
    a.mass[(long)n * NB + b] = 0;
    a.count[(long)n * NB + b] = 0;
  }
}

DEV_INLINE float parts_top(const Sample& a, int n) {
  float top = -kInf;
  for (int p = 0; p < a.parts; ++p)
    top = fmaxf(top, a.pmax[(long)n * a.parts + p]);
  return top;
}

// 2. number and weight of each bucket
template <int THREADS, typename T>
DEV_INLINE void count_row(const Sample& a, const T* x, long i0, long i1,
                          const Row& r, bool number, u64* mass,
                          unsigned* count) {
  scan<T, THREADS>(x, i0, i1, [&](long, float v) {
    const int b = bucket(v, r);
    if (number) atomicAdd(&count[b], 1u);
    const u64 w = weight(depth(v, r), a.sbits);
    if (w) atomicAdd(&mass[b], w);
  });
}

// how many the row may keep; 0: all.  The numbers are counted only for this
DEV_INLINE int number_kept(const Sample& a, int n, const Row& r) {
  const int k = r.greedy ? 1 : a.kp ? a.kp[n] : a.k;
  return k > 0 && k < a.V ? k : 0;
}

template <typename T>
__global__ __launch_bounds__(256) void sample_count_kernel(Sample a) {
  __shared__ u64 mass[NB];
  __shared__ unsigned count[NB];
  const int n = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
  for (int b = threadIdx.x; b < NB; b += 256) {
    mass[b] = 0;
    count[b] = 0;
  }
  const Row r = make_row(temperature(a, n), parts_top(a, n));
  __syncthreads();
  count_row<256>(a, (const T*)a.x + n * a.V, a.V * part / a.parts,
                 a.V * (part + 1) / a.parts, r, number_kept(a, n, r) != 0,
                 mass, count);
  __syncthreads();
  for (int b = threadIdx.x; b < NB; b += 256) {
    if (count[b]) atomicAdd(&a.count[(long)n * NB + b], count[b]);
    if (mass[b]) atomicAdd(&a.mass[(long)n * NB + b], mass[b]);
  }
}

// ---------------------------------------------------------------------------
// 3. the answers: a block a row
// ---------------------------------------------------------------------------
struct Lds {
  u64 mass[NB];
  unsigned count[NB];
  union {
    u64 list[LIST];
    struct {  // while a bucket is too full for the list
      u64 mass[NB];
      unsigned count[NB];
    } fine;
  };
  u64 wave[2][NT / 64];
  u64 at, before[2], through;
  int found;
  unsigned n;
};

// running sum of the threads before this one; *total: of all
DEV_INLINE u64 sum_before(u64 v, u64* wave, u64* total) {
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6;
  u64 in = v;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const u64 p = (u64)__shfl_up(in, off, 64);
    if (l >= off) in += p;
  }
  if (l == 63) wave[w] = in;
  __syncthreads();
  u64 b = 0, all = 0;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) {
    if (i == w) b = all;
    all += wave[i];
  }
  __syncthreads();
  *total = all;
  return b + in - v;
}

// a question to the order: its first entry ...
struct Ask {
  enum Kind {
    kNumber,  // ... whose running number is at least want
    kWeight,  // ... whose running weight is at least want
    kOver,    // ... whose running weight is over want
  } kind;
  double want;
};

DEV_INLINE bool reached(const Ask& q, u64 through) {
  return q.kind == Ask::kOver ? (double)through > q.want
                              : (double)through >= q.want;
}

// The first of NB buckets (two to a thread) with which the question is
// reached, NB if none, and the weight and number before it.  `weight0` and
// `number0` lie before all of them.  The first bucket that holds anything may
// be reached already by what lies before it.
DEV_INLINE int find_bucket(const Ask& q, const u64* mass,
                           const unsigned* count, u64 weight0, u64 number0,
                           Lds& s, u64* weight1, u64* number1) {
  const int b = threadIdx.x * 2;
  const bool number = q.kind == Ask::kNumber;
  const u64 m0 = mass[b], m1 = mass[b + 1];
  const u64 v0 = number ? count[b] : m0, v1 = number ? count[b + 1] : m1;
  const u64 base = number ? number0 : weight0;
  if (threadIdx.x == 0) s.found = NB;
  u64 all, m = 0;
  const u64 p0 = base + sum_before(v0 + v1, s.wave[0], &all), p1 = p0 + v0,
            p2 = p1 + v1;
  if (number) m = weight0 + sum_before(m0 + m1, s.wave[1], &all);
  // an empty bucket reaches nothing
  if (v0 && reached(q, p1) && !(p0 > base && reached(q, p0))) {
    s.found = b;
    s.before[0] = number ? m : p0;
    s.before[1] = p0;
  } else if (v1 && reached(q, p2) && !(p1 > base && reached(q, p1))) {
    s.found = b + 1;
    s.before[0] = number ? m + m0 : p1;
    s.before[1] = p1;
  }
  __syncthreads();
  const int k = s.found;
  *weight1 = s.before[0];
  *number1 = s.before[1];
  __syncthreads();
  return k;
}

// The least logit whose bucket is at most b, by a search in which each lane
// looks at one of 64 places.  Buckets follow the order, so a bucket is a
// range of logits, and a scan needs two comparisons for each.
DEV_INLINE float least_logit(int b, const Row& r) {
  auto number = [](float v) {
    const unsigned u = __float_as_uint(v);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
  };
  auto value = [](unsigned k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
  };
  // the bucket is over b at lo and at most b at hi
  unsigned lo = number(-kInf), hi = number(r.top);
  while (hi - lo > 1) {
    const unsigned step = (hi - lo + 63) / 64;
    const unsigned at = min(lo + step * ((threadIdx.x & 63) + 1), hi);
    const int first = __ffsll((unsigned long long)__ballot(
                          bucket(value(at), r) <= b)) - 1;
    const unsigned to = min(lo + step * (first + 1), hi);
    lo += step * first;
    hi = to;
  }
  return value(hi);
}

// which entries the list holds, so that the next question to the same bucket
// need not gather them again
struct Held {
  int bucket;
  unsigned n;
};

// The list in order: a pair of entries to a thread.  A wave's pairs lie in
// 128 places of its own while they are at most 64 apart, so only wider steps
// wait for the other waves.
DEV_INLINE void sort_list(Lds& s, int size) {
  const int i = threadIdx.x;
  for (int k = 2; k <= size; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      if (i < size / 2) {
        const int i0 = 2 * i - (i & (j - 1)), i1 = i0 + j;
        const u64 e0 = s.list[i0], e1 = s.list[i1];
        if ((e0 > e1) == ((i0 & k) == 0)) {
          s.list[i0] = e1;
          s.list[i1] = e0;
        }
      }
      if (j > 64 || (j == 1 && k >= 128)) {
        __syncthreads();
      } else {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
      }
    }
  __syncthreads();
}

// The question's entry, and the weight through it.  False where it lies in the
// last bucket or nowhere: the weights there add up to less than 2^-24 of the
// row's, so no random number below 1 draws them.
template <typename T>
DEV_INLINE bool ask(const Sample& a, const T* x, const Row& r, const Ask& q,
                    Lds& s, Held& held, u64* at, u64* through) {
  u64 weight0, number0;
  const int b = find_bucket(q, s.mass, s.count, 0, 0, s, &weight0, &number0);
  if (b >= NB - 1) return false;
  if (held.bucket != b) {
    held.bucket = -1;
    const float vlo = least_logit(b, r);
    const float vhi = b ? least_logit(b - 1, r) : kInf;
    // entries of the bucket between lo and hi, both included
    auto each = [&](u64 lo, u64 hi, auto f) {
      scan<T, NT>(x, 0, a.V, [&](long i, float v) {
        if (!(v >= vlo && (v < vhi || b == 0))) return;
        const u64 e = entry(v, i);
        if (e >= lo && e <= hi) f(v, e);
      });
    };
    auto gather = [&](u64 lo, u64 hi) {
      if (threadIdx.x == 0) s.n = 0;
      __syncthreads();
      each(lo, hi, [&](float, u64 e) {
        const unsigned k = atomicAdd(&s.n, 1u);
        if (k < LIST) s.list[k] = e;
      });
      __syncthreads();
      return s.n;
    };
    u64 lo = 0, hi = ~0ull;
    unsigned n = gather(lo, hi);
    const bool whole = n <= LIST;
    // a bucket that the list cannot hold (many equal logits) is divided by
    // the entries' own bits until it can: by 2^10 or more each time
    while (n > LIST) {
      u64 least = ~0ull, most = 0;
      each(lo, hi, [&](float, u64 e) {
        least = min(least, e);
        most = max(most, e);
      });
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) {
        least = min(least, (u64)__shfl_xor(least, off, 64));
        most = max(most, (u64)__shfl_xor(most, off, 64));
      }
      if ((threadIdx.x & 63) == 0) {
        s.wave[0][threadIdx.x >> 6] = least;
        s.wave[1][threadIdx.x >> 6] = most;
      }
      __syncthreads();  // (and every thread has read s.n)
      for (int i = threadIdx.x; i < NB; i += NT) {
        s.fine.mass[i] = 0;
        s.fine.count[i] = 0;
      }
#pragma unroll
      for (int i = 0; i < NT / 64; ++i) {
        least = min(least, s.wave[0][i]);
        most = max(most, s.wave[1][i]);
      }
      __syncthreads();
      // more than LIST different entries: most - least has 11 bits or more
      const int shift = 53 - (int)__clzll((long long)(most - least));
      each(least, most, [&](float v, u64 e) {
        const int k = (int)((e - least) >> shift);
        atomicAdd(&s.fine.count[k], 1u);
        const u64 w = weight(depth(v, r), a.sbits);
        if (w) atomicAdd(&s.fine.mass[k], w);
      });
      __syncthreads();
      const int k = find_bucket(q, s.fine.mass, s.fine.count, weight0,
                                number0, s, &weight0, &number0);
      if (k == NB) return false;
      n = s.fine.count[k];
      lo = least + ((u64)k << shift);
      hi = lo + ((1ull << shift) - 1);
      __syncthreads();
      if (n <= LIST) n = gather(lo, hi);
    }
    int size = 2;
    while (size < (int)n) size <<= 1;
    for (int i = n + threadIdx.x; i < size; i += NT) s.list[i] = ~0ull;
    __syncthreads();
    sort_list(s, size);
    // (a part of a bucket is not kept for the next question)
    held = Held{whole ? b : -1, n};
  }
  const int n = (int)held.n, i0 = threadIdx.x * 2;
  const bool number = q.kind == Ask::kNumber;
  u64 w[2];
#pragma unroll
  for (int j = 0; j < 2; ++j)
    w[j] = i0 + j < n
               ? weight(depth(entry_logit(s.list[i0 + j]), r), a.sbits) : 0;
  if (threadIdx.x == 0) s.found = LIST;
  u64 all;
  const u64 p1 = weight0 + sum_before(w[0] + w[1], s.wave[0], &all) + w[0],
            p2 = p1 + w[1];
  const int hit =
      i0 < n && reached(q, number ? number0 + i0 + 1 : p1)       ? i0
      : i0 + 1 < n && reached(q, number ? number0 + i0 + 2 : p2) ? i0 + 1
                                                                 : LIST;
  if (hit < LIST) atomicMin(&s.found, hit);
  __syncthreads();
  const int first = s.found;
  if (first < LIST && first == hit) {
    s.at = s.list[first];
    s.through = first & 1 ? p2 : p1;
  }
  __syncthreads();
  *at = s.at;
  *through = s.through;
  __syncthreads();
  return first < LIST;
}

// the weight of the entries that are at most `most` deep
template <typename T>
DEV_INLINE u64 shallow(const Sample& a, const T* x, const Row& r, double most,
                       Lds& s) {
  // the buckets' bounds are rounded by less than one bucket
  const int b = max((int)(most * (double)STEP) - 1, 0);
  u64 v = 0, all;
  for (int i = threadIdx.x; i < b; i += NT) v += s.mass[i];
  const float vlo = least_logit(b + 2, r);
  const float vhi = b ? least_logit(b - 1, r) : kInf;
  scan<T, NT>(x, 0, a.V, [&](long, float z) {
    if (!(z >= vlo && (z < vhi || b == 0))) return;
    const double d = depth(z, r);
    if (d <= most) v += weight(d, a.sbits);
  });
  sum_before(v, s.wave[0], &all);
  return all;
}

template <typename T, bool COUNTED>
__global__ __launch_bounds__(NT) void sample_kernel(Sample a) {
  __shared__ Lds s;
  const int n = blockIdx.x, t = threadIdx.x;
  const T* x = (const T*)a.x + n * a.V;
  float top = -kInf;
  if constexpr (COUNTED) {
    top = parts_top(a, n);
    for (int b = t; b < NB; b += NT) {
      s.mass[b] = a.mass[(long)n * NB + b];
      s.count[b] = a.count[(long)n * NB + b];
    }
  } else {
    for (int b = t; b < NB; b += NT) {
      s.mass[b] = 0;
      s.count[b] = 0;
    }
    scan<T, NT>(x, 0, a.V, [&](long, float v) { top = fmaxf(top, v); });
    top = wave_reduce_max(top);
    float* red = (float*)s.wave;
    if ((t & 63) == 0) red[t >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) top = fmaxf(top, red[i]);
    __syncthreads();
  }
  if (top == -kInf) {  // nothing can be drawn
    if (t == 0) {
      a.token[n] = -1;
      if (a.logp) a.logp[n] = __builtin_nanf("");
    }
    return;
  }
  const Row r = make_row(temperature(a, n), top);
  const int k = number_kept(a, n, r);
  if constexpr (!COUNTED)
    count_row<NT>(a, x, 0, a.V, r, k != 0, s.mass, s.count);
  __syncthreads();

  Held held = {-1, 0};
  u64 at = 0, keep, sum, v = 0;
  for (int b = t; b < NB; b += NT) v += s.mass[b];
  sum_before(v, s.wave[0], &keep);
  if (k && ask(a, x, r, Ask{Ask::kNumber, (double)k}, s, held, &at, &sum))
    keep = sum;
  const double p = a.pp ? (double)a.pp[n] : a.p;
  if (p < 1.0 &&
      ask(a, x, r, Ask{Ask::kWeight, fmax(p, 0.0) * (double)keep}, s, held,
          &at, &sum))
    keep = min(keep, sum);
  const double mp = a.mp ? (double)a.mp[n] : a.m;
  if (mp > 0.0 && !r.greedy) {
    const double most = fmax(-log(mp), 0.0);
    if (most * STEP < NB - 4) keep = min(keep, shallow(a, x, r, most, s));
  }
  const float u = fmaxf(fminf(a.u[n], 1.f - 0x1p-24f), 0.f);
  const bool got = ask(a, x, r, Ask{Ask::kOver, (double)u * (double)keep}, s,
                       held, &at, &sum);
  if (t == 0) {
    a.token[n] = got ? (int)(unsigned)at : -1;
    if (a.logp)
      a.logp[n] = !got ? __builtin_nanf("")
                       : (float)(-depth(entry_logit(at), r) -
                                 log(ldexp((double)keep, -a.sbits)));
  }
}

template <typename T>
void launch(const LaunchCtx& lc, const Sample& a) {
  if (a.parts == 1) {
    sample_kernel<T, false><<<a.N, NT, 0, lc.stream>>>(a);
    return;
  }
  sample_max_kernel<T><<<a.N * a.parts, 256, 0, lc.stream>>>(a);
  sample_count_kernel<T><<<a.N * a.parts, 256, 0, lc.stream>>>(a);
  sample_kernel<T, true><<<a.N, NT, 0, lc.stream>>>(a);
}

// Parts of a row: enough blocks for the chip, none with less than 4096
// logits; 1 where a block a row is enough
int parts_of(int64_t N, int64_t V) {
  if (V <= 32768 || N >= 192) return 1;
  return (int)std::max<int64_t>(1, std::min(1024 / std::max<int64_t>(N, 1),
                                            V / 4096));
}

}  // namespace

int64_t sample_tokens_workspace(int64_t N, int64_t V) {
  const int64_t parts = parts_of(N, V);
  return parts == 1 ? 0 : N * (NB * 12 + parts * 4);
}

void sample_tokens_raw(const LaunchCtx& lc, const Arr& logits, const Arr& u,
                       const Arr& temperature, const Arr& top_k,
                       const Arr& top_p, const Arr& min_p, double t,
                       int64_t k, double p, double m, const Arr& token,
                       const Arr& logp, const Arr& work) {
  MX_CHECK(logits.dim() == 2, "sample_tokens: logits must have two axes");
  const int64_t N = logits.size(0), V = logits.size(1);
  if (N == 0) return;
  MX_CHECK(V >= 1 && V <= (1 << 19) && N < (1 << 20),
           "sample_tokens: 1 to 2^19 logits a row, less than 2^20 rows");
  MX_CHECK(u.dtype == kFloat32 && u.numel() == N && token.dtype == kInt32 &&
               token.numel() == N,
           "sample_tokens: one float32 number and int32 token a row");
  MX_CHECK(!logp.defined() || (logp.dtype == kFloat32 && logp.numel() == N),
           "sample_tokens: one float32 log-probability a row");
  for (const Arr* x : {&temperature, &top_p, &min_p})
    MX_CHECK(!x->defined() || (x->dtype == kFloat32 && x->numel() == N),
             "sample_tokens: parameters are one number, or a float32 a row");
  MX_CHECK(!top_k.defined() || (top_k.dtype == kInt32 && top_k.numel() == N),
           "sample_tokens: top_k is one number, or an int32 a row");
  MX_CHECK((work.defined() ? work.numel() * (int64_t)dtype_size(work.dtype)
                           : 0) >= sample_tokens_workspace(N, V),
           "sample_tokens: workspace too small");
  Sample a = {};
  a.x = logits.ptr;
  a.V = V;
  a.N = (int)N;
  a.parts = parts_of(N, V);
  a.u = u.data<float>();
  a.tp = temperature.data<float>();
  a.pp = top_p.data<float>();
  a.mp = min_p.data<float>();
  a.kp = top_k.data<int>();
  a.t = t;
  a.p = p;
  a.m = m;
  a.k = (int)std::max<int64_t>(0, std::min<int64_t>(k, V));
  a.sbits = 62;
  while ((int64_t)1 << (62 - a.sbits) < V) --a.sbits;
  a.sbits = std::min(a.sbits, 51);
  a.token = token.data<int>();
  a.logp = logp.data<float>();
  a.mass = work.data<u64>();
  a.count = (unsigned*)(a.mass + N * NB);
  a.pmax = (float*)(a.count + N * NB);
  DISPATCH_FLOAT_NATIVE(logits.dtype, "sample_tokens",
                        [&] { launch<scalar_t>(lc, a); });
  HIP_CHECK_LAST();
}

}  // namespace mxcore
