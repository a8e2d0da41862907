// The next token of each row of logits, from given random numbers.
//
//   order: by logit, the largest first; the lower index first among equals
//   w_i = exp((x_i - max) / T)
//   kept: the first top_k of the order; of those the shortest prefix that
//         holds top_p of their sum; of those the ones with w_i >= min_p
//   token: the first in the order whose running sum exceeds u * (kept sum)
//
// Every step asks for a prefix of one order, so the row is never sorted: it is
// counted into 4096 buckets of the weight's logarithm, 1/64 octave wide (the
// weight of each, and for top_k the number), whose running sums answer every
// question up to one bucket or two.  One scan gathers the entries of all
// those buckets, and only they are sorted and looked at one by one.
//
// Weights are 64-bit: whether a token is kept or drawn lies next to a border.
// They are counted as whole numbers of 2^-s (s = 62 - ceil(log2 V), at most
// 51), so that sums cannot overflow and do not depend on the order in which
// lanes and blocks add.
//
// Bound by latency for few rows and by the 64-bit weights for many.  The
// logits are read from memory once and scanned again from the cache.  Rows
// that fill the chip, and short ones, take one launch with a block a row; else
// two launches cut each row into parts for the maximum and the counts, and a
// third answers.  Measured, with the phases in us:
//                     in all  maximum  counts  sums  scan  sort  answers
//   1 x 10000 fp32        15        2       2     3     2     2        2
//   32 x 30522 fp16       24        2       7     4     4     2        3
//   256 x 131072 bf16     63       10      25     4    15     6        3
// The counts are 19 vector instructions a logit, 13 of them 64-bit, and two
// accesses to LDS that take 22 cycles a wave; the maximum is bound by HBM.
#include "ops_api.h"

namespace mxcore {
namespace {

constexpr int NB = 4096;    // buckets
constexpr int STEP = 64;    // buckets for each halving of the weight
constexpr int LIST = 2048;  // entries that are sorted in LDS
constexpr int NT = 1024;    // threads of the block that answers for a row
constexpr float kInf = __builtin_huge_valf();
typedef unsigned long long u64;

struct Sample {
  const void* x;
  long V;
  int N, parts;
  const float* u;
  // one a row where the pointer is given, else the value
  const float *tp, *pp, *mp;
  const void* kp;  // int32 or (k64) int64
  bool k64;
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
  double top;    // the maximum; above all float32 where that is infinite
  double scale;  // buckets for each unit of logit
  double inv;    // 1 / T
  float ftop;
  bool greedy;
};

// f(index, 16 bytes of logits) and g(index, logit) over [i0, i1) by the
// block's threads, the first where the memory is aligned.  The next two loads
// are on their way while f looks at one (256 rows of 131072: 65 us to 64; at
// 32 of 30522, 24 us either way).
template <typename T, int THREADS, typename F, typename G>
DEV_INLINE void scan_vectors(const T* x, long i0, long i1, F f, G g) {
  constexpr int N = 16 / sizeof(T);
  using VecT = T __attribute__((ext_vector_type(N)));
  const long a =
      min(i1, i0 + (long)((-(uintptr_t)(x + i0) & 15) / sizeof(T)));
  const long nv = (i1 - a) / N;
  for (long i = i0 + threadIdx.x; i < a; i += THREADS) g(i, (float)x[i]);
  const VecT* p = (const VecT*)(x + a);
  long k = threadIdx.x;
  if (k < nv) {
    VecT v0 = p[k], v1 = p[min(k + THREADS, nv - 1)];
    for (; k < nv; k += THREADS) {
      const VecT v = v0;
      v0 = v1;
      v1 = p[min(k + 2 * THREADS, nv - 1)];
      f(a + k * N, v);
    }
  }
  for (long i = a + nv * N + threadIdx.x; i < i1; i += THREADS)
    g(i, (float)x[i]);
}

// f(index, logit) over [i0, i1)
template <typename T, int THREADS, typename F>
DEV_INLINE void scan(const T* x, long i0, long i1, F f) {
  scan_vectors<T, THREADS>(x, i0, i1, [&](long i, auto v) {
#pragma unroll
    for (int j = 0; j < (int)(16 / sizeof(T)); ++j) f(i + j, (float)v[j]);
  }, f);
}

// f(index, logit) for the few logits of the row that `some` picks: those of 16
// bytes are looked at without a branch, and then one by one
template <typename T, int THREADS, typename S, typename F>
DEV_INLINE void scan_some(const T* x, long n, S some, F f) {
  scan_vectors<T, THREADS>(x, 0, n, [&](long i, auto v) {
    unsigned m = 0;
#pragma unroll
    for (int j = 0; j < (int)(16 / sizeof(T)); ++j)
      m |= (unsigned)some((float)v[j]) << j;
    while (m) {
      const int j = __ffs(m) - 1;
      m &= m - 1;
      // the j-th of the vector, by its 32-bit words
      union {
        decltype(v) v;
        unsigned w[4];
      } u = {v};
      constexpr int P = 4 / sizeof(T);
      const int k = j / P;
      union {
        unsigned w;
        T t[P];
      } e = {k == 0 ? u.w[0] : k == 1 ? u.w[1] : k == 2 ? u.w[2] : u.w[3]};
      if (P == 2) e.w >>= 16 * (j & 1);
      f(i + j, (float)e.t[0]);
    }
  }, [&](long i, float v) {
    if (some(v)) f(i, v);
  });
}

// How far a logit lies below the maximum, in buckets: -64 log2 of its weight,
// at most the last one's number (which weighs nothing), also for -inf and NaN.
// Not increasing in v, so that buckets follow the order.
DEV_INLINE double depth(float v, const Row& r) {
  return fmax(fmin((r.top - (double)v) * r.scale, (double)(NB - 1)), 0.0);
}

// Adding 1.5 * 2^52 rounds a double to a whole number in its lowest bits
struct Whole {
  int n;
  double f;
};
DEV_INLINE Whole whole(double d) {
  const double t = d + 0x1.8p52;
  return {(int)__double2loint(t), t - 0x1.8p52};
}

DEV_INLINE int bucket(double d) { return whole(d).n; }

// 2^s 2^(-d / 64), rounded to a whole number.  d = n - f with |f| <= 1/2:
// 2^s 2^(-n / 64) comes from the table (0 for the last bucket, whose weights
// are less than half of one) and 2^(f / 64) from its Taylor series to the 5th
// power (off by 4e-17 at most: (ln(2) / 128)^6 / 720).  Adding 2^52 rounds it.
struct Weight {
  int b;  // the bucket
  u64 w;
};
DEV_INLINE Weight weight(double d, const double* table) {
  constexpr double c = 0.010830424696249145;  // ln(2) / 64
  const Whole n = whole(d);
  const double f = n.f - d;
  double e = c * c * c * c * c / 120;
  e = fma(e, f, c * c * c * c / 24);
  e = fma(e, f, c * c * c / 6);
  e = fma(e, f, c * c / 2);
  e = fma(e, f, c);
  e = fma(e, f, 1.0);
  return {n.n, (u64)__double_as_longlong(fma(e, table[n.n], 0x1p52)) -
                   0x4330000000000000ull};
}

// the table, by all threads of a block; `octave` has room for STEP values
template <int THREADS>
DEV_INLINE void fill_table(double* table, double* octave, int sbits) {
  if (threadIdx.x < STEP) octave[threadIdx.x] = exp2(threadIdx.x / -64.0);
  __syncthreads();
  for (int i = threadIdx.x; i < NB; i += THREADS)
    table[i] = i == NB - 1 ? 0.0
                           : octave[i % STEP] *
                                 __hiloint2double(
                                     (1023 + sbits - i / STEP) << 20, 0);
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
  if (!a.tp) return a.t;
  const double t = (double)a.tp[n];
  return t > 1e30 ? 1e30 : t;
}

DEV_INLINE Row make_row(double temp, float top) {
  Row r;
  r.greedy = !(temp > 0.0);
  // finite, so that the maximum itself lies no way below it, whatever T
  r.inv = r.greedy ? 1e300 : fmin(1.0 / temp, 1e300);
  r.scale = r.inv * (STEP * 1.4426950408889634);
  r.top = top == kInf ? 0x1p129 : (double)top;
  r.ftop = top;
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
                          const Row& r, bool number, const double* table,
                          u64* mass, unsigned* count) {
  // (nothing in the loop branches, so that the logits' chains of 64-bit
  // operations overlap)
  auto each = [&](auto numbers) {
    scan<T, THREADS>(x, i0, i1, [&](long, float v) {
      const Weight w = weight(depth(v, r), table);
      if (decltype(numbers)::value) atomicAdd(&count[w.b], 1u);
      atomicAdd(&mass[w.b], w.w);
    });
  };
  if (number) each(std::true_type{});
  else each(std::false_type{});
}

// how many the row may keep; 0: all.  The numbers are counted only for this
DEV_INLINE int number_kept(const Sample& a, int n, const Row& r) {
  const long k = r.greedy ? 1
                 : !a.kp  ? a.k
                 : a.k64  ? ((const long*)a.kp)[n]
                          : ((const int*)a.kp)[n];
  return k > 0 && k < a.V ? (int)k : 0;
}

template <typename T>
__global__ __launch_bounds__(512) void sample_count_kernel(Sample a) {
  __shared__ u64 mass[NB];
  __shared__ unsigned count[NB];
  __shared__ double table[NB];
  // (a place that is read as numbers only after the next barrier)
  fill_table<512>(table, (double*)count, a.sbits);
  __syncthreads();
  const int n = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
  for (int b = threadIdx.x; b < NB; b += 512) {
    mass[b] = 0;
    count[b] = 0;
  }
  const Row r = make_row(temperature(a, n), parts_top(a, n));
  __syncthreads();
  count_row<512>(a, (const T*)a.x + n * a.V, a.V * part / a.parts,
                 a.V * (part + 1) / a.parts, r, number_kept(a, n, r) != 0,
                 table, mass, count);
  __syncthreads();
  for (int b = threadIdx.x; b < NB; b += 512) {
    if (count[b]) atomicAdd(&a.count[(long)n * NB + b], count[b]);
    if (mass[b]) atomicAdd(&a.mass[(long)n * NB + b], mass[b]);
  }
}

// ---------------------------------------------------------------------------
// 3. the answers: a block a row
// ---------------------------------------------------------------------------
struct Lds {
  u64 mass[NB];  // running sums, once the row is counted
  unsigned count[NB];
  u64 list[LIST];
  // a bucket too full for the list
  u64 fine_mass[LIST];
  unsigned fine_count[LIST];
  double table[NB];
  u64 wave[NT / 64];
  float bound[8];
  unsigned n;
  // for each of the three questions
  struct Answer {
    u64 before;  // of the list, where the question's bucket begins: weight
    int first;   // and number
    int found;
    u64 at, through;
  } answer[3];
};

// v and what the lanes that CTRL (a DPP control) names hold, in the rows of
// 16 lanes that ROWS names
template <int CTRL, int ROWS>
DEV_INLINE u64 add_lanes(u64 v) {
  const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp(
      0, (int)(unsigned)v, CTRL, ROWS, 0xf, false);
  const unsigned hi = (unsigned)__builtin_amdgcn_update_dpp(
      0, (int)(unsigned)(v >> 32), CTRL, ROWS, 0xf, false);
  return v + ((u64)hi << 32 | lo);
}

// sum of the lanes up to this one
DEV_INLINE u64 sum_lanes(u64 v) {
  v = add_lanes<0x111, 0xf>(v);  // 1, 2, 4 and 8 lanes below, in the row
  v = add_lanes<0x112, 0xf>(v);
  v = add_lanes<0x114, 0xf>(v);
  v = add_lanes<0x118, 0xf>(v);
  v = add_lanes<0x142, 0xa>(v);  // the row below's last, for rows 1 and 3
  return add_lanes<0x143, 0xc>(v);  // lane 31, for rows 2 and 3
}

// running sum of the threads before this one; *total: of all
DEV_INLINE u64 sum_before(u64 v, u64* wave, u64* total) {
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6;
  const u64 in = sum_lanes(v);
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

// values to their running sums, N = NT * PER of them
template <int PER, typename V>
DEV_INLINE void run_sums(V* v, u64* wave) {
  u64 in[PER], sum = 0, all;
#pragma unroll
  for (int j = 0; j < PER; ++j) in[j] = sum += v[threadIdx.x * PER + j];
  const u64 before = sum_before(sum, wave, &all);
#pragma unroll
  for (int j = 0; j < PER; ++j)
    v[threadIdx.x * PER + j] = (V)(before + in[j]);
  __syncthreads();
}

// a question to the order: its first entry ...
struct Ask {
  enum Kind {
    kNumber,  // ... whose running number is at least want
    kWeight,  // ... whose running weight is at least want
    kOver,    // ... whose running weight is over want
  } kind;
  double want;
  int index;  // which of the answers is its own
};

DEV_INLINE bool reached(const Ask& q, u64 through) {
  return q.kind == Ask::kOver ? (double)through > q.want
                              : (double)through >= q.want;
}

// First of n running sums (behind `base`) with which the question is reached,
// n if none: each lane looks at one of 64 places, twice.  Every wave does the
// same search.
template <typename V>
DEV_INLINE int find(const Ask& q, const V* sums, int n, u64 base = 0) {
  const int l = threadIdx.x & 63, step = n / 64;
  u64 hit = __ballot(reached(q, base + sums[(l + 1) * step - 1]));
  if (!hit) return n;
  const int at = (__ffsll((long long)hit) - 1) * step;
  hit = __ballot(l < step && reached(q, base + sums[at + min(l, step - 1)]));
  return at + __ffsll((long long)hit) - 1;
}

DEV_INLINE int find_bucket(const Ask& q, const Lds& s) {
  return q.kind == Ask::kNumber ? find(q, s.count, NB) : find(q, s.mass, NB);
}

template <typename V>
DEV_INLINE u64 before(const V* sums, int b) { return b ? sums[b - 1] : 0; }

// Float32 and whole numbers in the same order
DEV_INLINE unsigned rank(float v) {
  const unsigned u = __float_as_uint(v);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
DEV_INLINE float of_rank(unsigned k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// The rank of the least logit whose bucket is at most b, by a search in which
// each lane looks at one of 64 places
DEV_INLINE unsigned least_rank(int b, const Row& r) {
  // the bucket is over b at lo and at most b at hi
  unsigned lo = rank(-kInf), hi = rank(r.ftop);
  while (hi - lo > 1) {
    const unsigned step = (hi - lo + 63) / 64;
    const unsigned at = min(lo + step * ((threadIdx.x & 63) + 1), hi);
    const int first = __ffsll((long long)__ballot(
                          bucket(depth(of_rank(at), r)) <= b)) - 1;
    hi = min(lo + step * (first + 1), hi);
    lo += step * first;
  }
  return hi;
}

// Buckets follow the order, so buckets (0 to NB - 2) are ranges of logits, and
// a scan needs two comparisons for each: from low_end on, up to high_end
DEV_INLINE float low_end(int b, const Row& r) {
  return of_rank(least_rank(b, r));
}
DEV_INLINE float high_end(int b, const Row& r) {
  return b == 0 ? kInf : of_rank(least_rank(b - 1, r) - 1);
}

// The list in order: a pair of entries to a thread.  A wave's pairs lie in
// 128 places of its own while they are at most 64 apart, so only wider steps
// wait for the other waves.
DEV_INLINE void sort_list(Lds& s, int n) {
  int size = 2;
  while (size < n) size <<= 1;
  for (int i = n + threadIdx.x; i < size; i += NT) s.list[i] = ~0ull;
  __syncthreads();
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

// What the list holds, in order: n entries, those of the buckets lo[i] to
// hi[i] (none where lo > hi) among them all; and this thread's two of them
struct Held {
  int lo[3], hi[3];
  int n;
  int b[2];      // their buckets (NB: no entry),
  int before;    // that of the one before them (-1: none)
  u64 w[2], sum; // weights, and the list's running sum before them
};

DEV_INLINE void weigh_list(Lds& s, const Row& r, Held* held) {
  const int i0 = threadIdx.x * 2;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    held->b[j] = NB;
    held->w[j] = 0;
    if (i0 + j < held->n) {
      const Weight e = weight(depth(entry_logit(s.list[i0 + j]), r), s.table);
      held->b[j] = e.b;
      held->w[j] = e.w;
    }
  }
  held->before = i0 > 0 && i0 < held->n
                     ? bucket(depth(entry_logit(s.list[i0 - 1]), r)) : -1;
  u64 all;
  held->sum = sum_before(held->w[0] + held->w[1], s.wave, &all);
}

// Brings the one bucket b to the list; where that cannot hold it (many equal
// logits), the part of it in which the question is reached, and *weight0 and
// *number0 then lie before that part.
template <typename T>
DEV_INLINE void gather(const Sample& a, const T* x, const Row& r, const Ask& q,
                       int b, Lds& s, Held* held, u64* weight0,
                       u64* number0) {
  const float vlo = low_end(b, r), vhi = high_end(b, r);
  // entries of the bucket between lo and hi, both included
  auto each = [&](u64 lo, u64 hi, auto f) {
    scan_some<T, NT>(
        x, a.V, [&](float v) { return (v >= vlo) & (v <= vhi); },
        [&](long i, float v) {
          const u64 e = entry(v, i);
          if (e >= lo && e <= hi) f(v, e);
        });
  };
  u64 lo = 0, hi = ~0ull;
  bool whole_bucket = true;
  for (;;) {
    __syncthreads();
    if (threadIdx.x == 0) s.n = 0;
    __syncthreads();
    each(lo, hi, [&](float, u64 e) {
      const unsigned k = atomicAdd(&s.n, 1u);
      if (k < LIST) s.list[k] = e;
    });
    __syncthreads();
    if (s.n <= LIST) break;
    // divide it by the entries' own bits: by 2^10 or more each time
    whole_bucket = false;
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
      s.list[threadIdx.x >> 6] = least;
      s.wave[threadIdx.x >> 6] = most;
    }
    for (int i = threadIdx.x; i < LIST; i += NT) {
      s.fine_mass[i] = 0;
      s.fine_count[i] = 0;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) {
      least = min(least, s.list[i]);
      most = max(most, s.wave[i]);
    }
    __syncthreads();
    // more than LIST = 2^11 different entries: most - least has 12 bits or
    // 11 of them set, and its 11 highest number the parts
    const int shift = 53 - (int)__clzll((long long)(most - least));
    each(least, most, [&](float v, u64 e) {
      const int k = (int)((e - least) >> shift);
      atomicAdd(&s.fine_count[k], 1u);
      const u64 w = weight(depth(v, r), s.table).w;
      if (w) atomicAdd(&s.fine_mass[k], w);
    });
    __syncthreads();
    run_sums<LIST / NT>(s.fine_mass, s.wave);
    run_sums<LIST / NT>(s.fine_count, s.wave);
    // (the parts' sums are the bucket's, with which the question is reached)
    const int k = min(LIST - 1, q.kind == Ask::kNumber
                                    ? find(q, s.fine_count, LIST, *number0)
                                    : find(q, s.fine_mass, LIST, *weight0));
    *weight0 += before(s.fine_mass, k);
    *number0 += before(s.fine_count, k);
    lo = least + ((u64)k << shift);
    hi = min(most, lo + ((1ull << shift) - 1));
  }
  *held = Held{{whole_bucket ? b : 0, 0, 0}, {whole_bucket ? b : -1, -1, -1},
               (int)s.n};
  sort_list(s, held->n);
  weigh_list(s, r, held);
}

// The question's entry, and the weight through it.  False where it lies in the
// last bucket or nowhere: the weights there add up to less than 2^-24 of the
// row's, so no random number below 1 draws them.
template <typename T>
DEV_INLINE bool ask(const Sample& a, const T* x, const Row& r, const Ask& q,
                    Lds& s, Held* held, u64* at, u64* through) {
  const int b = find_bucket(q, s);
  if (b >= NB - 1) return false;
  u64 weight0 = before(s.mass, b), number0 = 0;
  const bool number = q.kind == Ask::kNumber;
  if (number) number0 = before(s.count, b);
  bool have = false;
#pragma unroll
  for (int i = 0; i < 3; ++i) have |= held->lo[i] <= b && b <= held->hi[i];
  if (!have) gather(a, x, r, q, b, s, held, &weight0, &number0);
  // the bucket's entries follow each other: the first tells where they begin
  Lds::Answer& mine = s.answer[q.index];
  const int i0 = threadIdx.x * 2;
  const bool first[2] = {held->b[0] == b && held->before != b,
                         held->b[1] == b && held->b[0] != b};
  if (first[0] || first[1]) {
    mine.before = held->sum + (first[1] ? held->w[0] : 0);
    mine.first = i0 + first[1];
  }
  __syncthreads();
  // running number and weight before each entry: one entry is the first with
  // which the question is reached
  u64 k = number0 + (i0 - mine.first), m = weight0 + held->sum - mine.before;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const u64 k1 = k + 1, m1 = m + held->w[j];
    if (held->b[j] == b && reached(q, number ? k1 : m1) &&
        (first[j] || !reached(q, number ? k : m))) {
      mine.at = s.list[i0 + j];
      mine.through = m1;
      mine.found = 1;
    }
    k = k1;
    m = m1;
  }
  __syncthreads();
  *at = mine.at;
  *through = mine.through;
  return mine.found;
}

template <typename T, bool COUNTED>
__global__ __launch_bounds__(NT) void sample_kernel(Sample a) {
  __shared__ Lds s;
  const int n = blockIdx.x, t = threadIdx.x;
  const T* x = (const T*)a.x + n * a.V;
  float top = -kInf;
  if (t < 3) s.answer[t].found = s.answer[t].first = 0;
  fill_table<NT>(s.table, (double*)s.list, a.sbits);
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
    count_row<NT>(a, x, 0, a.V, r, k != 0, s.table, s.mass, s.count);
  __syncthreads();
  run_sums<NB / NT>(s.mass, s.wave);
  if (k) run_sums<NB / NT>(s.count, s.wave);

  // The kept weight lies between keep0 and keep1, as far as whole buckets
  // say, and so do the buckets of each later question
  const double p = a.pp ? (double)a.pp[n] : a.p;
  const double mp = a.mp ? (double)a.mp[n] : a.m;
  const float u = fmaxf(fminf(a.u[n], 1.f - 0x1p-24f), 0.f);
  u64 keep = s.mass[NB - 1], keep0 = keep, keep1 = keep;
  Held held = {{0, 0, 0}, {-1, -1, -1}, 0};
  const Ask ask_k = {Ask::kNumber, (double)k, 0};
  if (k) {
    const int b = find_bucket(ask_k, s);
    if (b < NB - 1) {
      held.lo[0] = held.hi[0] = b;
      keep0 = before(s.mass, b);
      keep1 = s.mass[b];
    }
  }
  const double want_p = fmax(p, 0.0);
  if (p < 1.0) {
    const int b0 = find_bucket(Ask{Ask::kWeight, want_p * (double)keep0, 1}, s),
              b1 = find_bucket(Ask{Ask::kWeight, want_p * (double)keep1, 1}, s);
    held.lo[1] = b0;
    held.hi[1] = min(b1, NB - 2);
    keep0 = min(keep0, before(s.mass, b0));
    if (b1 < NB) keep1 = min(keep1, s.mass[b1]);
  }
  // min_p: whole buckets, and of one the entries that are not too deep
  const double most = mp > 0.0 ? fmax(-log2(mp) * STEP, 0.0) : 1e9;
  const bool limit = most < NB - 2 && !r.greedy;
  const int bm = limit ? bucket(most) : NB;
  if (limit) {
    keep0 = min(keep0, before(s.mass, bm));
    keep1 = min(keep1, s.mass[bm]);
  }
  held.lo[2] = find_bucket(Ask{Ask::kOver, (double)u * (double)keep0, 2}, s);
  held.hi[2] = min(
      find_bucket(Ask{Ask::kOver, (double)u * (double)keep1, 2}, s), NB - 2);

  // one scan for them all: a wave finds each end of each range
  if (t < 8 * 64) {
    const int i = t >> 7, end = t >> 6 & 1;
    const int lo = i == 0   ? held.lo[0]
                   : i == 1 ? held.lo[1]
                   : i == 2 ? held.lo[2]
                            : bm;
    const int hi = i == 0   ? held.hi[0]
                   : i == 1 ? held.hi[1]
                   : i == 2 ? held.hi[2]
                            : (limit ? bm : -1);
    const float v = lo > hi ? __builtin_nanf("")  // no range: holds nothing
                    : end   ? high_end(lo, r)
                            : low_end(hi, r);
    if ((t & 63) == 0) s.bound[t >> 6] = v;
  }
  if (t == 0) s.n = 0;
  __syncthreads();
  // a range holds what lies within half its width of its middle; the widest
  // range's half width, a little rounded up, lets all of them through and
  // little else
  float vb[8], mid[4], half = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    vb[2 * i] = s.bound[2 * i];
    vb[2 * i + 1] = fminf(s.bound[2 * i + 1], top);
    mid[i] = 0.5f * vb[2 * i] + 0.5f * vb[2 * i + 1];
    half = fmaxf(half, fmaxf(vb[2 * i + 1] - mid[i], mid[i] - vb[2 * i]) *
                           1.0001f + fabsf(mid[i]) * 1e-6f);
  }
  if (top == kInf || !(half < kInf)) {  // no middle of infinite ends
    half = kInf;
    mid[0] = 0.f;
  }
  u64 part = 0;
  scan_some<T, NT>(
      x, a.V,
      [&](float v) {
        return fminf(fminf(fabsf(v - mid[0]), fabsf(v - mid[1])),
                     fminf(fabsf(v - mid[2]), fabsf(v - mid[3]))) <= half;
      },
      [&](long i, float v) {
        if ((v >= vb[0] && v <= vb[1]) || (v >= vb[2] && v <= vb[3]) ||
            (v >= vb[4] && v <= vb[5])) {
          const unsigned at = atomicAdd(&s.n, 1u);
          if (at < LIST) s.list[at] = entry(v, i);
        }
        if (v >= vb[6] && v <= vb[7]) {
          const double d = depth(v, r);
          if (d <= most) part += weight(d, s.table).w;
        }
      });
  __syncthreads();
  held.n = (int)s.n;
  if (held.n <= LIST) {
    sort_list(s, held.n);
    weigh_list(s, r, &held);
  } else {  // too many: each question brings its own
    held = Held{{0, 0, 0}, {-1, -1, -1}, 0};
  }

  u64 at = 0, sum;
  if (k && ask(a, x, r, ask_k, s, &held, &at, &sum)) keep = sum;
  if (p < 1.0 && ask(a, x, r, Ask{Ask::kWeight, want_p * (double)keep, 1},
                     s, &held, &at, &sum))
    keep = min(keep, sum);
  if (limit) {
    sum_before(part, s.wave, &sum);
    keep = min(keep, before(s.mass, bm) + sum);
  }
  const bool got = ask(a, x, r, Ask{Ask::kOver, (double)u * (double)keep, 2},
                       s, &held, &at, &sum);
  if (t == 0) {
    a.token[n] = got ? (int)(unsigned)at : -1;
    if (a.logp) {
      const float v = entry_logit(at);
      const double d = v == top ? 0.0 : ((double)top - (double)v) * r.inv;
      a.logp[n] = !got ? __builtin_nanf("")
                       : (float)(-d - log(ldexp((double)keep, -a.sbits)));
    }
  }
}

template <typename T>
void launch(const LaunchCtx& lc, const Sample& a) {
  if (a.parts == 1) {
    sample_kernel<T, false><<<a.N, NT, 0, lc.stream>>>(a);
    return;
  }
  sample_max_kernel<T><<<a.N * a.parts, 256, 0, lc.stream>>>(a);
  sample_count_kernel<T><<<a.N * a.parts, 512, 0, lc.stream>>>(a);
  sample_kernel<T, true><<<a.N, NT, 0, lc.stream>>>(a);
}

// Parts of a row: enough blocks for the chip, none with less than 4096
// logits; 1, and one launch, where the rows are short or many.  In us, one
// launch against three, bf16:
//   V = 65536:  1 row 34, 31      8 rows 34, 34     32 rows 36, 42
//   V = 131072: 1 row 51, 39     64 rows 56, 52    128 rows 57, 61
//   V = 262144: 1 row 88, 56     64 rows 98, 79    128 rows 104, 95
int parts_of(int64_t N, int64_t V) {
  if (V - 1024 * N < 56 << 10) return 1;
  return (int)std::max<int64_t>(1, std::min(512 / std::max<int64_t>(N, 1),
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
  MX_CHECK(!top_k.defined() ||
               ((top_k.dtype == kInt32 || top_k.dtype == kInt64) &&
                top_k.numel() == N),
           "sample_tokens: top_k is one number, or an int32 or int64 a row");
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
  a.kp = top_k.ptr;
  a.k64 = top_k.dtype == kInt64;
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
