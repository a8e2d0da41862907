// Attention of a decoder over an encoder's states of another length.
//
//   S = Q K^T / sqrt(d),  P = softmax over the kept keys,  O = P V
//   (a row without a key: zeros)
//   dV = P^T dO,  dP = dO V^T,  D = sum_d dO * O,  dS = P * (dP - D)
//   dQ = dS K / sqrt(d),  dK = dS^T Q / sqrt(d)
//
// The scores are never stored: one pass over the keys with the running
// maximum and sum of the softmax, and the backward computes P again from the
// row's log-sum, which the forward stores.  Query heads that share a key head
// are rows of one matrix (row m = g * Sq + s for the g-th of them), so shared
// keys are read once and their gradient is summed in the accumulators.
//
// Products run on the matrix cores with 32-bit accumulators, 32x32 tiles:
// lane l (h = l / 32) holds of A row l % 32 and of B column l % 32, elements
// k = 8 h + j; of C column l % 32, and in register i row
// 8 (i / 4) + 4 h + i % 4.  The forward computes S transposed (keys by
// queries): a query's scores lie in one lane pair's registers, the softmax
// needs one exchange between the two, and the registers ARE the B operand of
// the next product when its 16 keys are taken in the order
// {4h..4h+3, 8+4h..8+4h+3}; V's fragment is read in that order by the
// transposing LDS load.  dQ does the same with dS; dK and dV use S untransposed,
// whose registers are the A operand of P^T dO and dS^T Q.
//
// fp32 uses the fp32 matrix instructions (eight of k = 2 for one of k = 16).
//
// Measured at 4x16 heads, 1024 over 2048 keys, all of them kept, kernels back
// to back, medians, bf16 (and backward in fp16, which scales P and dS):
//   head size 64:   forward 57 us (600 TFLOP/s), backward 147 us (580; 156)
//   head size 96:   forward 79 us (650), backward 233 us (550; 257)
//   head size 128:  forward 88 us (780), backward 393 us (440; 385)
// and in fp32 at 2x16 heads, 1024 over 1024 keys of 64: 82 us (105), 272 us
// (79).  A large library product reaches 1198 in bf16, 154 in fp32.  As
// scheduled here, what surrounds the products takes longest: a wave spends 980
// cycles of vector instructions (32 exponentials of eight cycles, scaling,
// sums, rounding) beside 517 of matrix instructions on 64 keys by 32 rows of
// size 64; a wave's products hide about half of another's vector work, and the
// waves of a block pass these phases together.  Single tokens are bound by HBM.
//
// Roundings to 16 bits, besides the results': the weights P and dS when they
// become operands (half a step of each, as the inputs have), and the output O
// that the backward reads for dO . O (half a step of it, times dO).  Maxima,
// sums, O, dQ, dK, dV and the split's partial results are 32 bits.
//
// fp16 holds no more than 2^-14 to 2^16 in full, and P and dS are smaller than
// that in long rows and under small gradients.  So there the backward takes
// them times 2^shift, and the factor out of the sums: 15, which P of at most 1
// allows, as long as dS allows it too.  dQ looks at each tile's largest dS and
// lowers its row's shift where it has to; dK and dV, whose sums go over rows,
// take the lowest of their rows' shifts, which dQ leaves in the workspace.
// (Of 1024 over 2048 keys of 64, dK was off by 23% under dO of 1e-5, where its
// own rounding is 7%, and by 2.7% under 1e-4.)
#include "ops_api.h"

namespace mxcore {
namespace {

typedef short trs4_t __attribute__((ext_vector_type(4)));
typedef float float8_t __attribute__((ext_vector_type(8)));

constexpr float kNegInf = -__builtin_huge_valf();
constexpr float kLog2e = 1.4426950408889634f;

template <typename T> struct Mat;
template <> struct Mat<_Float16> {
  using Frag = half8_t;
  static DEV_INLINE float16_t mma(Frag a, Frag b, float16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};
template <> struct Mat<__bf16> {
  using Frag = bf168_t;
  static DEV_INLINE float16_t mma(Frag a, Frag b, float16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
template <> struct Mat<float> {
  using Frag = float8_t;
  static DEV_INLINE float16_t mma(Frag a, Frag b, float16_t c) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
    return c;
  }
};

// whether P and dS go times a power of two (see above)
template <typename T>
constexpr bool kShifted = std::is_same<T, _Float16>::value;
constexpr float kMostDs = 0x1p15f;  // half of what fp16 holds
// The shift goes into a row's log-sum, where that is small enough to take it
// (and at 2^20, what float32 loses of a log-sum makes weights 4% wrong anyway);
// a row's first shift
constexpr float kMostLse = 0x1p20f;
DEV_INLINE int first_shift(float lse) { return fabsf(lse) < kMostLse ? 15 : 0; }

// Waves a SIMD: two where the `n` operands of a row take at most `most` bytes,
// so that a wave's 256 registers hold them and their accumulators; else one.
// The second hides most of the first's latencies: dK and dV of size 96 in 16
// bits are faster with two, of which 12 registers (14 in fp16) lie in scratch
// memory, than with one (backward of 4x16 heads, 1024 over 2048 keys in bf16:
// 236 us, 332); of size 128, where 59 would, with one (412 us, 527).
template <typename T, int DP>
constexpr int waves(int n, int most = 256) {
  return n * DP * (int)sizeof(T) <= most ? 2 : 1;
}

// one [B, S, heads, D] view: strides in elements, D contiguous
struct View {
  void* p;
  long sb, ss, sh;
};

struct Att {
  View q, k, v, o, dout, dq, dk, dv;
  const void* len;       // [B] int32 or (len64) int64, or null
  const uint8_t* mask;   // [B, Sk], 0: masked, or null
  float* lse;            // [B, H, Sq] log2 of the row's sum, +inf: no key
  float* delta;          // [B, H, Sq]
  int* shift;            // [B, Hk][splits of dQ][G, Sq], fp16 only
  int dq_splits;
  float* part;           // partial results of a split, fp32
  int B, H, Hk, G, Sq, Sk, D;
  int nsplit;
  int vec;               // 16-byte accesses
  bool len64;
  float scale;           // 1 / sqrt(D)
  float inv_sq;          // 1 / Sq
};

// ---------------------------------------------------------------------------
// LDS tiles [rows][DP] in 16-byte chunks (rows of 96 lie as those of 128, whose
// last quarter nobody reads).  The chunk's place in its row is
// XORed with a function of the row, chosen so that both readers are free of
// bank conflicts: 16 rows at one chunk (row fragments), and 4 rows at 4
// neighbouring chunks (the transposing read).
// ---------------------------------------------------------------------------
template <typename T, int DP>
struct Tile {
  static constexpr int EPC = 16 / sizeof(T);  // elements a chunk
  static constexpr int WIDE = DP == 96 ? 128 : DP;
  static constexpr int CPR = WIDE / EPC;      // chunks a row
  static constexpr int RB = WIDE * (int)sizeof(T);
  static DEV_INLINE int swz(int row) {
    if constexpr (RB == 64) return (row >> 2) & 3;
    if constexpr (RB == 128) return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
    return ((row & 3) << 2) | ((row >> 2) & 3);
  }
  // byte offset of a chunk
  static DEV_INLINE int at(int row, int chunk) {
    return row * RB + ((chunk ^ swz(row)) << 4);
  }
  // elements d = 16 ks + 8 h + j of one row
  static DEV_INLINE typename Mat<T>::Frag row_frag(const char* t, int row,
                                                   int ks, int h) {
    typename Mat<T>::Frag f;
    if constexpr (sizeof(T) == 2) {
      f = *(const typename Mat<T>::Frag*)(t + at(row, ks * 2 + h));
    } else {
      const float4_t a = *(const float4_t*)(t + at(row, ks * 4 + h * 2));
      const float4_t b = *(const float4_t*)(t + at(row, ks * 4 + h * 2 + 1));
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        f[j] = a[j];
        f[4 + j] = b[j];
      }
    }
    return f;
  }
  // column c0 + l % 32, rows k0 + {4h..4h+3, 8+4h..8+4h+3}
  static DEV_INLINE typename Mat<T>::Frag col_frag(const char* t, int k0,
                                                   int c0, int l) {
    typename Mat<T>::Frag f;
    const int h = l >> 5;
    if constexpr (sizeof(T) == 2) {
      // 16 lanes read four rows of 16 columns and get one column each
      const int row = k0 + 4 * h + ((l & 15) >> 2);
      const int col = c0 + ((l >> 4) & 1) * 16 + (l & 3) * 4;
      const int sub = (col & 4) * 2;  // which half of the chunk, in bytes
      union {
        trs4_t s[2];
        typename Mat<T>::Frag f;
      } u;
      u.s[0] = tr(t + at(row, col >> 3) + sub);
      u.s[1] = tr(t + at(row + 8, col >> 3) + sub);
      f = u.f;
    } else {
      const int col = c0 + (l & 31);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int row = k0 + 4 * h + (j & 3) + (j >> 2) * 8;
        f[j] = *(const float*)(t + at(row, col >> 2) + (col & 3) * 4);
      }
    }
    return f;
  }
  static DEV_INLINE trs4_t tr(const char* p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) trs4_t*)(uintptr_t)p);
  }
};

// 16 bytes of a row from element d on; zeros from D on
template <typename T>
DEV_INLINE int4_t load_chunk(const T* row, int d, int D, bool vec) {
  int4_t r = {0, 0, 0, 0};
  if (vec) {
    if (d < D) r = *(const int4_t*)(row + d);
  } else {
    constexpr int N = 16 / sizeof(T);
    union {
      T e[N];
      int4_t v;
    } u;
    u.v = r;
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (d + j < D) u.e[j] = row[d + j];
    r = u.v;
  }
  return r;
}

// fragment elements d = 16 ks + 8 h + j straight from a row in memory
template <typename T>
DEV_INLINE typename Mat<T>::Frag load_frag(const T* row, int ks, int h, int D,
                                           bool vec, bool valid) {
  union {
    int4_t c[sizeof(T) / 2];
    typename Mat<T>::Frag f;
  } u;
  constexpr int N = 16 / sizeof(T);
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
    u.c[i] = int4_t{0, 0, 0, 0};
    if (valid) u.c[i] = load_chunk<T>(row, ks * 16 + h * 8 + i * N, D, vec);
  }
  return u.f;
}

// the fragment of accumulator registers r0..r0+7, rounded to the type
template <typename T>
DEV_INLINE typename Mat<T>::Frag pack(const float16_t& a, int r0) {
  typename Mat<T>::Frag f;
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = (T)a[r0 + j];
  return f;
}

template <typename T>
DEV_INLINE const T* row_ptr(const View& v, long b, int head, int s) {
  return (const T*)v.p + b * v.sb + s * v.ss + head * v.sh;
}

// row m of the G * Sq rows that share a key head
template <typename T>
DEV_INLINE T* q_row(const View& v, const Att& a, long b, int hk, int m) {
  // m / Sq by the reciprocal, at most one off
  int g = (int)((float)m * a.inv_sq), s = m - g * a.Sq;
  if (s < 0) {
    --g;
    s += a.Sq;
  } else if (s >= a.Sq) {
    ++g;
    s -= a.Sq;
  }
  return (T*)row_ptr<T>(v, b, hk * a.G + g, s);
}

// the value of the lane 32 away, and this lane's: their maximum and sum
DEV_INLINE float pair_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(
      __float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
DEV_INLINE float pair_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(
      __float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

DEV_INLINE int kept_keys(const Att& a, int b) {
  if (!a.len) return a.Sk;
  const long n = a.len64 ? ((const long*)a.len)[b] : ((const int*)a.len)[b];
  return (int)min((long)a.Sk, max(0L, n));
}

// The sequence and key head of the i-th of B * Hk.  Neighbours are sequences,
// not heads, the longest first, and the shortest first in every second head:
// so each chiplet has work of every length, a CU's two blocks are a long and a
// short one where all blocks run at once, and where they do not the short ones
// come last.  A wave sorts up to 64 lengths by counting.
DEV_INLINE void seq_head(const Att& a, int i, int* b, int* hk) {
  *hk = i / a.B;
  int k = i - *hk * a.B;
  if (*hk & 1) k = a.B - 1 - k;
  *b = k;
  if (!a.len || a.B > 64) return;
  const int l = threadIdx.x & 63;
  const int n = l < a.B ? kept_keys(a, l) : -1;
  int place = 0;
  for (int j = 0; j < a.B; ++j) {
    const int m = __builtin_amdgcn_readlane(n, j);
    place += m > n || (m == n && j < l);
  }
  *b = __ffsll((long long)__ballot(l < a.B && place == k)) - 1;
}

// ---------------------------------------------------------------------------
// staging: NT threads bring ROWS rows of DP elements to registers, then LDS.
// Every load is done, from a row that exists, and what is not wanted (a row
// past the end, a masked key, columns from D on) becomes zeros on its way to
// LDS: loads under a condition would be waited for where the branch ends, and
// a NaN in a masked key's memory meets no product.  Most tiles are whole, and
// their rows lie at one distance: those need no arithmetic at all, a scalar
// base for each load and one offset a thread.
// ---------------------------------------------------------------------------
template <typename T, int DP, int ROWS, int NT>
struct Stage {
  using TL = Tile<T, DP>;
  static constexpr int N = ROWS * TL::CPR / NT;
  static constexpr int STEP = NT / TL::CPR;  // rows between a thread's chunks
  static_assert(ROWS * TL::CPR % NT == 0 && NT % TL::CPR == 0,
                "whole chunks and rows");
  int4_t r[N];
  unsigned want;  // a bit a chunk
  // the thread's offset in bytes, for rows `ss` elements apart
  static DEV_INLINE unsigned offset(int t, long ss, int D) {
    const int d = t % TL::CPR * TL::EPC;
    return (unsigned)((t / TL::CPR * ss + (d < D ? d : 0)) * sizeof(T));
  }
  // all rows from `base` on; `once`: nobody reads them again
  template <bool once = false>
  DEV_INLINE void load(const T* base, long ss, unsigned off, int t, int D) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int4_t* p =
          (const int4_t*)((const char*)(base + i * STEP * ss) + off);
      r[i] = once ? __builtin_nontemporal_load(p) : *p;
    }
    want = t % TL::CPR * TL::EPC < D ? ~0u : 0;
  }
  // ptr(i): the i-th row, or another that exists; ok(i): whether it is wanted
  template <typename P, typename K>
  DEV_INLINE void load(P ptr, K ok, int t, int D, bool vec) {
    want = 0;
    if (vec) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int row = i * STEP + t / TL::CPR, d = t % TL::CPR * TL::EPC;
        r[i] = *(const int4_t*)(ptr(row) + (d < D ? d : 0));
        if (d < D && ok(row)) want |= 1u << i;
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int row = i * STEP + t / TL::CPR;
        r[i] = load_chunk<T>(ptr(row), t % TL::CPR * TL::EPC, D, false);
        if (ok(row)) want |= 1u << i;
      }
    }
  }
  // `all`: every chunk is wanted
  DEV_INLINE void store(char* tile, int t, bool all) const {
    if (all) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        *(int4_t*)(tile + TL::at(i * STEP + t / TL::CPR, t % TL::CPR)) = r[i];
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int4_t zero = {0, 0, 0, 0};
        *(int4_t*)(tile + TL::at(i * STEP + t / TL::CPR, t % TL::CPR)) =
            want >> i & 1 ? r[i] : zero;
      }
    }
  }
};

// the keys and values of one tile; `n` keys are kept (n >= 1), of those the
// ones whose mask is not 0
template <typename T, int DP, int BN, int NT, bool once = false>
struct KeyTiles {
  using S = Stage<T, DP, BN, NT>;
  S k, v;
  const T *kb, *vb;
  long ks, vs;
  const uint8_t* mask;
  int n, D, t;
  unsigned ko, vo;
  bool vec;
  DEV_INLINE KeyTiles(const Att& a, int b, int hk, int kept, int thread)
      : kb(row_ptr<T>(a.k, b, hk, 0)), vb(row_ptr<T>(a.v, b, hk, 0)),
        ks(a.k.ss), vs(a.v.ss),
        mask(a.mask ? a.mask + (long)b * a.Sk : nullptr), n(kept), D(a.D),
        t(thread), ko(S::offset(thread, a.k.ss, a.D)),
        vo(S::offset(thread, a.v.ss, a.D)), vec(a.vec) {}
  DEV_INLINE bool ok(int key) const {
    return key < n && (!mask || mask[min(key, n - 1)]);
  }
  // whether a tile has keys that are left out
  DEV_INLINE bool partial(int tile) const {
    return mask || (tile + 1) * BN > n;
  }
  DEV_INLINE void load(int tile) {
    const int k0 = tile * BN;
    if (vec && !partial(tile)) {
      k.template load<once>(kb + k0 * ks, ks, ko, t, D);
      v.template load<once>(vb + k0 * vs, vs, vo, t, D);
      return;
    }
    auto good = [&](int r) { return ok(k0 + r); };
    k.load([&](int r) { return kb + min(k0 + r, n - 1) * ks; }, good, t, D,
           vec);
    v.load([&](int r) { return vb + min(k0 + r, n - 1) * vs; }, good, t, D,
           vec);
  }
  DEV_INLINE void store(char* lk, char* lv, uint8_t* keep, int tile) const {
    const bool all = D == DP && !partial(tile);
    k.store(lk, t, all);
    v.store(lv, t, all);
    if (partial(tile))
      for (int r = t; r < BN; r += NT) keep[r] = ok(tile * BN + r);
  }
};

// f(0), f(1), ... for i in [t0, t1), with the buffer's number as a constant:
// addresses in LDS then differ by constants only
template <typename F>
DEV_INLINE void in_turn(int t0, int t1, F f) {
  for (int i = t0; i < t1; i += 2) {
    f(i, std::integral_constant<int, 0>{});
    if (i + 1 < t1) f(i + 1, std::integral_constant<int, 1>{});
  }
}

// O^T (or dQ^T) accumulators of one row per lane pair to memory
template <typename T, int DP>
DEV_INLINE void store_row(T* row, const float16_t (&acc)[DP / 32], float f,
                          int h, int D, bool vec) {
  using V4 = T __attribute__((ext_vector_type(4)));
#pragma unroll
  for (int n = 0; n < DP / 32; ++n)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const int d = n * 32 + 2 * i + 4 * h;
      if (vec) {
        if (d < D) {
          V4 o;
#pragma unroll
          for (int j = 0; j < 4; ++j) o[j] = (T)(acc[n][i + j] * f);
          *(V4*)(row + d) = o;
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (d + j < D) row[d + j] = (T)(acc[n][i + j] * f);
      }
    }
}

template <int DP>
DEV_INLINE void store_part(float* row, const float16_t (&acc)[DP / 32],
                           int h) {
#pragma unroll
  for (int n = 0; n < DP / 32; ++n)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      float4_t o = {acc[n][i], acc[n][i + 1], acc[n][i + 2], acc[n][i + 3]};
      *(float4_t*)(row + n * 32 + 2 * i + 4 * h) = o;
    }
}

// ---------------------------------------------------------------------------
// one tile's step of the running softmax: KB blocks of 32 keys in `s`
// (transposed scores, raw), O^T in `acc`; m and l are the row's reference
// maximum (raw) and this lane's share of the sum.
// ---------------------------------------------------------------------------
template <typename T, int DP, int KB>
DEV_INLINE void softmax_step(float16_t (&s)[KB], float16_t (&acc)[DP / 32],
                             float& m, float& l, float c) {
  // (four chains each for the maximum and the sum: one of 32 dependent
  // operations would be as long as the products)
  float t4[4] = {kNegInf, kNegInf, kNegInf, kNegInf};
#pragma unroll
  for (int kb = 0; kb < KB; ++kb)
#pragma unroll
    for (int i = 0; i < 16; i += 8)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        t4[j] = fmaxf(fmaxf(t4[j], s[kb][i + j]), s[kb][i + 4 + j]);
  const float top =
      pair_max(fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3])));
  // The reference follows the maximum only when that leaves it by more than
  // 2^8: until then the weights are at most 256, which no accumulator
  // minds, and the output is not scaled again
  const bool move = (top - m) * c > 8.f || (m == kNegInf && top > m);
  if (__any(move)) {
    const float to = move ? top : m;
    const float f = to == kNegInf ? 1.f
                                  : __builtin_amdgcn_exp2f((m - to) * c);
    m = to;
    l *= f;
#pragma unroll
    for (int n = 0; n < DP / 32; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[n][i] *= f;
  }
  const float off = m == kNegInf ? 0.f : m * c;
  float l4[4] = {};
#pragma unroll
  for (int kb = 0; kb < KB; ++kb)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[kb][i] = __builtin_amdgcn_exp2f(fmaf(s[kb][i], c, -off));
      l4[i & 3] += s[kb][i];
    }
  l += (l4[0] + l4[1]) + (l4[2] + l4[3]);
}

// scores of KB blocks of 32 keys, transposed, added to `from`
template <typename T, int DP, int KB>
DEV_INLINE void scores(const char* kt,
                       const typename Mat<T>::Frag (&qf)[DP / 16],
                       float16_t (&s)[KB], int l, float16_t from) {
  const int r = l & 31, h = l >> 5;
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) {
    s[kb] = from;
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks)
      s[kb] = Mat<T>::mma(Tile<T, DP>::row_frag(kt, kb * 32 + r, ks, h),
                          qf[ks], s[kb]);
  }
}

// acc += (tile's columns) x (weights): O^T += V^T P^T, dQ^T += K^T dS^T
template <typename T, int DP, int KB>
DEV_INLINE void weigh(const char* t, const float16_t (&s)[KB],
                      float16_t (&acc)[DP / 32], int l) {
#pragma unroll
  for (int kb = 0; kb < KB; ++kb)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const auto p = pack<T>(s[kb], k * 8);
#pragma unroll
      for (int n = 0; n < DP / 32; ++n)
        acc[n] = Mat<T>::mma(
            Tile<T, DP>::col_frag(t, kb * 32 + k * 16, n * 32, l), p, acc[n]);
    }
}

// keys that are not kept get a score of -inf; `keep` holds a byte a key
template <int KB>
DEV_INLINE void drop_keys(const uint8_t* keep, float16_t (&s)[KB], int h) {
#pragma unroll
  for (int kb = 0; kb < KB; ++kb)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const uint32_t k4 = *(const uint32_t*)(keep + kb * 32 + 2 * i + 4 * h);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (!((k4 >> (8 * j)) & 0xff)) s[kb][i + j] = kNegInf;
    }
}

// the workspace of a split: [split][B * Hk][rows][DP] values, then for the
// forward [split][B * Hk][rows][2] maxima and sums
DEV_INLINE long part_row(const Att& a, int split, long bh, int m) {
  return ((long)split * a.B * a.Hk + bh) * (a.G * (long)a.Sq) + m;
}

template <typename T, int DP>
DEV_INLINE void finish_row(const Att& a, const float16_t (&acc)[DP / 32],
                           float m, float l, int split, int b, int hk,
                           int row, int h) {
  const int M = a.G * a.Sq;
  if (row >= M) return;
  const float c = a.scale * kLog2e;
  const long bh = (long)b * a.Hk + hk;
  if (a.nsplit > 1) {
    const long at = part_row(a, split, bh, row);
    store_part<DP>(a.part + at * DP, acc, h);
    if (h == 0) {
      float* ml = a.part + (long)a.nsplit * a.B * a.Hk * M * DP + at * 2;
      ml[0] = m;
      ml[1] = l;
    }
    return;
  }
  store_row<T, DP>(q_row<T>(a.o, a, b, hk, row), acc, l > 0.f ? 1.f / l : 0.f,
                   h, a.D, a.vec);
  if (a.lse && h == 0)
    a.lse[bh * M + row] = l > 0.f ? m * c + __builtin_amdgcn_logf(l)
                                  : -kNegInf;
}

// ---------------------------------------------------------------------------
// forward: NW waves of 32 rows each over tiles of BN keys that all share.
// 54 us for 4x16 heads, 1024 rows over 1024 to 2048 keys of 64 in bf16 (470
// TFLOP/s of the kept keys).  Not faster there: the next tile's scores beside
// this one's exponentials (60 us, in any order of the two), eight waves with
// half the keys each (58), a raised wave priority for the products (55).
// ---------------------------------------------------------------------------
template <typename T, int DP, int NW, int BN>
__global__ __launch_bounds__(NW * 64, (waves<T, DP>(1, 384))) void att_fwd_kernel(Att a) {
  using TL = Tile<T, DP>;
  constexpr int NT = NW * 64, KB = BN / 32, BYTES = BN * TL::RB;
  __shared__ __attribute__((aligned(16))) char lk[2][BYTES], lv[2][BYTES];
  __shared__ __attribute__((aligned(16))) uint8_t lkeep[2][BN];
  const int M = a.G * a.Sq, mt = (M + NW * 32 - 1) / (NW * 32);
  int id = xcd_swizzle(blockIdx.x, gridDim.x);
  const int tile = id % mt;
  id /= mt;
  const int split = id % a.nsplit;
  int b, hk;
  seq_head(a, id / a.nsplit, &b, &hk);
  const int bh = b * a.Hk + hk;
  const int t = threadIdx.x, l = t & 63, h = l >> 5;
  const int row = tile * NW * 32 + (t >> 6) * 32 + (l & 31);
  const bool vec = a.vec;
  const int n = kept_keys(a, b);
  const int tiles = (n + BN - 1) / BN;
  const int t0 = (int)((long)tiles * split / a.nsplit);
  const int t1 = (int)((long)tiles * (split + 1) / a.nsplit);

  typename Mat<T>::Frag qf[DP / 16];
  const T* qr = row < M ? q_row<T>(a.q, a, b, hk, row) : nullptr;
#pragma unroll
  for (int ks = 0; ks < DP / 16; ++ks)
    qf[ks] = load_frag<T>(qr, ks, h, a.D, vec, row < M);
  float16_t acc[DP / 32] = {};
  float m = kNegInf, sum = 0.f;

  KeyTiles<T, DP, BN, NT> kt(a, b, hk, n, t);
  if (t0 < t1) {
    kt.load(t0);
    kt.store(lk[0], lv[0], lkeep[0], t0);
  }
  __syncthreads();
  in_turn(t0, t1, [&](int i, auto number) __attribute__((always_inline)) {
    constexpr int buf = decltype(number)::value;
    if (i + 1 < t1) kt.load(i + 1);
    float16_t s[KB];
    scores<T, DP, KB>(lk[buf], qf, s, l, float16_t{});
    if (kt.partial(i)) drop_keys<KB>(lkeep[buf], s, h);
    softmax_step<T, DP, KB>(s, acc, m, sum, a.scale * kLog2e);
    weigh<T, DP, KB>(lv[buf], s, acc, l);
    if (i + 1 < t1)
      kt.store(lk[buf ^ 1], lv[buf ^ 1], lkeep[buf ^ 1], i + 1);
    __syncthreads();
  });
  sum = pair_sum(sum);
  finish_row<T, DP>(a, acc, m, sum, split, b, hk, row, h);
}

// ---------------------------------------------------------------------------
// forward of at most 32 rows (single tokens): each wave takes its own keys, in
// its own part of LDS and without a barrier; the waves' results are joined at
// the end.  Bound by HBM: 8x8 heads of four rows over up to 16384 keys of 128
// in bf16 take 69 us (400 MB of kept keys: 5.8 TB/s) and the join 4.6; 32x16
// heads over up to 512 keys of 64, 15 us (50 MB), which latency bounds.  In fp32
// the two at full lengths take 237 us (4.5 TB/s; one wave a SIMD from size 65
// on) and 31 (4.4).
// ---------------------------------------------------------------------------
template <typename T, int DP, int BN>
__global__ __launch_bounds__(256, (waves<T, DP>(1))) void att_token_kernel(Att a) {
  using TL = Tile<T, DP>;
  constexpr int NW = 4, KB = BN / 32, BYTES = BN * TL::RB;
  constexpr int JOIN = 32 * (DP + 4) * 4;  // one wave's O^T, m and l
  constexpr int PER_WAVE = 2 * BYTES > JOIN ? 2 * BYTES : JOIN;
  __shared__ __attribute__((aligned(16))) char lds[NW][PER_WAVE];
  __shared__ __attribute__((aligned(16))) uint8_t lkeep[NW][BN];
  const int M = a.G * a.Sq;
  const int id = xcd_swizzle(blockIdx.x, gridDim.x);
  const int split = id % a.nsplit;
  int b, hk;
  seq_head(a, id / a.nsplit, &b, &hk);
  const int bh = b * a.Hk + hk;
  const int t = threadIdx.x, l = t & 63, h = l >> 5, w = t >> 6;
  const int row = l & 31;
  const bool vec = a.vec;
  const int n = kept_keys(a, b);
  const int tiles = (n + BN - 1) / BN, parts = a.nsplit * NW;
  const int t0 = (int)((long)tiles * (split * NW + w) / parts);
  const int t1 = (int)((long)tiles * (split * NW + w + 1) / parts);

  typename Mat<T>::Frag qf[DP / 16];
  const T* qr = row < M ? q_row<T>(a.q, a, b, hk, row) : nullptr;
#pragma unroll
  for (int ks = 0; ks < DP / 16; ++ks)
    qf[ks] = load_frag<T>(qr, ks, h, a.D, vec, row < M);
  float16_t acc[DP / 32] = {};
  float m = kNegInf, sum = 0.f;
  char *lk = lds[w], *lv = lds[w] + BYTES;

  KeyTiles<T, DP, BN, 64, true> kt(a, b, hk, n, l);
  if (t0 < t1) kt.load(t0);
  for (int i = t0; i < t1; ++i) {
    kt.store(lk, lv, lkeep[w], i);
    // a wave's LDS accesses are done in order; the fence keeps the compiler
    // from moving the reads of other lanes' values over these writes
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    if (i + 1 < t1) kt.load(i + 1);
    float16_t s[KB];
    scores<T, DP, KB>(lk, qf, s, l, float16_t{});
    if (kt.partial(i)) drop_keys<KB>(lkeep[w], s, h);
    softmax_step<T, DP, KB>(s, acc, m, sum, a.scale * kLog2e);
    weigh<T, DP, KB>(lv, s, acc, l);
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
  sum = pair_sum(sum);

  // join the waves: O^T as rows of DP + 4 values (the pad keeps the 32 rows
  // off each other's banks), then m and l behind them
  __syncthreads();
  float* mine = (float*)lds[w] + row * (DP + 4);
  store_part<DP>(mine, acc, h);
  if (h == 0) {
    mine[DP] = m;
    mine[DP + 1] = sum;
  }
  __syncthreads();
  if (w != 0) return;
  float top = kNegInf;
  const float c = a.scale * kLog2e;
#pragma unroll
  for (int k = 0; k < NW; ++k)
    top = fmaxf(top, ((const float*)lds[k])[row * (DP + 4) + DP]);
  sum = 0.f;
#pragma unroll
  for (int k = 0; k < DP / 32; ++k) acc[k] = float16_t{};
#pragma unroll
  for (int k = 0; k < NW; ++k) {
    const float* o = (const float*)lds[k] + row * (DP + 4);
    const float f = o[DP] == kNegInf
                        ? 0.f : __builtin_amdgcn_exp2f((o[DP] - top) * c);
    sum += o[DP + 1] * f;
#pragma unroll
    for (int nn = 0; nn < DP / 32; ++nn)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const float4_t v = *(const float4_t*)(o + nn * 32 + 2 * i + 4 * h);
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[nn][i + j] += v[j] * f;
      }
  }
  finish_row<T, DP>(a, acc, top, sum, split, b, hk, row, h);
}

// joins the splits of the forward: a wave a row.  Lane k has the k-th split's
// maximum and sum (there are at most 64), so only the values are read in turn,
// and no read waits for another.
template <typename T>
__global__ __launch_bounds__(256) void att_join_kernel(Att a, int DP) {
  const int M = a.G * a.Sq, l = threadIdx.x & 63;
  const long rows = (long)a.B * a.Hk * M;
  const long at = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (at >= rows) return;
  const float* ml = a.part + (long)a.nsplit * rows * DP +
                    ((long)min(l, a.nsplit - 1) * rows + at) * 2;
  const float c = a.scale * kLog2e;
  const float m = l < a.nsplit ? ml[0] : kNegInf;
  const float top = wave_reduce_max(m);
  const float f =
      m == kNegInf ? 0.f : __builtin_amdgcn_exp2f((m - top) * c);
  const float sum = wave_reduce_sum(m == kNegInf ? 0.f : ml[1] * f);
  float o0 = 0.f, o1 = 0.f;
  const float* o = a.part + at * DP + min(l, DP - 1);
  const float* p = a.part + at * DP + min(l + 64, DP - 1);
#pragma unroll 4
  for (int k = 0; k < a.nsplit; ++k) {
    const float fk = __shfl(f, k, 64);
    // (a split without a key wrote zeros)
    o0 += o[k * rows * DP] * fk;
    if (DP > 64) o1 += p[k * rows * DP] * fk;
  }
  const long bh = at / M;
  T* out = q_row<T>(a.o, a, bh / a.Hk, (int)(bh % a.Hk), (int)(at - bh * M));
  const float inv = sum > 0.f ? 1.f / sum : 0.f;
  if (l < a.D) out[l] = (T)(o0 * inv);
  if (l + 64 < a.D) out[l + 64] = (T)(o1 * inv);
  if (a.lse && l == 0)
    a.lse[at] = sum > 0.f ? top * c + __builtin_amdgcn_logf(sum) : -kNegInf;
}

// ---------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------

// A row's dS 2^shift of one tile: where the largest is over kMostDs, the shift
// goes down until it lies between 2^13 and 2^14, for the row's sums too.  (An
// infinity, of an infinite gradient, stays one and lowers nothing.)
template <int DP, int KB>
DEV_INLINE void lower_shift(float16_t (&s)[KB], float16_t (&acc)[DP / 32],
                            float& lse) {
  float t4[4] = {};
#pragma unroll
  for (int kb = 0; kb < KB; ++kb)
#pragma unroll
    for (int i = 0; i < 16; i += 8)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        t4[j] = fmaxf(fmaxf(t4[j], fabsf(s[kb][i + j])),
                      fabsf(s[kb][i + 4 + j]));
  float top = fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3]));
  if (!__any(top > kMostDs)) return;
  top = pair_max(top);
  const int down = top > kMostDs && top < -kNegInf && fabsf(lse) < 2 * kMostLse
                       ? ilogbf(top) - 13
                       : 0;
  const float f = ldexpf(1.f, -down);
  lse += (float)down;
#pragma unroll
  for (int kb = 0; kb < KB; ++kb)
#pragma unroll
    for (int i = 0; i < 16; ++i) s[kb][i] *= f;
#pragma unroll
  for (int n = 0; n < DP / 32; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[n][i] *= f;
}

// dQ: rows as in the forward, over all keys (or a split's).  61 us where the
// forward takes 54, with 12 products for its 8; the row's dO . O costs one read
// of its output here, and no launch.
template <typename T, int DP, int NW, int BN>
__global__ __launch_bounds__(NW * 64, (waves<T, DP>(1))) void att_dq_kernel(Att a) {
  using TL = Tile<T, DP>;
  constexpr int NT = NW * 64, KB = BN / 32, BYTES = BN * TL::RB;
  __shared__ __attribute__((aligned(16))) char lk[2][BYTES], lv[2][BYTES];
  __shared__ __attribute__((aligned(16))) uint8_t lkeep[2][BN];
  const int M = a.G * a.Sq, mt = (M + NW * 32 - 1) / (NW * 32);
  int id = xcd_swizzle(blockIdx.x, gridDim.x);
  const int tile = id % mt;
  id /= mt;
  const int split = id % a.nsplit;
  int b, hk;
  seq_head(a, id / a.nsplit, &b, &hk);
  const int bh = b * a.Hk + hk;
  const int t = threadIdx.x, l = t & 63, h = l >> 5, r = l & 31;
  const int row = tile * NW * 32 + (t >> 6) * 32 + r;
  const bool vec = a.vec;
  const int n = kept_keys(a, b);
  const int tiles = (n + BN - 1) / BN;
  const int t0 = (int)((long)tiles * split / a.nsplit);
  const int t1 = (int)((long)tiles * (split + 1) / a.nsplit);
  const float c = a.scale * kLog2e;

  typename Mat<T>::Frag qf[DP / 16], gf[DP / 16];
  const T* qr = row < M ? q_row<T>(a.q, a, b, hk, row) : nullptr;
  const T* gr = row < M ? q_row<T>(a.dout, a, b, hk, row) : nullptr;
#pragma unroll
  for (int ks = 0; ks < DP / 16; ++ks) {
    qf[ks] = load_frag<T>(qr, ks, h, a.D, vec, row < M);
    gf[ks] = load_frag<T>(gr, ks, h, a.D, vec, row < M);
  }
  float lse = row < M ? a.lse[(long)bh * M + row] : -kNegInf;
  // (with the shift in it: exp2 then gives P 2^shift)
  if constexpr (kShifted<T>) lse -= (float)first_shift(lse);
  // the row's dO . O, which dK and dV need too
  float delta = 0.f;
  {
    const T* orow = row < M ? q_row<T>(a.o, a, b, hk, row) : nullptr;
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) {
      const auto of = load_frag<T>(orow, ks, h, a.D, vec, row < M);
#pragma unroll
      for (int j = 0; j < 8; ++j) delta += (float)of[j] * (float)gf[ks][j];
    }
    delta = pair_sum(delta);
    if (split == 0 && h == 0 && row < M)
      a.delta[(long)bh * M + row] = delta;
  }
  // dP is added to -delta by its products
  float16_t acc[DP / 32] = {}, less;
#pragma unroll
  for (int j = 0; j < 16; ++j) less[j] = -delta;

  KeyTiles<T, DP, BN, NT> kt(a, b, hk, n, t);
  if (t0 < t1) {
    kt.load(t0);
    kt.store(lk[0], lv[0], lkeep[0], t0);
  }
  __syncthreads();
  in_turn(t0, t1, [&](int i, auto number) __attribute__((always_inline)) {
    constexpr int buf = decltype(number)::value;
    if (i + 1 < t1) kt.load(i + 1);
    float16_t s[KB], dp[KB];
    if constexpr (DP > 64) {
      // (16 moves a tile: kept, these registers put others into scratch memory;
      // backward of 4x16 heads, 1024 over 2048 keys of 128: 412 us, 429)
      float d = -delta;
      asm volatile("" : "+v"(d));
#pragma unroll
      for (int j = 0; j < 16; ++j) less[j] = d;
    }
    scores<T, DP, KB>(lk[buf], qf, s, l, float16_t{});
    scores<T, DP, KB>(lv[buf], gf, dp, l, less);
    if (kt.partial(i)) drop_keys<KB>(lkeep[buf], s, h);
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int j = 0; j < 16; ++j)
        s[kb][j] =
            __builtin_amdgcn_exp2f(fmaf(s[kb][j], c, -lse)) * dp[kb][j];
    if constexpr (kShifted<T>) lower_shift<DP, KB>(s, acc, lse);
    weigh<T, DP, KB>(lk[buf], s, acc, l);
    if (i + 1 < t1)
      kt.store(lk[buf ^ 1], lv[buf ^ 1], lkeep[buf ^ 1], i + 1);
    __syncthreads();
  });
  if (row >= M) return;
  if (lse == -kNegInf) {  // no key: zeros, also where dO is not finite
#pragma unroll
    for (int n = 0; n < DP / 32; ++n) acc[n] = float16_t{};
  }
  float back = 1.f;
  if constexpr (kShifted<T>) {
    const float whole = a.lse[(long)bh * M + row];
    const int shift =
        fabsf(whole) < 4 * kMostLse ? (int)rintf(whole - lse) : 0;
    back = ldexpf(1.f, -shift);
    if (h == 0) a.shift[((long)bh * a.nsplit + split) * M + row] = shift;
  }
  if (a.nsplit > 1) {
    if constexpr (kShifted<T>)
#pragma unroll
      for (int n = 0; n < DP / 32; ++n)
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[n][j] *= back;
    store_part<DP>(a.part + part_row(a, split, bh, row) * DP, acc, h);
  } else {
    store_row<T, DP>(q_row<T>(a.dq, a, b, hk, row), acc, a.scale * back, h,
                     a.D, vec);
  }
}

// dK and dV: NW waves of 32 keys each over tiles of BM rows (or a split's).
// 97 us where the forward takes 54, with 16 products for its 8: every tile of
// rows is read from LDS as rows and as columns, 16 KB for 32x32 scores, so LDS
// is busy as long as the matrix cores.
template <typename T, int DP, int NW, int BM>
__global__ __launch_bounds__(NW * 64, (waves<T, DP>(2, 384))) void att_dkv_kernel(Att a) {
  using TL = Tile<T, DP>;
  constexpr int NT = NW * 64, BYTES = BM * TL::RB;
  __shared__ __attribute__((aligned(16))) char lq[2][BYTES], lg[2][BYTES];
  __shared__ __attribute__((aligned(16))) float llse[2][BM], ldel[2][BM];
  const int M = a.G * a.Sq, kt = (a.Sk + NW * 32 - 1) / (NW * 32);
  int id = xcd_swizzle(blockIdx.x, gridDim.x);
  const int tile = id % kt;
  id /= kt;
  const int split = id % a.nsplit;
  int b, hk;
  seq_head(a, id / a.nsplit, &b, &hk);
  const int bh = b * a.Hk + hk;
  const int t = threadIdx.x, l = t & 63, h = l >> 5, r = l & 31;
  const int k0 = tile * NW * 32 + (t >> 6) * 32, key = k0 + r;
  const bool vec = a.vec;
  const int n = kept_keys(a, b);
  const bool keep = key < n && (!a.mask || a.mask[(long)b * a.Sk + key]);
  const float c = a.scale * kLog2e;
  // a block whose keys are all past the length only writes its zeros
  const int tiles = tile * NW * 32 < n ? (M + BM - 1) / BM : 0;
  const int t0 = (int)((long)tiles * split / a.nsplit);
  const int t1 = (int)((long)tiles * (split + 1) / a.nsplit);

  // the rows' shifts, of which most launches have one a thread
  const int shifts = kShifted<T> && t0 < t1 ? a.dq_splits * M : 0;
  const int* ps = kShifted<T> ? a.shift + (long)bh * a.dq_splits * M : nullptr;
  int least = t < shifts ? ps[t] : 15;
  typename Mat<T>::Frag kf[DP / 16], vf[DP / 16];
  const T* kr = keep ? row_ptr<T>(a.k, b, hk, key) : nullptr;
  const T* vr = keep ? row_ptr<T>(a.v, b, hk, key) : nullptr;
#pragma unroll
  for (int ks = 0; ks < DP / 16; ++ks) {
    kf[ks] = load_frag<T>(kr, ks, h, a.D, vec, keep);
    vf[ks] = load_frag<T>(vr, ks, h, a.D, vec, keep);
  }
  float16_t dk[DP / 32] = {}, dv[DP / 32] = {};
  using S = Stage<T, DP, BM, NT>;
  S sq, sg;
  const unsigned qo = S::offset(t, a.q.ss, a.D),
                 go = S::offset(t, a.dout.ss, a.D);
  float rl = 0.f, rd = 0.f;  // one row's log-sum and dO . O
  static_assert(BM <= NT, "a row a thread");
  auto fetch = [&](int i) __attribute__((always_inline)) {
    const int m0 = i * BM, g = m0 / a.Sq, s0 = m0 - g * a.Sq;
    const long at = (long)bh * M + min(m0 + t, M - 1);
    rl = a.lse[at];
    rd = a.delta[at];
    if (vec && s0 + BM <= a.Sq) {  // rows of one head
      sq.load(row_ptr<T>(a.q, b, hk * a.G + g, s0), a.q.ss, qo, t, a.D);
      sg.load(row_ptr<T>(a.dout, b, hk * a.G + g, s0), a.dout.ss, go, t, a.D);
      return;
    }
    auto ok = [&](int rr) { return m0 + rr < M; };
    sq.load([&](int rr) -> const T* {
      return q_row<T>(a.q, a, b, hk, min(m0 + rr, M - 1));
    }, ok, t, a.D, vec);
    sg.load([&](int rr) -> const T* {
      return q_row<T>(a.dout, a, b, hk, min(m0 + rr, M - 1));
    }, ok, t, a.D, vec);
  };
  // Their lowest is the block's.  P takes it as far as it is not negative
  // (small gradients), dS all of it
  int shift = 0;
  if (t0 < t1) fetch(t0);
  if constexpr (kShifted<T>) {
    __shared__ int lshift[NW];
    for (int i = t + NT; i < shifts; i += NT) least = min(least, ps[i]);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1)
      least = min(least, __shfl_xor(least, off, 64));
    if (l == 0) lshift[t >> 6] = least;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < NW; ++k) least = min(least, lshift[k]);
    shift = __builtin_amdgcn_readfirstlane(least);
  }
  const int up = max(shift, 0);
  auto scalar = [](float v) {
    return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(v)));
  };
  const float fup = scalar((float)up),
              fdown = scalar(ldexpf(1.f, min(shift, 0)));
  // (where it is negative, through V and dO . O: 16 products for each 32x32
  // scores, or a branch, put registers into scratch memory)
  if (kShifted<T> && shift < 0) {
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks)
#pragma unroll
      for (int j = 0; j < 8; ++j) vf[ks][j] = (T)((float)vf[ks][j] * fdown);
  }
  auto put = [&](int i, int buf) __attribute__((always_inline)) {
    const bool all = a.D == DP && (i + 1) * BM <= M;
    sq.store(lq[buf], t, all);
    sg.store(lg[buf], t, all);
    if (t < BM) {
      // a row past the end has a weight of exp2(-inf)
      llse[buf][t] = i * BM + t < M ? rl - fup : -kNegInf;
      ldel[buf][t] = i * BM + t < M ? -rd * fdown : 0.f;
    }
  };
  if (t0 < t1) put(t0, 0);
  __syncthreads();
  in_turn(t0, t1, [&](int i, auto number) __attribute__((always_inline)) {
    constexpr int buf = decltype(number)::value;
    if (i + 1 < t1) fetch(i + 1);
#pragma unroll
    for (int mb = 0; mb < BM / 32; ++mb) {
      // dP is added to -delta by its products
      float16_t s = {}, dp;
#pragma unroll
      for (int j = 0; j < 16; j += 4) {
        const float4_t less =
            *(const float4_t*)&ldel[buf][mb * 32 + 2 * j + 4 * h];
#pragma unroll
        for (int e = 0; e < 4; ++e) dp[j + e] = less[e];
      }
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks)
        s = Mat<T>::mma(TL::row_frag(lq[buf], mb * 32 + r, ks, h), kf[ks], s);
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks)
        dp = Mat<T>::mma(TL::row_frag(lg[buf], mb * 32 + r, ks, h), vf[ks],
                         dp);
#pragma unroll
      for (int j = 0; j < 16; j += 4) {
        const int at = mb * 32 + 2 * j + 4 * h;
        const float4_t lse = *(const float4_t*)&llse[buf][at];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[j + e] = __builtin_amdgcn_exp2f(fmaf(s[j + e], c, -lse[e]));
          dp[j + e] *= s[j + e];
        }
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const auto p = pack<T>(s, k * 8), ds = pack<T>(dp, k * 8);
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) {
          dv[d] = Mat<T>::mma(
              p, TL::col_frag(lg[buf], mb * 32 + k * 16, d * 32, l), dv[d]);
          dk[d] = Mat<T>::mma(
              ds, TL::col_frag(lq[buf], mb * 32 + k * 16, d * 32, l), dk[d]);
        }
      }
    }
    if (i + 1 < t1) put(i + 1, buf ^ 1);
    __syncthreads();
  });
  // a key that is not kept had weights too (its scores were zeros), which went
  // to its own row alone and become zeros here
  const unsigned kept = (unsigned)__ballot(keep);
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const int k = k0 + 8 * (j / 4) + 4 * h + (j & 3), col = d * 32 + r;
      if (k >= a.Sk) continue;
      if constexpr (kShifted<T>) {
        dk[d][j] = ldexpf(dk[d][j], -shift);
        dv[d][j] = ldexpf(dv[d][j], -up);
      }
      if (!(kept >> (k - k0) & 1)) dk[d][j] = dv[d][j] = 0.f;
      if (a.nsplit > 1) {
        float* p = a.part +
                   (((long)split * a.B * a.Hk + bh) * a.Sk + k) * 2 * DP;
        p[col] = dk[d][j];
        p[DP + col] = dv[d][j];
      } else if (col < a.D) {
        ((T*)row_ptr<T>(a.dk, b, hk, k))[col] = (T)(dk[d][j] * a.scale);
        ((T*)row_ptr<T>(a.dv, b, hk, k))[col] = (T)dv[d][j];
      }
    }
}

// sums of the splits' dQ, in the splits' order: a wave a row
template <typename T>
__global__ __launch_bounds__(256) void att_dq_join_kernel(Att a, int DP) {
  const int M = a.G * a.Sq, l = threadIdx.x & 63;
  const long rows = (long)a.B * a.Hk * M;
  const long at = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (at >= rows) return;
  const long bh = at / M;
  T* out = q_row<T>(a.dq, a, bh / a.Hk, (int)(bh % a.Hk),
                    (int)(at - bh * M));
  for (int d = l; d < a.D; d += 64) {
    float v = 0.f;
    for (int k = 0; k < a.nsplit; ++k) v += a.part[(k * rows + at) * DP + d];
    out[d] = (T)(v * a.scale);
  }
}

template <typename T>
__global__ __launch_bounds__(256) void att_dkv_join_kernel(Att a, int DP) {
  const int l = threadIdx.x & 63;
  const long rows = (long)a.B * a.Hk * a.Sk;
  const long at = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (at >= rows) return;
  const long bh = at / a.Sk;
  const int key = (int)(at - bh * a.Sk);
  T* dk = (T*)row_ptr<T>(a.dk, bh / a.Hk, (int)(bh % a.Hk), key);
  T* dv = (T*)row_ptr<T>(a.dv, bh / a.Hk, (int)(bh % a.Hk), key);
  for (int d = l; d < a.D; d += 64) {
    float u = 0.f, v = 0.f;
    for (int k = 0; k < a.nsplit; ++k) {
      const float* p = a.part + (k * rows + at) * 2 * DP;
      u += p[d];
      v += p[DP + d];
    }
    dk[d] = (T)(u * a.scale);
    dv[d] = (T)v;
  }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
int pad_dim(int D) { return (D + 31) / 32 * 32; }

// As many splits as bring the launch to `want` blocks, none shorter than
// `least` tiles of 64
int splits(long blocks, long want, long tiles, long least) {
  const long n = std::min(want / std::max<long>(blocks, 1), tiles / least);
  return (int)std::max<long>(1, std::min<long>(n, 64));
}

constexpr int NW = 4;  // waves of rows (keys for dK and dV) in a block

struct Plan {
  int DP;
  bool token;         // the forward's kernel for at most 32 rows
  int fwd, dq, dkv;   // splits
};

// Up to 32 rows that share a key head, the kernel for single tokens (14 us
// against 17 for 32x16 heads over 512 keys of 64, 85 against 107 for 8x8 heads
// of four rows over 16384 of 128; at 32 rows over 128 keys both take 7).
// Blocks of two waves for 64 rows or keys gained nothing over four.
//
// One block a CU (256) is wanted: 512 rows of 8 heads over 4096 keys of 64
// take 22 us forward and 45 back with 256, 24 and 59 with 512, 70 and 96 with
// no split.  Single tokens, whose time is their longest sequence's, want twice
// that (8 sequences of up to 16384 keys: 75 us, and 79 with 256).
// A split costs a launch and its partial results, so it has four tiles (about
// 4 us) or more, eight of single tokens; one tile in fp32, whose products take
// 16 times as long.
Plan make_plan(long B, long H, long Hk, long Sq, long Sk, long D, int dtype) {
  Plan p;
  const long M = H / Hk * Sq, bh = B * Hk, tile = NW * 32;
  const long least = dtype == kFloat32 ? 1 : 4;
  const long rows = bh * ((M + tile - 1) / tile);
  const long tiles = (Sk + 63) / 64;
  p.DP = pad_dim((int)D);
  p.token = M <= 32;
  p.fwd = p.token ? splits(bh, 512, tiles, 8) : splits(rows, 256, tiles, least);
  p.dq = splits(rows, 256, tiles, least);
  p.dkv = splits(bh * ((Sk + tile - 1) / tile), 256, (M + 63) / 64, least);
  return p;
}

struct Heads {
  long B, S, sb, ss;
};

// [B, S, ...] or, time first, [S, B, ...]
Heads lead(const Arr& x, bool tnc, const char* name) {
  MX_CHECK(x.dim() == 3, name << " must have three axes");
  const long n = x.size(2), a = x.size(0), b = x.size(1);
  return tnc ? Heads{b, a, n, b * n} : Heads{a, b, b * n, n};
}

View view(const Arr& x, const Heads& h, long off, long sh) {
  return View{(char*)x.ptr + off * dtype_size(x.dtype), h.sb, h.ss, sh};
}

// whether the values come apart from the keys (an array of no keys has no
// memory, but axes)
bool given(const Arr& values) { return values.dim() > 0; }

Att make_att(const Arr& q, const Arr& kv, const Arr& values, int heads,
             int kv_heads, const Arr& len, const Arr& mask, bool tnc) {
  const char* name = "encdec_attention";
  const Heads hq = lead(q, tnc, name), hk = lead(kv, tnc, name);
  MX_CHECK(heads > 0 && kv_heads > 0 && heads % kv_heads == 0,
           name << ": kv_heads must divide heads");
  MX_CHECK(q.size(2) % heads == 0, name << ": heads must divide the queries");
  const long D = q.size(2) / heads;
  const bool apart = given(values);
  MX_CHECK(D >= 1 && D <= 128, name << ": head sizes of 1 to 128, got " << D);
  MX_CHECK(hq.B == hk.B && kv.dtype == q.dtype &&
               kv.size(2) == kv_heads * D * (apart ? 1 : 2),
           name << ": the keys do not fit the queries and heads");
  if (apart) {
    const Heads hv = lead(values, tnc, name);
    MX_CHECK(hv.B == hk.B && hv.S == hk.S && values.size(2) == kv.size(2) &&
                 values.dtype == kv.dtype,
             name << ": the values must be like the keys");
  }
  MX_CHECK(!len.defined() || ((len.dtype == kInt32 || len.dtype == kInt64) &&
                              len.numel() == hq.B),
           name << ": valid_length must hold one int32 or int64 for each "
                   "sequence");
  MX_CHECK(!mask.defined() || ((mask.dtype == kUint8 || mask.dtype == kBool) &&
                               mask.numel() == hk.B * hk.S),
           name << ": the mask must hold one byte for each key");
  // (the quotient of a row by Sq comes from a reciprocal in float32, at most
  // one off for up to 2^20 heads)
  MX_CHECK(hq.S * heads < (1L << 30) && hk.S < (1L << 30) &&
               hq.B * heads < (1L << 30) && heads <= (1 << 20),
           name << ": too many rows, keys, heads or sequences");
  Att a = {};
  a.q = view(q, hq, 0, D);
  if (apart) {
    a.k = view(kv, hk, 0, D);
    a.v = view(values, hk, 0, D);
  } else {
    a.k = view(kv, hk, 0, 2 * D);
    a.v = view(kv, hk, D, 2 * D);
  }
  a.len = len.ptr;
  a.len64 = len.dtype == kInt64;
  a.mask = mask.data<uint8_t>();
  a.B = (int)hq.B;
  a.H = heads;
  a.Hk = kv_heads;
  a.G = heads / kv_heads;
  a.Sq = (int)hq.S;
  a.Sk = (int)hk.S;
  a.D = (int)D;
  a.nsplit = 1;
  a.scale = 1.f / sqrtf((float)D);
  a.inv_sq = hq.S ? 1.f / (float)hq.S : 0.f;
  return a;
}

bool vectors(std::initializer_list<View> vs, int D, size_t size) {
  if ((D * size) % 16) return false;  // then so are all strides
  for (auto& v : vs)
    // (a tile's rows are offsets of 32 bits from its first)
    if (((uintptr_t)v.p & 15) || v.ss * 64 * (long)size >= 1L << 31)
      return false;
  return true;
}

// (a launch has fewer than 2^32 threads: 2^24 blocks of 256)
unsigned grid(long blocks) {
  MX_CHECK(blocks < (1L << 24), "encdec_attention: too many sequences");
  return (unsigned)blocks;
}

template <typename F>
void by_dim(int DP, F f) {
  if (DP == 32) f(std::integral_constant<int, 32>{});
  else if (DP == 64) f(std::integral_constant<int, 64>{});
  else if (DP == 96) f(std::integral_constant<int, 96>{});
  else f(std::integral_constant<int, 128>{});
}

// Rows a tile: 64 where two waves' registers hold it on its way beside their
// operands and accumulators, else 32 (forward of 4x16 heads, 1024 over 2048
// keys of 128 in bf16: 100 us with 32, 115 with 64, which spills)
template <typename T, int DP>
constexpr int tile_rows() { return sizeof(T) == 2 && DP <= 64 ? 64 : 32; }

template <typename T>
void fwd(const LaunchCtx& lc, Att a, const Plan& p) {
  a.vec = vectors({a.q, a.k, a.v, a.o}, a.D, sizeof(T));
  a.nsplit = p.fwd;
  const long bh = (long)a.B * a.Hk, M = (long)a.G * a.Sq;
  by_dim(p.DP, [&](auto dp) {
    constexpr int DP = decltype(dp)::value, BN = tile_rows<T, DP>();
    const unsigned n = grid(
        bh * a.nsplit * (p.token ? 1 : (M + NW * 32 - 1) / (NW * 32)));
    if (p.token)
      // a wave's own tile of 16 KB at most.  (Tiles of 32 keys in blocks of
      // eight waves, four a SIMD: 21 us for 32x16 heads over 512 keys of 64,
      // where this takes 17.)
      att_token_kernel<T, DP, sizeof(T) == 2 && DP <= 64 ? 64 : 32>
          <<<n, 256, 0, lc.stream>>>(a);
    else
      att_fwd_kernel<T, DP, NW, BN><<<n, NW * 64, 0, lc.stream>>>(a);
  });
  if (a.nsplit > 1)
    att_join_kernel<T><<<grid((bh * M + 3) / 4), 256, 0, lc.stream>>>(a, p.DP);
}

template <typename T>
void bwd(const LaunchCtx& lc, Att a, const Plan& p) {
  a.vec = vectors({a.q, a.k, a.v, a.o, a.dout, a.dq}, a.D, sizeof(T));
  const long bh = (long)a.B * a.Hk, M = (long)a.G * a.Sq;
  if (M) {
    a.nsplit = p.dq;
    by_dim(p.DP, [&](auto dp) {
      constexpr int DP = decltype(dp)::value, BN = tile_rows<T, DP>();
      const unsigned n = grid(bh * a.nsplit * ((M + NW * 32 - 1) / (NW * 32)));
      att_dq_kernel<T, DP, NW, BN><<<n, NW * 64, 0, lc.stream>>>(a);
    });
    if (a.nsplit > 1)
      att_dq_join_kernel<T>
          <<<grid((bh * M + 3) / 4), 256, 0, lc.stream>>>(a, p.DP);
  }
  if (a.Sk) {
    a.nsplit = p.dkv;
    by_dim(p.DP, [&](auto dp) {
      constexpr int DP = decltype(dp)::value, BN = tile_rows<T, DP>();
      const unsigned n =
          grid(bh * a.nsplit * ((a.Sk + NW * 32 - 1) / (NW * 32)));
      att_dkv_kernel<T, DP, NW, BN><<<n, NW * 64, 0, lc.stream>>>(a);
    });
    if (a.nsplit > 1)
      att_dkv_join_kernel<T>
          <<<grid((bh * a.Sk + 3) / 4), 256, 0, lc.stream>>>(a, p.DP);
  }
}

// Behind delta of each row, and its shift in each split of dQ, the backward's
// partial results start at 16 bytes
int64_t behind_rows(const Plan& p, int64_t rows, int dtype) {
  const int64_t n = rows * (dtype == kFloat16 ? 1 + p.dq : 1);
  return (n + 3) & ~(int64_t)3;
}

}  // namespace

std::vector<int64_t> encdec_attention_workspace(int64_t B, int64_t H,
                                                int64_t Hk, int64_t Sq,
                                                int64_t Sk, int64_t D,
                                                int dtype) {
  MX_CHECK(H > 0 && Hk > 0 && H % Hk == 0 && D > 0,
           "encdec_attention: bad heads");
  const Plan p = make_plan(B, H, Hk, Sq, Sk, D, dtype);
  const int64_t rows = B * H * Sq;
  const int64_t fwd = p.fwd > 1 ? p.fwd * rows * (p.DP + 2) : 0;
  const int64_t dq = p.dq > 1 ? p.dq * rows * p.DP : 0;
  const int64_t dkv = p.dkv > 1 ? p.dkv * B * Hk * Sk * 2 * p.DP : 0;
  // the two splits of the backward use the workspace one after the other
  return {fwd, behind_rows(p, rows, dtype) + std::max(dq, dkv)};
}

void encdec_attention_fwd_raw(const LaunchCtx& lc, const Arr& q,
                              const Arr& kv, const Arr& values, int heads,
                              int kv_heads, const Arr& len, const Arr& mask,
                              bool tnc, const Arr& out, const Arr& lse,
                              const Arr& work) {
  if (out.numel() == 0) return;
  Att a = make_att(q, kv, values, heads, kv_heads, len, mask, tnc);
  const Plan p = make_plan(a.B, a.H, a.Hk, a.Sq, a.Sk, a.D, q.dtype);
  MX_CHECK(out.shape == q.shape && out.dtype == q.dtype,
           "encdec_attention: the output must be like the queries");
  MX_CHECK(!lse.defined() ||
               (lse.dtype == kFloat32 && lse.numel() == (long)a.B * a.H * a.Sq),
           "encdec_attention: one float32 for each row of each head");
  MX_CHECK((work.defined() && work.dtype == kFloat32 ? work.numel() : 0) >=
               encdec_attention_workspace(a.B, a.H, a.Hk, a.Sq, a.Sk, a.D,
                                          q.dtype)[0],
           "encdec_attention: workspace too small");
  a.o = view(out, lead(out, tnc, "out"), 0, a.D);
  a.lse = lse.data<float>();
  a.part = work.data<float>();
  DISPATCH_FLOAT_NATIVE(q.dtype, "encdec_attention",
                        [&] { fwd<scalar_t>(lc, a, p); });
  HIP_CHECK_LAST();
}

void encdec_attention_bwd_raw(const LaunchCtx& lc, const Arr& dout,
                              const Arr& q, const Arr& kv, const Arr& values,
                              int heads, int kv_heads, const Arr& len,
                              const Arr& mask, bool tnc, const Arr& out,
                              const Arr& lse, const Arr& dq, const Arr& dkv,
                              const Arr& dvalues, const Arr& work) {
  if (dkv.numel() == 0 && dq.numel() == 0) return;
  Att a = make_att(q, kv, values, heads, kv_heads, len, mask, tnc);
  const Plan p = make_plan(a.B, a.H, a.Hk, a.Sq, a.Sk, a.D, q.dtype);
  MX_CHECK(dout.shape == q.shape && dout.dtype == q.dtype &&
               out.shape == q.shape && out.dtype == q.dtype &&
               dq.shape == q.shape && dq.dtype == q.dtype &&
               dkv.shape == kv.shape && dkv.dtype == kv.dtype &&
               given(values) == given(dvalues) &&
               (!given(values) || (dvalues.shape == values.shape &&
                                      dvalues.dtype == values.dtype)),
           "encdec_attention backward: a gradient must be like its input");
  const long rows = (long)a.B * a.H * a.Sq;
  MX_CHECK(rows == 0 || (lse.dtype == kFloat32 && lse.numel() == rows),
           "encdec_attention backward: one float32 for each row");
  MX_CHECK((work.defined() && work.dtype == kFloat32 ? work.numel() : 0) >=
               encdec_attention_workspace(a.B, a.H, a.Hk, a.Sq, a.Sk, a.D,
                                          q.dtype)[1],
           "encdec_attention backward: workspace too small");
  a.o = view(out, lead(out, tnc, "out"), 0, a.D);
  a.dout = view(dout, lead(dout, tnc, "dout"), 0, a.D);
  a.dq = view(dq, lead(dq, tnc, "dq"), 0, a.D);
  const Heads hk = lead(dkv, tnc, "dkv");
  if (given(values)) {
    a.dk = view(dkv, hk, 0, a.D);
    a.dv = view(dvalues, hk, 0, a.D);
  } else {
    a.dk = view(dkv, hk, 0, 2 * a.D);
    a.dv = view(dkv, hk, a.D, 2 * a.D);
  }
  a.lse = lse.data<float>();
  a.delta = work.data<float>();
  a.shift = (int*)(a.delta + rows);
  a.dq_splits = p.dq;
  a.part = a.delta + behind_rows(p, rows, q.dtype);
  DISPATCH_FLOAT_NATIVE(q.dtype, "encdec_attention backward",
                        [&] { bwd<scalar_t>(lc, a, p); });
  HIP_CHECK_LAST();
}

}  // namespace mxcore
