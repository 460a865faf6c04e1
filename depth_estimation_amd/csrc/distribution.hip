// Distributions over classes (disparity bins, tokens): log-probabilities of given classes with the
// entropy and the top alternatives, and distillation from a teacher's listed classes; forward and
// backward, for float32, bfloat16 and float16 logits.
//
// Per row, with z_j = scale * x_j and everything in base 2 (c = scale * log2 e):
//   m = the x_j of the largest z_j,  t_j = (x_j - m) c,  e_j = 2^t_j,  s = sum e_j,  w = sum e_j t_j
//   log p_j = ln2 t_j - ln s,   entropy = ln s - ln2 w / s
// one pass over the data with a running (m, s, w): when the extremum moves by d = (m_old - m_new) c,
// s <- s 2^d and w <- 2^d (w + s d).  The difference x_j - m is taken before the product, so rows
// at the end of the float32 range (all classes at the type's lowest value) keep their meaning.  A
// negative scale (costs) needs no sign change of the data: m is the smallest x_j then, c is negative,
// and `far`, the x of an impossible class, is +inf.
//
// Two families of kernels:
//   tile  one thread a row, 64 rows a wave; the waves of a block share the classes of their 64 rows.
//         The classes of a volume (B, V, inner) are read plane by plane (64 neighbouring pixels a
//         load); rows whose classes lie together are turned through LDS, 128 bytes of each row at
//         a time, or all of the 64 rows at once, as one stretch of memory ("flat"), if they are not whole lines.
//         No cross-lane work at all, and the top classes stay sorted in registers.
//   row   a block (or a few, joined by a second kernel) for each row, for rows that are long or few.
//
// Every pass reads the logits once and a backward pass writes as much again, so the bound is memory: a large copy
// moves 4.8 TB/s on this chip, a large read 5.4.  Next to it stands the vector pipe, with 11 instructions a class in
// the forward pass and a quarter-rate exp2 among them.  The figures at the kernels are times of the kernel alone.
#include <type_traits>

#include "dw_common.h"

namespace {
using namespace dw;

constexpr float kInf = __builtin_inff();
constexpr float kLn2 = 0x1.62e43p-1f;      // fl(ln 2)
constexpr float kLog2e = 0x1.715476p+0f;   // fl(log2 e)
constexpr float kLog2eRest = 0x1.4ae0cp-26f;  // log2 e - fl(log2 e)
constexpr float kFloor = -1e30f;           // stands in for an exponent of -inf where 0 * -inf would be NaN
// The same in a gradient, where it is multiplied by an upstream value: 2^-1000 is 0 already, and the product stays finite
// for upstream gradients up to 1e35
constexpr float kGradFloor = -1000.f;
constexpr int kMaxEntries = 64;

// ---- element types -------------------------------------------------------------------------
struct F32 {
  using S = float;
  static constexpr int VEC = 4;
  static __device__ __forceinline__ float up(float v) { return v; }
  static __device__ __forceinline__ float down(float v) { return v; }
};
struct BF16 {
  using S = uint16_t;
  static constexpr int VEC = 8;
  static __device__ __forceinline__ float up(uint16_t v) { return __builtin_bit_cast(float, (unsigned)v << 16); }
  static __device__ __forceinline__ uint16_t down(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }
  static __device__ __forceinline__ float lower(unsigned d) { return __builtin_bit_cast(float, d << 16); }
  static __device__ __forceinline__ float upper(unsigned d) { return __builtin_bit_cast(float, d & 0xffff0000u); }
};
struct F16 {
  using S = uint16_t;
  static constexpr int VEC = 8;
  static __device__ __forceinline__ float up(uint16_t v) { return (float)__builtin_bit_cast(_Float16, v); }
  static __device__ __forceinline__ uint16_t down(float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }
  static __device__ __forceinline__ float lower(unsigned d) { return up((uint16_t)d); }
  static __device__ __forceinline__ float upper(unsigned d) { return up((uint16_t)(d >> 16)); }
};

// 16 bytes of elements, kept as the four words they are loaded as: taken apart at the load, they would have
// to be waited for there
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 __attribute__((aligned(2))) u32x4_any;
template <class T>
struct Vec {
  u32x4 d;
  __device__ __forceinline__ float get(int e) const {
    const unsigned w = d[T::VEC == 4 ? e : e / 2];  // (a bit_cast of d[e] itself always takes the first element)
    if constexpr (T::VEC == 4) return __builtin_bit_cast(float, w);
    else return e & 1 ? T::upper(w) : T::lower(w);
  }
  __device__ __forceinline__ void put(const float* v) {
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if constexpr (T::VEC == 4) d[w] = __builtin_bit_cast(unsigned, v[w]);
      else d[w] = (unsigned)T::down(v[2 * w]) | (unsigned)T::down(v[2 * w + 1]) << 16;
    }
  }
};
// at any element-aligned address (gfx950 loads and stores 16 bytes unaligned); `at` counts bytes, so that the
// address is a scalar base and one 32-bit lane offset
template <class T>
__device__ __forceinline__ Vec<T> load_vec(const typename T::S* base, unsigned at) {
  return Vec<T>{*(const u32x4_any*)((const char*)base + at)};
}
template <class T, bool PAST = false>
__device__ __forceinline__ void store_vec(typename T::S* base, unsigned at, const Vec<T>& v) {
  if (PAST) __builtin_nontemporal_store(v.d, (u32x4_any*)((char*)base + at));
  else *(u32x4_any*)((char*)base + at) = v.d;
}
template <class S>
__device__ __forceinline__ S& at_byte(S* base, unsigned at) { return *(S*)((char*)base + at); }
template <class S>
__device__ __forceinline__ const S& at_byte(const S* base, unsigned at) { return *(const S*)((const char*)base + at); }
// the first `n` of a vector's elements (n < VEC; the others repeat the last one, nothing behind it is read)
template <class T>
__device__ __forceinline__ Vec<T> load_some(const typename T::S* base, unsigned at, int n) {
  using S = typename T::S;
  Vec<T> r;
  S e[T::VEC];
#pragma unroll
  for (int i = 0; i < T::VEC; ++i) e[i] = n > 0 ? at_byte(base, at + (unsigned)(min(i, n - 1) * (int)sizeof(S))) : S(0);
  __builtin_memcpy(&r.d, e, 16);
  return r;
}
template <class T>
__device__ __forceinline__ void store_some(typename T::S* base, unsigned at, int n, const Vec<T>& v) {
  using S = typename T::S;
  S e[T::VEC];
  __builtin_memcpy(e, &v.d, 16);
#pragma unroll
  for (int i = 0; i < T::VEC; ++i)
    if (i < n) at_byte(base, at + (unsigned)(i * (int)sizeof(S))) = e[i];
}

// v_max_f32 / v_min_f32 without the canonicalisation the compiler puts before fmaxf of loaded values; a quiet
// NaN operand gives the other one (the sum carries the NaN)
__device__ __forceinline__ float vmax(float a, float b) {
  float r;
  asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}
__device__ __forceinline__ float vmin(float a, float b) {
  float r;
  asm("v_min_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}
__device__ __forceinline__ float vmax3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
__device__ __forceinline__ float vmin3(float a, float b, float c) {
  float r;
  asm("v_min3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
// Which way the logits count (the same in every lane)
struct Side {
  bool neg;
  float c;     // scale * log2 e
  float sign;  // of the scale
  __device__ __forceinline__ float far() const { return neg ? kInf : -kInf; }
  __device__ __forceinline__ float best(float a, float b) const { return neg ? vmin(a, b) : vmax(a, b); }
  template <int N>
  __device__ __forceinline__ float best_of(const float (&v)[N]) const {
    float m;
    if (neg) {
      m = vmin(v[0], v[1]);
#pragma unroll
      for (int i = 2; i < N; i += 2) m = vmin3(m, v[i], v[i + 1]);
    } else {
      m = vmax(v[0], v[1]);
#pragma unroll
      for (int i = 2; i < N; i += 2) m = vmax3(m, v[i], v[i + 1]);
    }
    return m;
  }
};
__device__ __forceinline__ float exp2_(float t) { return __builtin_amdgcn_exp2f(t); }
// e^x: the rounding of x log2 e is put right to first order, so the error stays at two steps for any x.  (For
// |x| so large that the correction is infinite or NaN the power is 0, inf or NaN by itself.)
__device__ __forceinline__ float exp_(float x) {
  const float t = x * kLog2e, p = exp2_(t);
  const float r = fmaf(x, kLog2e, -t) + x * kLog2eRest;
  return p == 0.f || p == kInf ? p : fmaf(p, r * kLn2, p);
}

// Hides where a value comes from, so that addresses are formed from it where they are used, not kept in a
// register pair each across the loop
__device__ __forceinline__ unsigned fresh(unsigned v) {
  asm volatile("" : "+v"(v));
  return v;
}
__device__ __forceinline__ int64_t fresh_uniform(int64_t v) {
  asm volatile("" : "+s"(v));
  return v;
}
// a plane's start, to be used with a 32-bit lane offset (without this the compiler adds the lane's offset to
// the tensor's start once and then 64 bits to that for every plane, in vector registers)
template <class S>
using Global = __attribute__((address_space(1))) S*;
template <class P>
__device__ __forceinline__ P scalar_base(P p) {
  asm volatile("" : "+s"(p));
  return p;
}
template <class S>
using GlobalBytes = std::conditional_t<std::is_const_v<S>, const __attribute__((address_space(1))) char*,
                                       __attribute__((address_space(1))) char*>;
template <class S>
__device__ __forceinline__ Global<S> at_byte(Global<S> base, unsigned at) {
  return (Global<S>)((GlobalBytes<S>)base + at);
}
// keeps a branch that is hardly ever taken a branch
__device__ __forceinline__ void rare() { asm volatile(""); }
// Keeps the compiler from computing all 32 intermediate values at once (it would spill): nothing moves over
// every eighth value
__device__ __forceinline__ void fence_schedule(int i) {
  if (i % 8 == 7) __builtin_amdgcn_sched_barrier(0);
}

// ---- running soft-max ------------------------------------------------------------------------
struct Acc {
  float m, s, w;
};
using Stats3 = Acc;  // what the backward pass gets of a row; m is 0 in an empty one
// entropy = ln s - ln2 w / s: both terms are >= 0, nothing cancels
__device__ __forceinline__ float entropy_of(float s, float w, float ln_s) { return s == 0.f ? 0.f : ln_s - kLn2 * w / s; }
__device__ __forceinline__ Acc acc_empty(const Side& z) { return Acc{z.far(), 0.f, 0.f}; }

// top: best_of(v); nothing possible stands behind the n-th value
template <bool ENT, int N>
__device__ __forceinline__ void absorb(Acc& a, const float (&v)[N], int n, float top, const Side& z) {
  const float m = z.best(a.m, top);
  const float b = m == z.far() ? 0.f : m;
  const float d = fmaxf((a.m - b) * z.c, kFloor), al = exp2_(d);
  if (ENT) a.w = al * fmaf(a.s, d, a.w);
  a.s *= al;
#pragma unroll
  for (int i = 0; i < N; i += 8) {
    if (i >= n) break;
    float t[8], e[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) t[k] = (v[i + k] - b) * z.c;
#pragma unroll
    for (int k = 0; k < 8; ++k) e[k] = exp2_(t[k]);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      a.s += e[k];
      if (ENT) a.w = fmaf(e[k], vmax(t[k], kFloor), a.w);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  a.m = m;
}
__device__ __forceinline__ Acc acc_join(const Acc& a, const Acc& b, const Side& z) {
  const float m = z.best(a.m, b.m), o = m == z.far() ? 0.f : m;
  const float da = fmaxf((a.m - o) * z.c, kFloor), db = fmaxf((b.m - o) * z.c, kFloor);
  const float ea = exp2_(da), eb = exp2_(db);
  return Acc{m, a.s * ea + b.s * eb, ea * fmaf(a.s, da, a.w) + eb * fmaf(b.s, db, b.w)};
}
__device__ __forceinline__ float shfl_xor(float v, int mask) { return __shfl_xor(v, mask, 64); }
__device__ __forceinline__ Acc acc_wave(Acc a, const Side& z) {
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) {
    Acc b{shfl_xor(a.m, k), shfl_xor(a.s, k), shfl_xor(a.w, k)};
    // both lanes of a pair evaluate the same expression (lower lane's sums first): one result everywhere
    a = (threadIdx.x & k) ? acc_join(b, a, z) : acc_join(a, b, z);
  }
  return a;
}
__device__ __forceinline__ float wave_best_all(float v, const Side& z) {
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) v = z.best(v, shfl_xor(v, k));
  return v;
}
__device__ __forceinline__ float wave_sum_all(float v) {
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) v += shfl_xor(v, k);
  return v;
}

// (x - m) scale + add, also where x - m alone leaves float32's range (halving is exact)
__device__ __forceinline__ float scaled_difference(float x, float m, float scale, float add) {
  return fmaf(0.5f * x - 0.5f * m, 2.f * scale, add);
}
// log p of a class of value x in a row of (m, ln s): -inf for an impossible class, also where the whole row
// is impossible (ln s = -inf); NaN where the row holds NaN or z = +inf
// (in base e: in base 2 the log-probability of a class at float32's lowest value would overflow)
__device__ __forceinline__ float log_p(float x, float m, float ln_s, float scale) {
  return (x * scale == -kInf && fabsf(x) == kInf && ln_s == ln_s) ? -kInf : scaled_difference(x, m, scale, -ln_s);
}

// ---- order keys --------------------------------------------------------------------------------
// 64-bit whole number that orders classes by value, then by lowest index; NaN above everything.  No key is all ones
// (NaN at class 0 comes nearest) or 0: a search may begin above or below every key.
constexpr unsigned kLowestFirst = 0xfffffffeu;
__device__ __forceinline__ unsigned long long key_u64(float v, int idx) {
  unsigned b = __builtin_bit_cast(unsigned, v + 0.f);
  b = v != v ? 0xffffffffu : (b ^ ((unsigned)((int)b >> 31) | 0x80000000u));
  return ((unsigned long long)b << 32) | (kLowestFirst - (unsigned)idx);
}
__device__ __forceinline__ float key_value(unsigned long long k) {
  const unsigned b = (unsigned)(k >> 32);
  if (b == 0xffffffffu) return __builtin_nanf("");
  return __builtin_bit_cast(float, (b >> 31) ? (b ^ 0x80000000u) : ~b);
}
__device__ __forceinline__ int key_index(unsigned long long k) { return (int)(kLowestFirst - (unsigned)k); }

// Keys of the lists that are kept in registers: numbers of the same order.  A NaN has to be positive (order_nans()).
//
// As a float64, a comparator is one v_max_f64 and one v_min_f64: the upper word is the value as it is (the bits
// of a float32 read as the upper half of a float64 keep their order, and infinities stay finite numbers
// there), the lower word the index, complemented for positive values.
struct Wide {
  using Key = double;
  static constexpr double kNone = __builtin_bit_cast(double, 0xff90000000000000ull);  // below -inf of any index
  static __device__ __forceinline__ Key of(float v, float sign, int idx) {  // of sign * v
    const unsigned hi = __builtin_bit_cast(unsigned, fmaf(v, sign, 0.f));  // -0 counts as 0
    const unsigned lo = (unsigned)((int)hi >> 31) ^ ~(unsigned)idx;
    return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
  }
  static __device__ __forceinline__ float value(Key k) {
    return __builtin_bit_cast(float, (unsigned)(__builtin_bit_cast(unsigned long long, k) >> 32));
  }
  static __device__ __forceinline__ int index(Key k) {
    const unsigned long long b = __builtin_bit_cast(unsigned long long, k);
    return (int)((unsigned)((long long)b >> 63) ^ ~(unsigned)b);
  }
  static __device__ __forceinline__ Key larger(Key a, Key b) {
    Key r;
    asm("v_max_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
  }
  static __device__ __forceinline__ Key smaller(Key a, Key b) {
    Key r;
    asm("v_min_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
  }
};
// Values of 16-bit types leave the lower 13 bits of their float32 empty (bfloat16 16 bits): with fewer than 2^13
// classes the index goes there: a comparator costs half of one on float64, and twice as many entries fit the
// registers (192 classes of 2 x 192 x 640 pixels bf16: the top 16 in 47 us instead of 65, 20 in 60 instead of 110,
// 8 in 40 instead of 41; 27 without a list, 19.8 for reading it).
struct Narrow {
  using Key = int;
  static constexpr int kClasses = 1 << 13, kValue = 0x7fffffff & ~(kClasses - 1);
  static constexpr int kNone = (int)0x80000000;  // below -inf of any index
  static __device__ __forceinline__ Key of(float v, float sign, int idx) {
    const int b = __builtin_bit_cast(int, fmaf(v, sign, 0.f));
    return (b ^ (b >> 31 & kValue)) + (kClasses - 1 - idx);
  }
  static __device__ __forceinline__ float value(Key k) {
    const int b = k & ~(kClasses - 1);
    return __builtin_bit_cast(float, b ^ (b >> 31 & kValue));
  }
  static __device__ __forceinline__ int index(Key k) { return kClasses - 1 - (k & (kClasses - 1)); }
  static __device__ __forceinline__ Key larger(Key a, Key b) { return max(a, b); }
  static __device__ __forceinline__ Key smaller(Key a, Key b) { return min(a, b); }
};
// makes every NaN the positive one (written so that nothing of it is worked out where it is not asked for)
__device__ __forceinline__ void order_nans(float (&v)[32]) {
#pragma unroll
  for (int u = 0; u < 32; ++u)
    asm volatile("v_cmp_u_f32 vcc, %0, %0\n\ts_nop 1\n\tv_cndmask_b32 %0, %0, %1, vcc"
                 : "+v"(v[u]) : "v"(__builtin_nanf("")) : "vcc");
}
template <class P>
__device__ __forceinline__ void order2(typename P::Key& hi, typename P::Key& lo) {
  const typename P::Key a = P::larger(hi, lo), b = P::smaller(hi, lo);
  hi = a;
  lo = b;
}
// descending sort of K keys in registers: Batcher's odd-even merge network
template <class P, int K>
__device__ __forceinline__ void sort_desc(typename P::Key (&a)[K]) {
#pragma unroll
  for (int p = 1; p < K; p <<= 1)
#pragma unroll
    for (int k = p; k >= 1; k >>= 1)
#pragma unroll
      for (int j = k % p; j + k < K; j += 2 * k)
#pragma unroll
        for (int i = 0; i < k; ++i)
          if (i + j + k < K && (i + j) / (2 * p) == (i + j + k) / (2 * p)) order2<P>(a[i + j], a[i + j + k]);
}
// top <- the K largest of two descending lists, descending
template <class P, int K>
__device__ __forceinline__ void merge_desc(typename P::Key (&top)[K], const typename P::Key (&n)[K]) {
#pragma unroll
  for (int i = 0; i < K; ++i) top[i] = P::larger(top[i], n[K - 1 - i]);
#pragma unroll
  for (int h = K / 2; h >= 1; h >>= 1)
#pragma unroll
    for (int i = 0; i < K; ++i)
      if ((i & h) == 0) order2<P>(top[i], top[i + h]);
}
// ---- problem -----------------------------------------------------------------------------------
struct Prob {
  int64_t outer, inner, rows;  // rows = outer * inner
  int64_t es[3];               // strides of the teacher's list: outer, entry, inner
  int V, k;                    // classes, entries (top or teacher)
  int cpw;                     // tile kernels: classes a wave
  int chunks, chunk;           // row kernels: blocks a row, classes a block
  float scale, c;
  int flags;
  bool past;                   // gradients are stored past the caches (kPastBytes)
};
__device__ __forceinline__ Side side(const Prob& p) {
  const bool neg = __builtin_bit_cast(int, p.scale) < 0;
  return Side{neg, p.c, neg ? -1.f : 1.f};
}
constexpr int kIdx64 = DW_DIST_INDEX64, kRenorm = DW_DIST_RENORMALISE;

__device__ __forceinline__ int64_t load_index(const void* p, int64_t at, int flags) {
  return (flags & kIdx64) ? ((const int64_t*)p)[at] : (int64_t)((const int32_t*)p)[at];
}
__device__ __forceinline__ int valid_index(int64_t i, int V) { return (i >= 0 && i < V) ? (int)i : -1; }
__device__ __forceinline__ float load_teacher(const void* p, int64_t at, int flags) {
  if (flags & DW_DIST_TEACHER_BF16) return BF16::up(((const uint16_t*)p)[at]);
  if (flags & DW_DIST_TEACHER_F16) return F16::up(((const uint16_t*)p)[at]);
  return ((const float*)p)[at];
}

// N entries of a list from the e0-th on; -1 for what is padding or behind the k-th.  All loads are issued
// before the first is looked at.
template <int N>
__device__ __forceinline__ void load_indices(const Prob& p, const void* index, int64_t t0, int e0, int (&idx)[N]) {
  int64_t at[N];
#pragma unroll
  for (int i = 0; i < N; ++i) at[i] = t0 + min(e0 + i, p.k - 1) * p.es[1];
  if (p.flags & kIdx64) {
    int64_t v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = ((const int64_t*)index)[at[i]];
#pragma unroll
    for (int i = 0; i < N; ++i) idx[i] = e0 + i < p.k ? valid_index(v[i], p.V) : -1;
  } else {
    int v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = ((const int32_t*)index)[at[i]];
#pragma unroll
    for (int i = 0; i < N; ++i) idx[i] = e0 + i < p.k ? valid_index(v[i], p.V) : -1;
  }
}
template <int N>
__device__ __forceinline__ void load_teachers(const Prob& p, const void* teacher, int64_t t0, int e0, float (&l)[N]) {
  int64_t at[N];
#pragma unroll
  for (int i = 0; i < N; ++i) at[i] = t0 + min(e0 + i, p.k - 1) * p.es[1];
  if (p.flags & (DW_DIST_TEACHER_BF16 | DW_DIST_TEACHER_F16)) {
    uint16_t v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = ((const uint16_t*)teacher)[at[i]];
#pragma unroll
    for (int i = 0; i < N; ++i) l[i] = (p.flags & DW_DIST_TEACHER_BF16) ? BF16::up(v[i]) : F16::up(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) l[i] = ((const float*)teacher)[at[i]];
  }
}

// ---- tile kernels: where the 64 rows of a block are, and how their classes come in -----------------
enum Layout { kPlanes, kTurned, kFlat };
struct Place {
  int64_t row;    // this lane's row (planes: the last pixel again behind the end)
  int64_t o, i;   // its outer and inner index
  int64_t first;  // first row (LAST) or first pixel (planes) of the block
  int lane, wave;
  int skip;       // LAST: so many of the block's first rows belong to the block before
  bool live;      // this lane's row is the block's to write
};
// Backward passes take the blocks from the last to the first: what the forward pass read last is what the
// last-level cache still holds.
__device__ __forceinline__ unsigned block_from_end() { return gridDim.x - 1 - blockIdx.x; }
// Blocks go round the chip's eight dies; this gives each die one stretch of the tiles, so that the two halves of a
// line that lies in two tiles meet in one die's cache (256 x 375 x 1242 bf16 forward 99 -> 89 us, backward
// 138 -> 109; the same where planes are whole lines).
__device__ __forceinline__ unsigned on_one_die(unsigned block) {
  const unsigned die = block % 8, each = gridDim.x / 8, more = gridDim.x % 8;
  return die * each + min(die, more) + block / 8;
}
template <bool LAST>
__device__ __forceinline__ Place place(const Prob& p, unsigned block) {
  if (!LAST) block = on_one_die(block);
  Place q;
  q.lane = threadIdx.x & 63;
  q.wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (LAST) {
    // the last block starts 64 rows before the end (there are at least 64) and leaves the ones before its
    // own to their block
    const int64_t own = (int64_t)block * 64;
    q.first = own + 64 <= p.rows ? own : p.rows - 64;
    q.skip = (int)(own - q.first);
    q.row = q.first + q.lane;
    q.live = q.lane >= q.skip;
    if (p.inner == 1) {
      q.o = q.row;
      q.i = 0;
    } else if (p.inner >= 64) {  // the block's rows lie in one or two outer ones: one division, a scalar one
      q.o = q.first / p.inner;
      q.i = q.first - q.o * p.inner + q.lane;
      if (q.i >= p.inner) {
        q.i -= p.inner;
        q.o += 1;
      }
    } else {
      q.o = q.row / p.inner;
      q.i = q.row - q.o * p.inner;
    }
  } else {
    const unsigned tiles = (unsigned)((p.inner + 63) / 64);
    q.o = block / tiles;
    q.first = (int64_t)(block - (unsigned)q.o * tiles) * 64;
    q.i = q.first + q.lane;
    q.live = q.i < p.inner;
    if (!q.live) q.i = p.inner - 1;
    q.row = q.o * p.inner + q.i;
  }
  return q;
}
template <bool LAST>
__device__ __forceinline__ int64_t element(const Prob& p, const Place& q, int j) {
  return LAST ? q.row * p.V + j : (q.o * p.V + j) * p.inner + q.i;
}

__device__ __forceinline__ void wave_sync() {  // orders this wave's LDS accesses
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

constexpr int kSegBytes = 128;                 // of every row in a stage
constexpr int kRowBytes = kSegBytes + 16;      // LDS distance of two rows: spreads the 16-byte reads over the banks
constexpr int kStageBytes = 64 * kRowBytes;

// classes a wave takes at a time
template <class T, int L>
constexpr int stage_classes() { return L == kTurned ? kSegBytes / (int)sizeof(typename T::S) : 32; }

// The next stage on its way: loads are issued a stage ahead, while the one before is worked on.
template <class T, int L>
struct Feed;
template <class T>
struct Feed<T, kTurned> {  // 64 row segments of classes [c0, c0 + n), 8 lanes a row
  static constexpr int PER = kSegBytes / 16;
  Vec<T> v[PER];
  __device__ __forceinline__ void issue(const typename T::S* x, const Prob& p, const Place& q, int c0, int n) {
    using S = typename T::S;
    const int j = q.lane % PER * T::VEC;
    const unsigned at = fresh((unsigned)(q.lane / PER * p.V + j) * (unsigned)sizeof(S));
    int64_t off = q.first * p.V + c0;
    if (n == kSegBytes / (int)sizeof(S)) {
#pragma unroll
      for (int it = 0; it < PER; ++it) {
        v[it] = load_vec<T>(x + off, at);
        off = fresh_uniform(off + (64 / PER) * p.V);
      }
    } else {
#pragma unroll
      for (int it = 0; it < PER; ++it) {
        // what a vector reaches of the next row is read and not used; behind the last row nothing is read
        const int64_t left = (p.rows - q.first - it * (64 / PER) - q.lane / PER) * p.V - c0 - j;
        v[it].d = u32x4{0, 0, 0, 0};
        if (j < n) {
          if (left >= T::VEC) v[it] = load_vec<T>(x + off, at);
          else v[it] = load_some<T>(x + off, at, n - j);
        }
        off = fresh_uniform(off + (64 / PER) * p.V);
      }
    }
  }
  __device__ __forceinline__ void to_lds(const Place& q, char* lds) const {
#pragma unroll
    for (int it = 0; it < PER; ++it)
      *(Vec<T>*)(lds + (it * (64 / PER) + q.lane / PER) * kRowBytes + q.lane % PER * 16) = v[it];
  }
};
template <class T>
struct Feed<T, kPlanes> {  // 32 planes from class c0 on; the planes behind the n-th repeat it
  typename T::S v[32];
  __device__ __forceinline__ void issue(const typename T::S* x, const Prob& p, const Place& q, int c0, int n) {
    using S = typename T::S;
    Global<const S> plane = (Global<const S>)(x + (q.o * p.V + c0) * p.inner + q.first);
    const unsigned at = fresh((unsigned)(q.i - q.first) * (unsigned)sizeof(S));
    if (n == 32) {
#pragma unroll
      for (int u = 0; u < 32; ++u) {
        plane = scalar_base(plane);
        v[u] = *at_byte<const S>(plane, at);
        plane += p.inner;
      }
    } else {
      const int last = (int)fresh_uniform(n) - 1;
#pragma unroll
      for (int u = 0; u < 32; ++u) {
        plane = scalar_base(plane);
        v[u] = *at_byte<const S>(plane, at);
        plane += u < last ? p.inner : 0;
      }
    }
  }
  __device__ __forceinline__ void take(float (&f)[32]) const {
#pragma unroll
    for (int u = 0; u < 32; ++u) f[u] = T::up(v[u]);
  }
};
template <class T>
struct Feed<T, kFlat> {  // all there already
  __device__ __forceinline__ void issue(const typename T::S*, const Prob&, const Place&, int, int) {}
};

// Rows of a flat tile: the 64 rows' bytes as they lie in memory, so that whole lines are read and written whatever the
// rows' length; where rows are whole 16-byte pieces, each with 16 bytes behind it, which spreads them over the banks.
constexpr int kFlatSlack = 128;  // behind the last row: a lane reads 32 classes at a time
__host__ __device__ constexpr bool flat_padded(int row) { return row % 16 == 0 && row > 16; }
__host__ __device__ constexpr int flat_row(int row) { return row + (flat_padded(row) ? 16 : 0); }
__host__ __device__ constexpr int flat_bytes(int row) { return (64 * flat_row(row) + kFlatSlack + 15) / 16 * 16; }
template <class T>
struct FlatTile {
  using S = typename T::S;
  char* lds;
  int row, step, threads;  // bytes of a row in memory, in LDS
  unsigned pieces, inv;    // 16-byte pieces of the tile; 2^32 / pieces of a row, rounded up: exact below 2^16 pieces
  __device__ __forceinline__ FlatTile(const Prob& p, char* smem)
      : lds(smem), row(p.V * (int)sizeof(S)), step(flat_row(row)), threads(blockDim.x), pieces(4u * row),
        inv(flat_padded(row) ? 0xffffffffu / (unsigned)(row / 16) + 1 : 0) {}
  __device__ __forceinline__ u32x4* at(unsigned piece) const {
    return (u32x4*)(lds + 16 * (piece + (flat_padded(row) ? __umulhi(piece, inv) : 0)));
  }
  __device__ __forceinline__ S* lane_row(int lane) const { return (S*)(lds + lane * step); }
  // the whole block; ends with a barrier
  __device__ __forceinline__ void in(const S* x, const Prob& p, const Place& q) const {
    const S* base = x + q.first * p.V;
    for (unsigned c0 = threadIdx.x; c0 < pieces; c0 += 8 * threads) {
      Vec<T> w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const unsigned c = c0 + i * threads;
        if (c < pieces) w[i] = load_vec<T>(base, c * 16);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const unsigned c = c0 + i * threads;
        if (c < pieces) *at(c) = w[i].d;
      }
    }
    __syncthreads();
  }
  // begins with a barrier
  __device__ __forceinline__ void out(S* g, const Prob& p, const Place& q) const {
    __syncthreads();
    S* base = g + q.first * p.V;
    const unsigned skip = (unsigned)(q.skip * row);
    for (unsigned c = threadIdx.x; c < pieces; c += threads) {
      const Vec<T> w{*at(c)};
      if (c * 16 >= skip && p.past) {
        rare();
        store_vec<T, true>(base, c * 16, w);
        rare();
      } else if (c * 16 >= skip) {
        store_vec<T>(base, c * 16, w);
      } else if (c * 16 + 16 > skip) {
        const S* e = (const S*)at(c);
        for (unsigned b = skip; b < c * 16 + 16; b += sizeof(S)) at_byte(base, b) = e[(b - c * 16) / sizeof(S)];
      }
    }
  }
  // 32 classes from c on; what lies behind the row's last is anything
  __device__ __forceinline__ void read(int lane, int c, float (&v)[32]) const {
    const S* r = lane_row(lane) + c;
    if (flat_padded(row)) {
#pragma unroll
      for (int u = 0; u < 32 / T::VEC; ++u) {
        const Vec<T> w{((const u32x4*)r)[u]};
#pragma unroll
        for (int e = 0; e < T::VEC; ++e) v[u * T::VEC + e] = w.get(e);
      }
    } else {
#pragma unroll
      for (int u = 0; u < 32; ++u) v[u] = T::up(r[u]);
    }
  }
  // n of them (whole pieces, where rows are)
  __device__ __forceinline__ void write(int lane, int c, int n, const float (&v)[32]) const {
    S* r = lane_row(lane) + c;
    if (flat_padded(row)) {
#pragma unroll
      for (int u = 0; u < 32 / T::VEC; ++u) {
        Vec<T> w;
        w.put(v + u * T::VEC);
        if (u * T::VEC < n) ((u32x4*)r)[u] = w.d;
      }
    } else if (n == 32) {
#pragma unroll
      for (int u = 0; u < 32; ++u) r[u] = T::down(v[u]);
    } else {
      n = (int)fresh_uniform(n);
#pragma unroll
      for (int u = 0; u < 32; ++u)
        if (u < n) r[u] = T::down(v[u]);
    }
  }
};
template <class T>
__device__ __forceinline__ void stage_out(typename T::S* g, const Prob& p, const Place& q, int c0, int n,
                                          const char* lds) {
  using S = typename T::S;
  constexpr int PER = kSegBytes / 16;
  const int j = q.lane % PER * T::VEC;
  const unsigned at = fresh((unsigned)(q.lane / PER * p.V + j) * (unsigned)sizeof(S));
  int64_t off = q.first * p.V + c0;
#pragma unroll
  for (int it = 0; it < PER; ++it) {
    const int r = it * (64 / PER) + q.lane / PER;
    if (r >= q.skip) {
      const Vec<T> v = *(const Vec<T>*)(lds + r * kRowBytes + q.lane % PER * 16);
      if (j + T::VEC <= n) store_vec<T>(g + off, at, v);
      else store_some<T>(g + off, at, n - j, v);
    }
    off = fresh_uniform(off + (64 / PER) * p.V);
  }
}
// 32 classes of this lane's row from the stage, from class h of the segment on
template <class T>
__device__ __forceinline__ void stage_read(const char* lds, int lane, int h, float (&v)[32]) {
#pragma unroll
  for (int u = 0; u < 32 / T::VEC; ++u) {
    const Vec<T> w = *(const Vec<T>*)(lds + lane * kRowBytes + h * (int)sizeof(typename T::S) + u * 16);
#pragma unroll
    for (int e = 0; e < T::VEC; ++e) v[u * T::VEC + e] = w.get(e);
  }
}
template <class T>
__device__ __forceinline__ void stage_write(char* lds, int lane, int h, const float (&v)[32]) {
#pragma unroll
  for (int u = 0; u < 32 / T::VEC; ++u) {
    Vec<T> w;
    w.put(v + u * T::VEC);
    *(Vec<T>*)(lds + lane * kRowBytes + h * (int)sizeof(typename T::S) + u * 16) = w;
  }
}
template <class T>
__device__ __forceinline__ void planes_out(typename T::S* g, const Prob& p, const Place& q, int c0, int n,
                                           const typename T::S (&v)[32]) {
  using S = typename T::S;
  Global<S> plane = (Global<S>)(g + (q.o * p.V + c0) * p.inner + q.first);
  const unsigned at = fresh((unsigned)(q.i - q.first) * (unsigned)sizeof(S));
  if (!q.live) return;
  if (n == 32 && p.past) {
#pragma unroll
    for (int u = 0; u < 32; ++u) {
      plane = scalar_base(plane);
      __builtin_nontemporal_store(v[u], at_byte<S>(plane, at));
      plane += p.inner;
    }
  } else if (n == 32) {
#pragma unroll
    for (int u = 0; u < 32; ++u) {
      plane = scalar_base(plane);
      *at_byte<S>(plane, at) = v[u];
      plane += p.inner;
    }
  } else {
    const int m = (int)fresh_uniform(n);
#pragma unroll
    for (int u = 0; u < 32; ++u) {
      plane = scalar_base(plane);
      if (u < m) *at_byte<S>(plane, at) = v[u];
      plane += p.inner;
    }
  }
}
// nothing possible behind the n-th class
__device__ __forceinline__ void settle(float (&v)[32], float far, int n) {
  if (n < 32) {
    n = (int)fresh_uniform(n);
#pragma unroll
    for (int u = 0; u < 32; ++u) v[u] = u < n ? v[u] : far;
  }
}

// ---- log-probabilities, forward, tile ---------------------------------------------------------------
// A thread a row keeps the whole soft-max in its own registers: a block a row, as in the row kernels, would spend a
// reduction over 64 lanes on every few hundred classes.  The waves of a block split the classes where there are
// too few rows to fill the chip, and join through LDS.  Loads of the next 32 classes are issued before the ones at
// hand are worked on.  12 x 64 x 96 x 320 bf16 (47 MB): 15.2 us, 3.1 TB/s, vector instructions in
// 63 % of the busy cycles, so neither alone is the bound; 1 x 256 x 256 x 512 f32 with
// the top 8 (134 MB): 34 us, 4.0 TB/s; 4 x 193 x 96 x 320 f16, classes last (47 MB): 17.8 us.
// K: top classes kept in registers as keys of kind P (0: none).  More than K wanted: further passes over the data,
// each for the next K below the last key of the pass before.
// Turning rows and keeping their lists takes up to 180 registers: those blocks have at most 8 waves, so that they get
// them (192 classes of 2 x 192 x 320 pixels f32: the top 8 in 31 us, 41 with 128 registers; bf16 the same either way).
constexpr int list_waves(bool last, bool list) { return last && list ? 8 : 16; }
template <class T, int L, class P, int K>
__global__ __launch_bounds__(64 * list_waves(L != kPlanes, K > 0))
void lp_tile_fwd(Prob p, const typename T::S* __restrict__ x, const void* __restrict__ index,
                            float* __restrict__ log_prob, float* __restrict__ entropy, float* __restrict__ top_lp,
                            int32_t* __restrict__ top_idx, Stats3* __restrict__ stats) {
  extern __shared__ __align__(16) char smem[];
  constexpr bool LAST = L != kPlanes;
  const Place q = place<LAST>(p, blockIdx.x);
  const int nw = blockDim.x >> 6;
  char* stage = smem + q.wave * kStageBytes;                       // kTurned only
  const FlatTile<T> tile(p, smem);                                 // kFlat only
  char* joint = smem + (L == kTurned ? nw * kStageBytes : L == kFlat ? flat_bytes(tile.row) : 0);
  float* red = (float*)joint;                                      // [3][nw][64]
  using Key = typename P::Key;
  Key* keys = (Key*)(joint + 3 * nw * 64 * sizeof(float));         // [nw][K][64]
  constexpr int CH = stage_classes<T, L>();
  const Side z = side(p);
  const int c_lo = q.wave * p.cpw, c_hi = min(p.V, c_lo + p.cpw);

  // the given class, on its way while the classes are read
  const int64_t given_raw = index ? load_index(index, q.row, p.flags) : -1;
  Feed<T, L> feed;
  if (c_lo < c_hi) feed.issue(x, p, q, c_lo, min(CH, c_hi - c_lo));
  const int given = valid_index(given_raw, p.V);
  const typename T::S x_given = given >= 0 ? x[element<LAST>(p, q, given)] : typename T::S(0);

  if constexpr (L == kFlat) tile.in(x, p, q);
  Acc a = acc_empty(z);
  Key limit = P::kNone;
  float ln_s = 0.f, base = 0.f;
  for (int done = 0; done == 0 || done < p.k; done += (K ? K : 1)) {
    Key top[K ? K : 1];
#pragma unroll
    for (int i = 0; i < K; ++i) top[i] = P::kNone;
    if (done > 0 && c_lo < c_hi) feed.issue(x, p, q, c_lo, min(CH, c_hi - c_lo));
    for (int c0 = c_lo; c0 < c_hi; c0 += CH) {
      const int n = min(CH, c_hi - c0), ahead = min(CH, c_hi - c0 - CH);
      float v[32];
      if constexpr (L == kTurned) {
        wave_sync();
        feed.to_lds(q, stage);
        wave_sync();
      } else if constexpr (L == kPlanes) {
        feed.take(v);
      }
      if (ahead > 0) feed.issue(x, p, q, c0 + CH, ahead);
      for (int h = 0; h < n; h += 32) {
        if constexpr (L == kTurned) stage_read<T>(stage, q.lane, h, v);
        if constexpr (L == kFlat) tile.read(q.lane, c0 + h, v);
        settle(v, z.far(), n - h);
        if (done == 0) absorb<true>(a, v, n - h, z.best_of(v), z);
        if constexpr (K > 0) {
          if (__any(a.s != a.s)) order_nans(v);  // NaN or +inf in some row
#pragma unroll
          for (int g = 0; g < 32; g += K) {
            Key nk[K];
#pragma unroll
            for (int i = 0; i < K; ++i) nk[i] = P::of(v[g + i], z.sign, c0 + h + g + i);  // (a wave's share is whole
            // steps of 32, or ends with the row: what settle() filled up has numbers from V on, behind every class)
            if (done > 0) {
#pragma unroll
              for (int i = 0; i < K; ++i) nk[i] = nk[i] < limit ? nk[i] : P::kNone;
            }
            sort_desc<P, K>(nk);
            merge_desc<P, K>(top, nk);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      }
    }
    if (nw > 1) {
      if (done == 0) {
        red[(0 * nw + q.wave) * 64 + q.lane] = a.m;
        red[(1 * nw + q.wave) * 64 + q.lane] = a.s;
        red[(2 * nw + q.wave) * 64 + q.lane] = a.w;
      }
#pragma unroll
      for (int i = 0; i < K; ++i) keys[(q.wave * K + i) * 64 + q.lane] = top[i];
      __syncthreads();
      // every wave joins everything (the further passes need the limit): same order, same result
      if (done == 0) {
        a = Acc{red[q.lane], red[nw * 64 + q.lane], red[2 * nw * 64 + q.lane]};
        for (int w = 1; w < nw; ++w)
          a = acc_join(a, Acc{red[w * 64 + q.lane], red[(nw + w) * 64 + q.lane], red[(2 * nw + w) * 64 + q.lane]}, z);
      }
      if constexpr (K > 0) {
#pragma unroll
        for (int i = 0; i < K; ++i) top[i] = keys[i * 64 + q.lane];
        for (int w = 1; w < nw; ++w) {
          Key other[K];
#pragma unroll
          for (int i = 0; i < K; ++i) other[i] = keys[(w * K + i) * 64 + q.lane];
          merge_desc<P, K>(top, other);
        }
      }
      __syncthreads();
    }
    if (done == 0) {
      base = a.m == z.far() ? 0.f : a.m;
      ln_s = logf(a.s);
      if (q.wave == 0 && q.live) {
        const float lp = given >= 0 ? log_p(T::up(x_given), base, ln_s, p.scale) : 0.f;
        if (log_prob) log_prob[q.row] = lp;
        if (entropy) entropy[q.row] = entropy_of(a.s, a.w, ln_s);
        if (stats) stats[q.row] = Stats3{base, a.s, a.w};
      }
    }
    if constexpr (K > 0) {
      limit = top[K - 1];
      if (q.wave == 0 && q.live) {
#pragma unroll
        for (int i = 0; i < K; ++i) {
          if (done + i < p.k) {
            const float v = P::value(top[i]) * z.sign;
            const int64_t at = LAST ? q.row * p.k + done + i : (q.o * p.k + done + i) * p.inner + q.i;
            top_lp[at] = log_p(v, base, ln_s, p.scale);
            top_idx[at] = P::index(top[i]);
          }
        }
      }
    }
  }
}

// Coefficients of a row's gradient: dx_j = e_j (k0 + k1 t_j) [+ hit at the given class]
struct LpCoef {
  float m, k0, k1, hit;
  int target;
  bool dead;  // nothing comes back (or nothing is left of the row): the gradient is zero whatever the row holds
};
template <bool ENT>
__device__ __forceinline__ LpCoef lp_coef(const Prob& p, int64_t row, const void* index, const Stats3* stats,
                                          const float* g_lp, const float* g_ent) {
  LpCoef r;
  const Stats3 st = stats[row];
  r.target = (index && g_lp) ? valid_index(load_index(index, row, p.flags), p.V) : -1;
  const float gl = r.target >= 0 ? g_lp[row] : 0.f, gh = ENT ? g_ent[row] : 0.f;
  r.m = st.m;
  r.dead = st.s == 0.f || (gl == 0.f && gh == 0.f);
  const float f = p.scale / st.s;
  r.k0 = ENT ? -f * (gl - gh * kLn2 * st.w / st.s) : -f * gl;
  r.k1 = ENT ? -f * gh * kLn2 : 0.f;
  r.hit = gl * p.scale;
  if (r.dead) r.target = -1;
  return r;
}
template <bool ENT>
__device__ __forceinline__ float lp_grad(const LpCoef& r, float v, float c, float add) {
  const float t = (v - r.m) * c, e = exp2_(t);
  return fmaf(e, ENT ? fmaf(vmax(t, kGradFloor), r.k1, r.k0) : r.k0, add);
}

// The rows' sums come from the forward pass, so this is one read and one write: dx_j = e_j (k0 + k1 t_j), and the
// given class on top.  12 x 64 x 96 x 320 bf16 (94 MB): 20.0 us, 4.7 TB/s, what a copy takes.  4 x 193 x 96 x 320 f16,
// classes last (95 MB): 24 us; 28 where its rows of 386 bytes were turned 128 bytes at a time, and the halves of a line,
// written long after each other, reached memory one by one (66 MB written for 47).
template <class T, int L, bool ENT>
__global__ void lp_tile_bwd(Prob p, const typename T::S* __restrict__ x, const void* __restrict__ index,
                            const Stats3* __restrict__ stats, const float* __restrict__ g_lp, const float* __restrict__ g_ent,
                            typename T::S* __restrict__ g) {
  extern __shared__ __align__(16) char smem[];
  constexpr bool LAST = L != kPlanes;
  const Place q = place<LAST>(p, block_from_end());
  char* stage = smem + q.wave * kStageBytes;
  const FlatTile<T> tile(p, smem);  // kFlat only
  const Side z = side(p);
  const int c_lo = q.wave * p.cpw, c_hi = min(p.V, c_lo + p.cpw);
  constexpr int CH = stage_classes<T, L>();
  Feed<T, L> feed;
  if (c_lo < c_hi) feed.issue(x, p, q, c_lo, min(CH, c_hi - c_lo));
  const LpCoef r = lp_coef<ENT>(p, q.row, index, stats, g_lp, g_ent);
  const bool any_dead = __any(r.dead);
  if constexpr (L == kFlat) tile.in(x, p, q);
  for (int c0 = c_lo; c0 < c_hi; c0 += CH) {
    const int n = min(CH, c_hi - c0), ahead = min(CH, c_hi - c0 - CH);
    float v[32];
    if constexpr (L == kTurned) {
      wave_sync();
      feed.to_lds(q, stage);
      wave_sync();
    } else if constexpr (L == kPlanes) {
      feed.take(v);
    }
    if (ahead > 0) feed.issue(x, p, q, c0 + CH, ahead);
    for (int h = 0; h < n; h += 32) {
      if constexpr (L == kTurned) stage_read<T>(stage, q.lane, h, v);
      if constexpr (L == kFlat) tile.read(q.lane, c0 + h, v);
      settle(v, z.far(), n - h);
      const int rel = r.target - c0 - h;
#pragma unroll
      for (int u = 0; u < 32; ++u) {
        v[u] = lp_grad<ENT>(r, v[u], p.c, rel == u ? r.hit : 0.f);
        fence_schedule(u);
      }
      if (any_dead) {
#pragma unroll
        for (int u = 0; u < 32; ++u) v[u] = r.dead ? 0.f : v[u];
      }
      if constexpr (L == kTurned) {
        stage_write<T>(stage, q.lane, h, v);
      } else if constexpr (L == kFlat) {
        tile.write(q.lane, c0, n, v);
      } else {
        typename T::S raw[32];
#pragma unroll
        for (int u = 0; u < 32; ++u) raw[u] = T::down(v[u]);
        planes_out<T>(g, p, q, c0, n, raw);
      }
    }
    if constexpr (L == kTurned) {
      wave_sync();
      stage_out<T>(g, p, q, c0, n, stage);
    }
  }
  if constexpr (L == kFlat) tile.out(g, p, q);
}

// ---- distillation: what both families share ---------------------------------------------------------
// Everything the loss and its gradient need of a row, from the student's sums.
//   rest (m_r, s_r): running soft-max of the unlisted classes; all (b, s): of every class
//   mass = sum q + r.  dx_j: unlisted e_r coef, listed e_b member - q  (times upstream gradient and scale)
struct RowSums {
  float m_r, s_r, b, s, ln_s;
};
__device__ __forceinline__ float rest_term(const RowSums& r, float scale, float rr) {
  // log of the unlisted classes' probability
  const float lp = scaled_difference(r.m_r, r.b, scale, logf(r.s_r) - r.ln_s);
  return rr > 0.f ? rr * (logf(rr) - lp) : 0.f;
}
__device__ __forceinline__ float4 distill_stats(const RowSums& r, float c, float mass, float rr, bool alive) {
  float4 st = make_float4(0.f, 0.f, r.b, 0.f);
  if (!alive || r.s == 0.f) return st;
  if (r.s_r != 0.f) {
    st.x = r.m_r;
    st.y = mass * exp2_((r.m_r - r.b) * c) / r.s - rr / r.s_r;
  } else {
    st.y = fmaf(0.f, r.s, 0.f * mass);  // 0 for classes that are all impossible; NaN where a listed class or the list holds one
  }
  st.w = mass / r.s;
  return st;
}

// Column of this lane's row inside the stage: planes [class][64], or the row's own bytes.  What a
// lane does for a listed class that is not in the stage goes to a place of its own.
template <class T, int L>
struct Column {
  using S = typename T::S;
  using M = T;
  S *first, *nowhere;
  __device__ __forceinline__ Column(char* stage, const FlatTile<T>& tile, int c_lo, int wave, int lane) {
    if (L == kPlanes) {
      first = (S*)stage + lane;
      nowhere = first + 32 * 64;
    } else if (L == kTurned) {
      first = (S*)(stage + lane * kRowBytes);
      nowhere = first + kSegBytes / (int)sizeof(S);
    } else {
      first = tile.lane_row(lane) + c_lo;
      nowhere = (S*)(tile.lds + flat_bytes(tile.row)) + wave * 64 + lane;
    }
  }
  __device__ __forceinline__ S* at(int u) const { return first + (L == kPlanes ? u * 64 : u); }
  __device__ __forceinline__ S* at(bool hit, int u) const { return hit ? at(u) : nowhere; }
};
// LDS of the classes: a stage a wave, or the flat tile of the block and the lanes' places of their own
__host__ __device__ constexpr int distill_stage_bytes(int layout, int esize) {
  return layout == kTurned ? kStageBytes : layout == kPlanes ? 33 * 64 * esize : 0;
}
__host__ __device__ inline size_t distill_stages(int layout, int nw, int V, int esize) {
  return layout == kFlat ? flat_bytes(V * esize) + (size_t)nw * 64 * 4 : nw * (size_t)distill_stage_bytes(layout, esize);
}
constexpr int kGroup = 8;  // entries handled at once: their LDS accesses overlap
__host__ __device__ constexpr int padded(int k) { return (k + kGroup - 1) / kGroup * kGroup; }
// LDS of a block besides the stages: columns of 64 lanes, of list entries and of the waves' sums
__host__ __device__ constexpr size_t distill_lds(int nw, int k, bool backward) {
  return (size_t)256 * (padded(k) * (backward ? 3 : 2) + 1 + (backward || nw == 1 ? 0 : 2 * nw));
}

template <class S>
__device__ __forceinline__ void read_group(const S* column, int e0, S (&v)[kGroup]) {
#pragma unroll
  for (int i = 0; i < kGroup; ++i) v[i] = column[(e0 + i) * 64];
}
// Natural log of what the listed values' exponentials sum to (0 where that is nothing): the shift that
// makes log-probabilities of them.  group(e0, l) gives eight of the values, -inf for padding.
template <class G>
__device__ __forceinline__ float list_shift(int KP, G group) {
  float tm = -kInf, ts = 0.f;  // fmaxf drops a NaN; the sum brings it back
  for (int e0 = 0; e0 < KP; e0 += kGroup) {
    float l[kGroup];
    group(e0, l);
#pragma unroll
    for (int i = 0; i < kGroup; ++i) tm = fmaxf(tm, l[i]);
  }
  if (tm == -kInf) tm = 0.f;
  for (int e0 = 0; e0 < KP; e0 += kGroup) {
    float l[kGroup];
    group(e0, l);
#pragma unroll
    for (int i = 0; i < kGroup; ++i) ts += exp_(l[i] - tm);
  }
  return ts == 0.f ? 0.f : tm + logf(ts);
}

// The first entry before e of the same class, or e.  Asked only where a listed class was found impossible:
// masked, or taken out for an earlier entry.
__device__ __forceinline__ int listed_before(const int* idx, int e) {
  const int mine = idx[e * 64];
  for (int k = 0; k < e; ++k)
    if (idx[k * 64] == mine) return k;
  return e;
}

// Reads the listed classes of the stage [c0, c0 + n) out of the lane's column and leaves `far` in their
// places (so a class listed twice reads `far` the second time); f(e, hit, value) gets what was read.
template <class C, class F>
__device__ __forceinline__ void take_listed(const C& col, const int* idx, int K, int c0, int n, float far, F f) {
  for (int e0 = 0; e0 < K; e0 += kGroup) {
    float old[kGroup];
    bool hit[kGroup];
#pragma unroll
    for (int i = 0; i < kGroup; ++i) {
      const int rel = idx[(e0 + i) * 64] - c0;
      hit[i] = (unsigned)rel < (unsigned)n;
      typename C::S* at = col.at(hit[i], rel);
      old[i] = C::M::up(*at);
      *at = C::M::down(far);
    }
#pragma unroll
    for (int i = 0; i < kGroup; ++i) f(e0 + i, hit[i], old[i]);
  }
}

// ---- distillation, forward, tile ------------------------------------------------------------------------
// Each listed class is taken out of its column before the running soft-max sees the column, so the
// unlisted classes are summed on their own (1 - sum of the listed would cancel where the list holds
// nearly everything).  The list lies in LDS, a column a lane, so that 64 entries cost no registers; every
// entry is looked up in every stage, eight at a time, which is what long lists cost (192 classes of 2 x 192 x 640
// pixels bf16: 36 us with 8 entries, 49 with 16).  4 x 256 x 192 x 640 bf16, 8 entries (252 + 31 MB): 68 us, 4.2 TB/s;
// 12 x 128 x 96 x 320 f16, classes last (94 + 25 MB): 32 us, 3.7 TB/s; 1 x 64 x 24 x 80: 6.6 us, the launch's latency.
template <class T, int L>
__global__ void ds_tile_fwd(Prob p, const typename T::S* __restrict__ x, const void* __restrict__ teacher,
                            const void* __restrict__ index, float* __restrict__ loss, float4* __restrict__ stats) {
  extern __shared__ __align__(16) char smem[];
  constexpr bool LAST = L != kPlanes;
  const Place q = place<LAST>(p, blockIdx.x);
  const int nw = blockDim.x >> 6, K = p.k, KP = padded(K);
  char* stage = smem + q.wave * distill_stage_bytes(L, sizeof(typename T::S));
  char* rest = smem + distill_stages(L, nw, p.V, sizeof(typename T::S));
  int* idx = (int*)rest + q.lane;                            // [KP][64]
  float* xs = (float*)rest + KP * 64 + q.lane;               // [KP + 1][64]: the listed classes' values
  float* red = (float*)rest + (2 * KP + 1) * 64 + q.lane;    // [2][nw][64], where there are several waves
  constexpr int CH = stage_classes<T, L>();
  const Side z = side(p);
  const int c_lo = q.wave * p.cpw, c_hi = min(p.V, c_lo + p.cpw);
  const Column<T, L> col(stage, FlatTile<T>(p, smem), c_lo, q.wave, q.lane);
  const int64_t t0 = q.o * p.es[0] + q.i * p.es[2];
  Feed<T, L> feed;
  if (c_lo < c_hi) feed.issue(x, p, q, c_lo, min(CH, c_hi - c_lo));

  for (int e0 = q.wave * kGroup; e0 < KP; e0 += nw * kGroup) {
    int i8[kGroup];
    load_indices(p, index, t0, e0, i8);
#pragma unroll
    for (int i = 0; i < kGroup; ++i) {
      idx[(e0 + i) * 64] = i8[i];
      xs[(e0 + i) * 64] = z.far();
    }
  }
  float first[kGroup];  // the teacher's first values: in most lists all of them
  load_teachers(p, teacher, t0, 0, first);
  __syncthreads();
  bool alive = false;
  for (int e0 = 0; e0 < KP; e0 += kGroup) {
    int i8[kGroup];
    read_group(idx, e0, i8);
#pragma unroll
    for (int i = 0; i < kGroup; ++i) alive |= i8[i] >= 0;
  }
  Acc a = acc_empty(z);
  if (__any(alive)) {  // the same in every wave of the block
    for (int c0 = c_lo; c0 < c_hi; c0 += CH) {
      const int n = min(CH, c_hi - c0), ahead = min(CH, c_hi - c0 - CH);
      float v[32];
      wave_sync();
      if constexpr (LAST) {
        feed.to_lds(q, stage);
      } else {
#pragma unroll
        for (int u = 0; u < 32; ++u) *col.at(u) = feed.v[u];
      }
      if (ahead > 0) feed.issue(x, p, q, c0 + CH, ahead);
      wave_sync();
      take_listed(col, idx, K, c0, n, z.far(), [&](int e, bool hit, float old) { xs[(hit ? e : KP) * 64] = old; });
      wave_sync();
      for (int h = 0; h < n; h += 32) {
        if constexpr (LAST) {
          stage_read<T>(stage, q.lane, h, v);
        } else {
#pragma unroll
          for (int u = 0; u < 32; ++u) v[u] = T::up(*col.at(u));
        }
        settle(v, z.far(), n - h);
        absorb<false>(a, v, n - h, z.best_of(v), z);
      }
    }
  }
  if (nw > 1) {
    red[q.wave * 64] = a.m;
    red[(nw + q.wave) * 64] = a.s;
    __syncthreads();
    if (q.wave != 0) return;
    a = Acc{red[0], red[nw * 64], 0.f};
    for (int w = 1; w < nw; ++w) a = acc_join(a, Acc{red[w * 64], red[(nw + w) * 64], 0.f}, z);
  } else {
    wave_sync();
  }
  if (!q.live) return;
  const auto values = [&](int e0, float (&l)[kGroup]) {
    int i8[kGroup];
    read_group(idx, e0, i8);
    if (e0 > 0) load_teachers(p, teacher, t0, e0, l);
#pragma unroll
    for (int i = 0; i < kGroup; ++i) l[i] = i8[i] < 0 ? -kInf : e0 > 0 ? l[i] : first[i];
  };

  RowSums r;
  r.m_r = a.m;
  r.s_r = a.s;
  float m = a.m;
  for (int e0 = 0; e0 < KP; e0 += kGroup) {
    float v[kGroup];
    read_group(xs, e0, v);
#pragma unroll
    for (int i = 0; i < kGroup; ++i) m = z.best(m, v[i]);
  }
  r.b = m == z.far() ? 0.f : m;
  r.s = a.s * exp2_((a.m - r.b) * p.c);
  for (int e0 = 0; e0 < KP; e0 += kGroup) {
    float v[kGroup];
    read_group(xs, e0, v);
#pragma unroll
    for (int i = 0; i < kGroup; ++i) r.s += exp2_((v[i] - r.b) * p.c);
  }
  r.ln_s = logf(r.s);
  const float shift = (p.flags & kRenorm) ? list_shift(KP, values) : 0.f;
  float mass = 0.f, l = 0.f;
  for (int e0 = 0; e0 < KP; e0 += kGroup) {
    float v[kGroup], t[kGroup];
    read_group(xs, e0, v);
    values(e0, t);
#pragma unroll
    for (int i = 0; i < kGroup; ++i) {
      const float lq = t[i] - shift, qe = exp_(lq);  // 0 for padding
      mass += qe;
      if (v[i] == z.far() && idx[(e0 + i) * 64] >= 0) v[i] = xs[listed_before(idx, e0 + i) * 64];
      if (qe != 0.f) l = fmaf(qe, lq - log_p(v[i], r.b, r.ln_s, p.scale), l);
    }
  }
  const float rr = (alive && !(p.flags & kRenorm) && r.s_r != 0.f) ? fmaxf(1.f - mass, 0.f) : 0.f;
  if (rr > 0.f) l += rest_term(r, p.scale, rr);
  loss[q.row] = alive ? l : 0.f;
  if (stats) stats[q.row] = distill_stats(r, p.c, mass + rr, rr, alive);
}

// ---- distillation, backward, tile -------------------------------------------------------------------------
// The stage becomes gradients in place: the listed classes' values are taken out and their gradients worked out in
// the list's columns, the others' are e_j times one factor, and the listed ones are put back last, a class that is
// listed twice with the sum.  4 x 256 x 192 x 640 bf16, 8 entries (503 + 31 MB): 112 us, 4.8 TB/s, what a copy takes.
template <class T, int L>
__global__ void ds_tile_bwd(Prob p, const typename T::S* __restrict__ x, const void* __restrict__ teacher,
                            const void* __restrict__ index, const float4* __restrict__ stats,
                            const float* __restrict__ g_loss, typename T::S* __restrict__ g) {
  extern __shared__ __align__(16) char smem[];
  constexpr bool LAST = L != kPlanes;
  const Place q = place<LAST>(p, block_from_end());
  const int nw = blockDim.x >> 6, K = p.k, KP = padded(K);
  char* stage = smem + q.wave * distill_stage_bytes(L, sizeof(typename T::S));
  char* rest = smem + distill_stages(L, nw, p.V, sizeof(typename T::S));
  int* idx = (int*)rest + q.lane;                    // [KP][64]
  float* gq = (float*)rest + KP * 64 + q.lane;       // [KP][64]: upstream gradient * scale * teacher's probability
  float* gv = (float*)rest + 2 * KP * 64 + q.lane;   // [KP + 1][64]: the listed classes' gradients
  constexpr int CH = stage_classes<T, L>();
  const Side z = side(p);
  const bool renorm = p.flags & kRenorm;
  const int c_lo = q.wave * p.cpw, c_hi = min(p.V, c_lo + p.cpw);
  const FlatTile<T> tile(p, smem);  // kFlat only
  const Column<T, L> col(stage, tile, c_lo, q.wave, q.lane);
  const int64_t t0 = q.o * p.es[0] + q.i * p.es[2];
  const float4 st = stats[q.row];
  const float up = g_loss[q.row];
  const bool dead = up == 0.f || st.w == 0.f;
  const float gs = up * p.scale, rest_f = gs * st.y, member_f = gs * st.w;
  Feed<T, L> feed;
  if (c_lo < c_hi) feed.issue(x, p, q, c_lo, min(CH, c_hi - c_lo));

  for (int e0 = q.wave * kGroup; e0 < KP; e0 += nw * kGroup) {
    int i8[kGroup];
    float l8[kGroup];
    load_indices(p, index, t0, e0, i8);
    load_teachers(p, teacher, t0, e0, l8);
#pragma unroll
    for (int i = 0; i < kGroup; ++i) {
      if (dead) i8[i] = -1;
      idx[(e0 + i) * 64] = i8[i];
      gq[(e0 + i) * 64] = i8[i] < 0 ? (renorm ? -kInf : 0.f) : renorm ? l8[i] : gs * exp_(l8[i]);
    }
  }
  if (renorm) {  // values first, probabilities when their sum is known
    __syncthreads();
    const float shift = list_shift(KP, [&](int e0, float (&l)[kGroup]) { read_group(gq, e0, l); });
    __syncthreads();
    for (int e0 = q.wave * kGroup; e0 < KP; e0 += nw * kGroup) {
#pragma unroll
      for (int i = 0; i < kGroup; ++i) gq[(e0 + i) * 64] = gs * exp_(gq[(e0 + i) * 64] - shift);
    }
  }
  if constexpr (L == kFlat) tile.in(x, p, q);  // with the barrier
  else __syncthreads();
  const bool any_dead = __any(dead);
  // p Q - q of the listed classes; one that is listed again goes on from its earlier entry's value
  const auto take = [&](int c0, int n) {
    take_listed(col, idx, K, c0, n, z.far(), [&](int e, bool hit, float old) {
      float f = fmaf(exp2_((old - st.z) * p.c), member_f, -gq[e * 64]);
      if (hit && old == z.far()) {
        for (int k = 0; k < e; ++k)
          if (idx[k * 64] == idx[e * 64]) f = gv[k * 64] - gq[e * 64];
      }
      gv[(hit ? e : KP) * 64] = f;
    });
    wave_sync();
  };
  const auto put = [&](int c0, int n) {
    wave_sync();
    for (int e0 = 0; e0 < K; e0 += kGroup) {
#pragma unroll
      for (int i = 0; i < kGroup; ++i) {
        const int rel = idx[(e0 + i) * 64] - c0;
        *col.at((unsigned)rel < (unsigned)n, rel) = T::down(gv[(e0 + i) * 64]);
      }
    }
    wave_sync();
  };
  const int mine = max(c_hi - c_lo, 0);
  if constexpr (L == kFlat) take(c_lo, mine);
  for (int c0 = c_lo; c0 < c_hi; c0 += CH) {
    const int n = min(CH, c_hi - c0), ahead = min(CH, c_hi - c0 - CH);
    float v[32];
    if constexpr (L != kFlat) {
      wave_sync();
      if constexpr (L == kTurned) {
        feed.to_lds(q, stage);
      } else {
        feed.take(v);
#pragma unroll
        for (int u = 0; u < 32; ++u) *col.at(u) = feed.v[u];
      }
      if (ahead > 0) feed.issue(x, p, q, c0 + CH, ahead);
      wave_sync();
      take(c0, n);
    }
    for (int h = 0; h < n; h += 32) {
      if constexpr (L == kTurned) stage_read<T>(stage, q.lane, h, v);
      if constexpr (L == kFlat) tile.read(q.lane, c0 + h, v);
      settle(v, z.far(), n - h);
#pragma unroll
      for (int u = 0; u < 32; ++u) {
        v[u] = exp2_((v[u] - st.x) * p.c) * rest_f;
        fence_schedule(u);
      }
      if (any_dead) {
#pragma unroll
        for (int u = 0; u < 32; ++u) v[u] = dead ? 0.f : v[u];
      }
      if constexpr (L == kTurned) {
        stage_write<T>(stage, q.lane, h, v);
      } else if constexpr (L == kFlat) {
        tile.write(q.lane, c0, n, v);
      } else {
#pragma unroll
        for (int u = 0; u < 32; ++u) *col.at(u) = T::down(v[u]);
      }
    }
    if constexpr (L != kFlat) put(c0, n);
    if constexpr (L == kTurned) {
      stage_out<T>(g, p, q, c0, n, stage);
    } else if constexpr (L == kPlanes) {
      typename T::S raw[32];
#pragma unroll
      for (int u = 0; u < 32; ++u) raw[u] = *col.at(u);
      planes_out<T>(g, p, q, c0, n, raw);
    }
  }
  if constexpr (L == kFlat) {
    put(c_lo, mine);
    tile.out(g, p, q);
  }
}

// ---- row kernels -------------------------------------------------------------------------------------------
// A wave takes 2048 neighbouring classes at a time, 32 a lane in 16-byte pieces: every instruction moves 1 KB
// of neighbouring bytes, whatever the row's alignment.  64 threads a block up to 4096 classes, else 256; few rows are split
// until 2048 waves are at work, and joined in a fixed order, so that a result does not depend on which block
// ends first.  Forward, 4096 x 32768 bf16 (268 MB): 56 us, 4.8 TB/s.  Backward (537 MB): 85 us, 6.3 TB/s, part of the logits
// still in the last-level cache.  One row of 32768: 8.4 us with its top 20 and 4.6 for the join, both latency.
constexpr int kWaveTile = 64 * 32;
template <class T>
__device__ __forceinline__ int tile_class(int lane, int u) {  // class of a lane's u-th value inside the wave's tile
  return (u / T::VEC) * 64 * T::VEC + lane * T::VEC + u % T::VEC;
}
template <class T>
__device__ __forceinline__ void row_out(typename T::S* row, int base, int end, int lane, const float (&v)[32]) {
  const unsigned first = fresh((unsigned)(base + lane * T::VEC));
#pragma unroll
  for (int u = 0; u < 32 / T::VEC; ++u) {
    const unsigned j = first + u * 64 * T::VEC;
    const int n = end - (int)j;
    Vec<T> w;
    w.put(v + u * T::VEC);
    if (n >= T::VEC) store_vec<T>(row, j * (unsigned)sizeof(typename T::S), w);
    else store_some<T>(row, j * (unsigned)sizeof(typename T::S), n, w);
  }
}
template <class T, int NT>
__device__ __forceinline__ void row_zero(typename T::S* row, int begin, int end, int lane, int wave) {
  float v[32];
#pragma unroll
  for (int u = 0; u < 32; ++u) v[u] = 0.f;
  for (int base = begin + wave * kWaveTile; base < end; base += NT * 32) row_out<T>(row, base, end, lane, v);
}
template <class T>
__device__ __forceinline__ void row_put(typename T::S* row, int base, int end, int lane, const float (&v)[32], bool past,
                                        bool full) {
  if (!full) {
    rare();
    row_out<T>(row, base, end, lane, v);
    return;
  }
  const unsigned first = fresh((unsigned)(base + lane * T::VEC) * (unsigned)sizeof(typename T::S));
  Vec<T> w[32 / T::VEC];
#pragma unroll
  for (int u = 0; u < 32 / T::VEC; ++u) w[u].put(v + u * T::VEC);
  if (past) {
    rare();  // (keeps the compiler from making one of the two kinds of stores)
#pragma unroll
    for (int u = 0; u < 32 / T::VEC; ++u) store_vec<T, true>(row, first + u * 1024, w[u]);
    rare();
  } else {
#pragma unroll
    for (int u = 0; u < 32 / T::VEC; ++u) store_vec<T>(row, first + u * 1024, w[u]);
  }
}
// the next full tile of a wave, loaded while the one before is worked on
template <class T>
struct RowFeed {
  Vec<T> w[32 / T::VEC];
  __device__ __forceinline__ void issue(const typename T::S* row, int base, int lane) {
    const unsigned first = fresh((unsigned)(base + lane * T::VEC) * (unsigned)sizeof(typename T::S));
#pragma unroll
    for (int u = 0; u < 32 / T::VEC; ++u) w[u] = load_vec<T>(row, first + u * 1024);
  }
  __device__ __forceinline__ void take(float (&v)[32]) const {
#pragma unroll
    for (int u = 0; u < 32; ++u) v[u] = w[u / T::VEC].get(u % T::VEC);
  }
  __device__ __forceinline__ void issue_some(const typename T::S* row, int base, int end, int lane) {
    const unsigned first = fresh((unsigned)(base + lane * T::VEC));
#pragma unroll
    for (int u = 0; u < 32 / T::VEC; ++u) {
      const unsigned j = first + u * 64 * T::VEC;
      const int n = end - (int)j;
      w[u].d = u32x4{0, 0, 0, 0};
      if (n >= T::VEC) w[u] = load_vec<T>(row, j * (unsigned)sizeof(typename T::S));
      else if (n > 0) w[u] = load_some<T>(row, j * (unsigned)sizeof(typename T::S), n);
    }
  }
};
template <class T>
__device__ __forceinline__ void mask_tail(float (&v)[32], int base, int end, int lane, float far) {
  const int n = end - (int)fresh((unsigned)(base + lane * T::VEC));
#pragma unroll
  for (int u = 0; u < 32; ++u) v[u] = tile_class<T>(0, u) < n ? v[u] : far;
}
// f(v, base, it, full) for every block-wide step `it` of [begin, end); v is all `far` for a wave that has nothing in
// the last one.  The body is there once: three copies of it (first step, last step, loop) spilled, and waiting
// for a spilled value waits for the loads that are on their way.
template <class T, int NT, class F>
__device__ __forceinline__ void walk_row(const typename T::S* row, int begin, int end, int lane, int wave, float far, F f) {
  const int steps = (end - begin + NT * 32 - 1) / (NT * 32), full = (end - begin) / (NT * 32);
  int base = begin + wave * kWaveTile;
  RowFeed<T> feed;
  if (full > 0) feed.issue(row, base, lane);
  else feed.issue_some(row, base, end, lane);
#pragma clang loop unroll(disable)
  for (int it = 0; it < steps; ++it) {
    float v[32];
    feed.take(v);
    if (it >= full) {
      rare();
      mask_tail<T>(v, base, end, lane, far);
    }
    const int next = base + NT * 32;
    if (it + 1 < full) {
      feed.issue(row, next, lane);
    } else if (it + 1 < steps) {
      rare();
      feed.issue_some(row, next, end, lane);
    }
    f(v, base, it, it < full);
    base = next;
  }
}
template <int NT>
__device__ __forceinline__ Acc acc_block(Acc a, const Side& z, Acc* red) {
  a = acc_wave(a, z);
  if (NT == 64) return a;
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = a;
  __syncthreads();
  a = red[0];
#pragma unroll
  for (int w = 1; w < NT / 64; ++w) a = acc_join(a, red[w], z);
  return a;
}

// ---- top classes of a stretch of a row ---------------------------------------------------------------------
// While the row is read, each thread only puts down the best of its 32 classes of every step (a cell; of
// several steps where there are more than 16), in LDS.
// The k-th largest of the threads' own maxima is then a bound that at least k classes reach, and few
// others do: the cells that reach it, hardly more than k of them, are read again, 32 lanes a cell, and the
// classes that reach it are ranked by counting.  (Collecting them from the registers in the loop, with a
// bound raised on the way, cost more than it saved: 45 us against 31 without a list, 1023 x 50001 f16.)
// Rows with more such cells or classes than LDS holds (constant ones, or masked but for a few classes), and
// rows with NaN, take row_top_again(): the classes above the bound, then the ones at it from the first
// on; and k rounds of "largest below the last" where that does not fit either.
constexpr int kCand = 1024, kCells = 512;
constexpr int kCellRows = 16;   // at most so many cells a thread
__host__ __device__ constexpr int cell_span(int steps) { return (steps + kCellRows - 1) / kCellRows; }  // steps a cell
constexpr int kBoundBits = 20;  // of a maximum's 32 order bits: a bound a little too low only lets a few more in
struct TopShared {
  unsigned long long cand[kCand];
  float maxima[256];
  unsigned long long best[4];
  unsigned cells[kCells];
  int count, cell_count, total[4];
  float bound;
};
__device__ __forceinline__ unsigned order_bits(float v) {
  const unsigned b = __builtin_bit_cast(unsigned, v + 0.f);
  return b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
}
// (just below) the k-th largest of the block's maxima, the same in every thread; two barriers
template <int NT>
__device__ __forceinline__ float raise_bound(float my_max, int k, TopShared& sh) {
  unsigned o[NT / 64];
  if (NT == 64) {
    o[0] = order_bits(my_max);
  } else {
    __syncthreads();
    sh.maxima[threadIdx.x] = my_max;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) o[w] = order_bits(sh.maxima[w * 64 + (threadIdx.x & 63)]);
  }
  unsigned t = 0;
#pragma unroll 4
  for (int bit = 31; bit > 31 - kBoundBits; --bit) {
    const unsigned c = t | 1u << bit;
    int n = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) n += __popcll(__ballot(o[w] >= c));
    t = n >= k ? c : t;
  }
  if (t <= 0x007fffffu) return -kInf;  // at or below the order bits of -inf
  return __builtin_bit_cast(float, (t >> 31) ? (t ^ 0x80000000u) : ~t);
}
// how many of the n keys are larger; eight are read at a time
__device__ __forceinline__ int rank_of(unsigned long long mine, const unsigned long long* keys, int n) {
  int rank = 0, j = 0;
  for (; j + 8 <= n; j += 8) {
#pragma unroll
    for (int i = 0; i < 8; ++i) rank += keys[j + i] > mine ? 1 : 0;
  }
  for (; j < n; ++j) rank += keys[j] > mine ? 1 : 0;
  return rank;
}
// ranks the candidates; out: the `want` largest, descending
template <int NT>
__device__ __forceinline__ void rank_candidates(int n, int want, unsigned long long* out, const TopShared& sh) {
  for (int i = threadIdx.x; i < n; i += NT) {
    const unsigned long long mine = sh.cand[i];
    const int rank = rank_of(mine, sh.cand, n);
    if (rank < want) out[rank] = mine;
  }
}
template <class T, int NT>
__device__ __forceinline__ void row_top_again(const typename T::S* row, int begin, int end, int k, float sign, float my_max,
                                           bool bad, unsigned long long* out, TopShared& sh) {
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int want = min(k, end - begin);
  __syncthreads();
  if (tid == 0) sh.count = 0;
  const float bound = raise_bound<NT>(my_max, k, sh);
  __syncthreads();
  bool slow = bad;
  int n = 0;
  if (!slow) {
    // the classes above the bound
    if (my_max > bound) {
      for (int base = begin + wave * kWaveTile; base < end; base += NT * 32) {
        float v[32];
        RowFeed<T> feed;
        feed.issue_some(row, base, end, lane);
        feed.take(v);
#pragma unroll
        for (int u = 0; u < 32; ++u) {
          const int j = base + tile_class<T>(lane, u);
          if (v[u] * sign > bound && j < end) {
            const int at = atomicAdd(&sh.count, 1);
            if (at < kCand) sh.cand[at] = key_u64(v[u] * sign, j);
          }
        }
      }
    }
    __syncthreads();
    n = sh.count;
    slow = n > kCand;
    if (!slow && n < want) {  // the ones at it, lowest index first
      for (int base = begin; base < end && n < want; base += NT) {
        const int j = base + tid;
        const float v = j < end ? T::up(row[j]) * sign : 0.f;
        const bool tie = j < end && v == bound;
        const unsigned long long b = __ballot(tie);
        if (lane == 0) sh.total[wave] = __popcll(b);
        __syncthreads();
        int at = n + __popcll(b & ((1ull << lane) - 1));
        for (int w = 0; w < wave; ++w) at += sh.total[w];
        if (tie && at < want) sh.cand[at] = key_u64(v, j);
        for (int w = 0; w < NT / 64; ++w) n += sh.total[w];
        __syncthreads();
      }
      n = min(n, want);
      slow = n < want;  // the bound lies between two values: too few above it, and none at it
    }
  }
  if (!slow) {
    __syncthreads();
    rank_candidates<NT>(n, want, out, sh);
  } else {
    unsigned long long last = ~0ull;
    for (int r = 0; r < want; ++r) {
      unsigned long long best = 0;
      for (int j = begin + tid; j < end; j += NT) {
        const unsigned long long key = key_u64(T::up(row[j]) * sign, j);
        if (key < last && key > best) best = key;
      }
#pragma unroll
      for (int s = 1; s < 64; s <<= 1) {
        const unsigned long long o = __shfl_xor(best, s, 64);
        best = o > best ? o : best;
      }
      __syncthreads();
      if (lane == 0) sh.best[wave] = best;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < NT / 64; ++w) best = sh.best[w] > best ? sh.best[w] : best;
      if (tid == 0) out[r] = best;
      last = best;
    }
  }
}

struct LpOut {
  float *log_prob, *entropy, *top_lp;
  int32_t* top_idx;
  Stats3* stats;
};
template <class T>
__device__ __forceinline__ void lp_row_write(const Prob& p, int64_t row, int given, typename T::S x_given, const Acc& a,
                                             const LpOut& o) {
  const Side z = side(p);
  const float base = a.m == z.far() ? 0.f : a.m, ln_s = logf(a.s);
  const float lp = given >= 0 ? log_p(T::up(x_given), base, ln_s, p.scale) : 0.f;
  if (o.log_prob) o.log_prob[row] = lp;
  if (o.entropy) o.entropy[row] = entropy_of(a.s, a.w, ln_s);
  if (o.stats) o.stats[row] = Stats3{base, a.s, a.w};
}
__device__ __forceinline__ void lp_row_top_write(const Prob& p, int64_t row, int rank, unsigned long long key,
                                                 const Acc& a, const LpOut& o) {
  const Side z = side(p);
  const float base = a.m == z.far() ? 0.f : a.m;
  o.top_lp[row * p.k + rank] = log_p(key_value(key) * z.sign, base, logf(a.s), p.scale);
  o.top_idx[row * p.k + rank] = key_index(key);
}

// partial results of a block of a split row
struct Part {
  float m, s, w, pad;
};
__host__ __device__ inline size_t parts_bytes(int64_t rows, int chunks) {
  return ((size_t)rows * chunks * sizeof(Part) + 255) / 256 * 256;
}

template <class T, int NT, bool TOP>
__global__ __launch_bounds__(NT, 4) void lp_row_fwd(Prob p, const typename T::S* __restrict__ x,
                                                 const void* __restrict__ index, LpOut o, Part* __restrict__ parts,
                                                 unsigned long long* __restrict__ part_keys) {
  __shared__ Acc red[NT / 64];
  const int64_t row = blockIdx.x / (unsigned)p.chunks;
  const int chunk = blockIdx.x - (unsigned)row * p.chunks;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const typename T::S* xr = x + row * p.V;
  const int begin = chunk * p.chunk, end = min(p.V, begin + p.chunk);
  const Side z = side(p);
  extern __shared__ float cell_best[];  // [cell][thread]
  // (the span is that of a whole chunk, which the launch makes room for: a short last one could have more cells)
  const int steps = (end - begin + NT * 32 - 1) / (NT * 32), span = cell_span((p.chunk + NT * 32 - 1) / (NT * 32));
  float so_far = -kInf;
  int cell = 0, in_cell = 0;
  // the given class, on its way while the row is read
  const int given = index && p.chunks == 1 ? valid_index(load_index(index, row, p.flags), p.V) : -1;
  const typename T::S x_given = given >= 0 ? xr[given] : typename T::S(0);
  Acc a = acc_empty(z);
  walk_row<T, NT>(xr, begin, end, lane, wave, z.far(), [&](const float (&v)[32], int base, int, bool) {
    const bool mine = base < end;  // (a row's last step may leave waves without classes: 1023 x 50001 f16 33 -> 32 us)
    const float top = mine ? z.best_of(v) : z.far();
    if constexpr (TOP) {
      so_far = vmax(so_far, top * z.sign);
      cell_best[cell * NT + threadIdx.x] = so_far;
      if (++in_cell == span) {
        in_cell = 0;
        ++cell;
        so_far = -kInf;
      }
    }
    if (mine) absorb<true>(a, v, 32, top, z);
  });
  const float my_max = a.m * z.sign;
  a = acc_block<NT>(a, z, red);
  if (p.chunks == 1) {
    if (threadIdx.x == 0) lp_row_write<T>(p, row, given, x_given, a, o);
  } else if (threadIdx.x == 0) {
    parts[row * p.chunks + chunk] = Part{a.m, a.s, a.w, 0.f};
  }
  if constexpr (TOP) {
    __shared__ TopShared sh;
    __shared__ unsigned long long best[kMaxEntries];
    const int want = min(p.k, end - begin), rows = (steps + span - 1) / span;
    if (threadIdx.x == 0) sh.count = sh.cell_count = 0;
    const float bound = raise_bound<NT>(my_max, p.k, sh);
    __syncthreads();
    for (int r = 0; r < rows; ++r) {
      if (cell_best[r * NT + threadIdx.x] >= bound) {
        const int at = atomicAdd(&sh.cell_count, 1);
        if (at < kCells) sh.cells[at] = r * NT + threadIdx.x;
      }
    }
    __syncthreads();
    const int cells = sh.cell_count;
    bool again = cells > kCells || a.s != a.s;
    if (!again) {
      for (int c = threadIdx.x / 32; c < cells * span; c += NT / 32) {
        const int which = sh.cells[c / span], t = which % NT, it = which / NT * span + c % span;
        const int j = begin + it * NT * 32 + t / 64 * kWaveTile + tile_class<T>(t % 64, threadIdx.x % 32);
        if (it < steps && j < end) {
          const float v = T::up(xr[j]) * z.sign;
          if (v >= bound) {
            const int at = atomicAdd(&sh.count, 1);
            if (at < kCand) sh.cand[at] = key_u64(v, j);
          }
        }
      }
      __syncthreads();
      again = sh.count > kCand;
    }
    if (again)
      row_top_again<T, NT>(xr, begin, end, p.k, z.sign, my_max, a.s != a.s, best, sh);
    else
      rank_candidates<NT>(sh.count, want, best, sh);
    __syncthreads();
    if ((int)threadIdx.x < p.k) {
      const unsigned long long key = (int)threadIdx.x < want ? best[threadIdx.x] : 0;
      if (p.chunks == 1)
        lp_row_top_write(p, row, threadIdx.x, key, a, o);
      else
        part_keys[(row * p.chunks + chunk) * p.k + threadIdx.x] = key;
    }
  }
}

// one block a row: the chunks' sums, and the best of their lists
template <class T>
__global__ __launch_bounds__(256) void lp_row_join(Prob p, const typename T::S* __restrict__ x,
                                                   const void* __restrict__ index, LpOut o,
                                                   const Part* __restrict__ parts,
                                                   const unsigned long long* __restrict__ part_keys) {
  __shared__ unsigned long long keys[kCand];
  const int64_t row = blockIdx.x;
  const Side z = side(p);
  const int given = index ? valid_index(load_index(index, row, p.flags), p.V) : -1;
  const typename T::S x_given = given >= 0 ? x[row * p.V + given] : typename T::S(0);
  const int n = p.chunks * p.k;  // at most kCand
  for (int i = threadIdx.x; i < n; i += 256) keys[i] = part_keys[row * n + i];
  Acc a = acc_empty(z);
  for (int i = threadIdx.x & 63; i < p.chunks; i += 64) {
    const Part q = parts[row * p.chunks + i];
    a = acc_join(a, Acc{q.m, q.s, q.w}, z);
  }
  a = acc_wave(a, z);
  if (threadIdx.x == 0) lp_row_write<T>(p, row, given, x_given, a, o);
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += 256) {
    const unsigned long long mine = keys[i];
    const int rank = rank_of(mine, keys, n);
    if (mine != 0 && rank < p.k) lp_row_top_write(p, row, rank, mine, a, o);
  }
}

template <class T, int NT, bool ENT>
__global__ __launch_bounds__(NT, 4) void lp_row_bwd(Prob p, const typename T::S* __restrict__ x,
                                                 const void* __restrict__ index, const Stats3* __restrict__ stats,
                                                 const float* __restrict__ g_lp,
                                                 const float* __restrict__ g_ent, typename T::S* __restrict__ g) {
  const unsigned block = block_from_end();
  const int64_t row = block / (unsigned)p.chunks;
  const int chunk = block - (unsigned)row * p.chunks;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const typename T::S* xr = x + row * p.V;
  typename T::S* gr = g + row * p.V;
  const int begin = chunk * p.chunk, end = min(p.V, begin + p.chunk);
  const Side z = side(p);
  const LpCoef r = lp_coef<ENT>(p, row, index, stats, g_lp, g_ent);
  if (r.dead) {
    row_zero<T, NT>(gr, begin, end, lane, wave);
    return;
  }
  walk_row<T, NT>(xr, begin, end, lane, wave, z.far(), [&](float (&v)[32], int base, int, bool full) {
#pragma unroll
    for (int u = 0; u < 32; ++u) {
      v[u] = lp_grad<ENT>(r, v[u], p.c, 0.f);
      fence_schedule(u);
    }
    const int rel = r.target - base;
    if ((unsigned)rel < (unsigned)kWaveTile) {
#pragma unroll
      for (int u = 0; u < 32; ++u) v[u] += tile_class<T>(lane, u) == rel ? r.hit : 0.f;
    }
    row_put<T>(gr, base, end, lane, v, p.past, full);
  });
}

// ---- distillation over long rows: every wave holds the whole list, one entry a lane --------------------
// Which of a wave's 2048 classes are listed is one ballot; what is listed, hardly one in a tile, is patched in
// registers.  2048 x 131072 bf16, 64 entries: forward (537 MB) 107 us, 5.0 TB/s, backward (1.07 GB) 194 us, 5.5 TB/s.
// 333 x 50001 f32, 20 entries: 19.4 us + 6.0 (join), backward 27; 5 x 131072: 7.5 + 6.3 and 8.0, latency.
struct Entry {
  int idx;      // -1: none
  float value;  // the teacher's, after the shift (a log-probability)
  bool again;   // the class was listed before
};
__device__ __forceinline__ Entry load_entry(const Prob& p, int64_t row, const void* teacher, const void* index, int lane) {
  const int64_t o = p.inner == 1 ? row : row / p.inner, i = p.inner == 1 ? 0 : row - o * p.inner;
  const int64_t at = o * p.es[0] + (int64_t)lane * p.es[1] + i * p.es[2];
  Entry e{-1, -kInf, false};
  if (lane < p.k) e.idx = valid_index(load_index(index, at, p.flags), p.V);
  if (teacher) {
    if (e.idx >= 0) e.value = load_teacher(teacher, at, p.flags);
    if (p.flags & kRenorm) {
      // fmaxf drops a NaN; the sum brings it back
      float tm = e.value;
#pragma unroll
      for (int k = 1; k < 64; k <<= 1) tm = fmaxf(tm, shfl_xor(tm, k));
      const float ts = wave_sum_all(exp_(e.value - (tm == -kInf ? 0.f : tm)));
      if (ts != 0.f) e.value -= tm + logf(ts);
    }
  }
  for (int k = 0; k + 1 < p.k; ++k) {
    const int other = __builtin_amdgcn_readlane(e.idx, k);
    e.again |= k < lane && other == e.idx && other >= 0;
  }
  return e;
}
// takes the listed classes that lie in this wave's tile out of v: `with` is what a listed class becomes
template <class T>
__device__ __forceinline__ void patch_tile(float (&v)[32], int base, int lane, int idx, float with) {
  unsigned long long hits = __ballot((unsigned)(idx - base) < (unsigned)kWaveTile && idx >= 0);
  while (hits) {
    const int k = __builtin_ctzll(hits);
    hits &= hits - 1;
    const int rel = __builtin_amdgcn_readlane(idx, k) - base;
    const float f = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, with), k));
    const int mine = rel % (64 * T::VEC) - lane * T::VEC, piece = rel / (64 * T::VEC);
#pragma unroll
    for (int u = 0; u < 32 / T::VEC; ++u) {
      if (piece == u) {
#pragma unroll
        for (int e = 0; e < T::VEC; ++e) v[u * T::VEC + e] = mine == e ? f : v[u * T::VEC + e];
      }
    }
  }
}
// loss and statistics of a row from the sums over its unlisted classes; one wave
template <class T>
__device__ __forceinline__ void ds_row_write(const Prob& p, int64_t row, const Entry& e, typename T::S x_listed,
                                             const Acc& a, float* loss, float4* stats) {
  const Side z = side(p);
  const float v = e.idx >= 0 ? T::up(x_listed) : z.far();
  const float first = e.again ? z.far() : v;
  RowSums r;
  r.m_r = a.m;
  r.s_r = a.s;
  const float m = z.best(a.m, wave_best_all(first, z));
  r.b = m == z.far() ? 0.f : m;
  r.s = fmaf(a.s, exp2_((a.m - r.b) * p.c), wave_sum_all(exp2_((first - r.b) * p.c)));
  r.ln_s = logf(r.s);
  const bool alive = __any(e.idx >= 0);
  const float qe = e.idx >= 0 ? exp_(e.value) : 0.f;
  const float mass = wave_sum_all(qe);
  float l = wave_sum_all(qe != 0.f ? qe * (e.value - log_p(v, r.b, r.ln_s, p.scale)) : 0.f);
  const float rr = (alive && !(p.flags & kRenorm) && r.s_r != 0.f) ? fmaxf(1.f - mass, 0.f) : 0.f;
  if (rr > 0.f) l += rest_term(r, p.scale, rr);
  if ((threadIdx.x & 63) == 0) {
    loss[row] = alive ? l : 0.f;
    if (stats) stats[row] = distill_stats(r, p.c, mass + rr, rr, alive);
  }
}

template <class T, int NT>
__global__ __launch_bounds__(NT, 4) void ds_row_fwd(Prob p, const typename T::S* __restrict__ x,
                                                 const void* __restrict__ teacher, const void* __restrict__ index,
                                                 float* __restrict__ loss, float4* __restrict__ stats,
                                                 Part* __restrict__ parts) {
  __shared__ Acc red[NT / 64];
  const int64_t row = blockIdx.x / (unsigned)p.chunks;
  const int chunk = blockIdx.x - (unsigned)row * p.chunks;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const typename T::S* xr = x + row * p.V;
  const int begin = chunk * p.chunk, end = min(p.V, begin + p.chunk);
  const Side z = side(p);
  const Entry e = load_entry(p, row, p.chunks == 1 ? teacher : nullptr, index, lane);
  const typename T::S x_listed = p.chunks == 1 && e.idx >= 0 ? xr[e.idx] : typename T::S(0);
  Acc a = acc_empty(z);
  if (__any(e.idx >= 0)) {  // the same in every wave
    walk_row<T, NT>(xr, begin, end, lane, wave, z.far(), [&](float (&v)[32], int base, int, bool full) {
      (void)full;
      if (base >= end) return;
      patch_tile<T>(v, base, lane, e.idx, z.far());
      absorb<false>(a, v, 32, z.best_of(v), z);
    });
  }
  a = acc_block<NT>(a, z, red);
  if (p.chunks > 1) {
    if (threadIdx.x == 0) parts[row * p.chunks + chunk] = Part{a.m, a.s, 0.f, 0.f};
  } else if (wave == 0) {
    ds_row_write<T>(p, row, e, x_listed, a, loss, stats);
  }
}
template <class T>
__global__ __launch_bounds__(64) void ds_row_join(Prob p, const typename T::S* __restrict__ x,
                                                  const void* __restrict__ teacher, const void* __restrict__ index,
                                                  float* __restrict__ loss, float4* __restrict__ stats,
                                                  const Part* __restrict__ parts) {
  const int64_t row = blockIdx.x;
  const Side z = side(p);
  const Entry e = load_entry(p, row, teacher, index, threadIdx.x);
  const typename T::S x_listed = e.idx >= 0 ? x[row * p.V + e.idx] : typename T::S(0);
  Acc a = acc_empty(z);
  for (int i = threadIdx.x; i < p.chunks; i += 64) {
    const Part q = parts[row * p.chunks + i];
    a = acc_join(a, Acc{q.m, q.s, 0.f}, z);
  }
  a = acc_wave(a, z);
  ds_row_write<T>(p, row, e, x_listed, a, loss, stats);
}

template <class T, int NT>
__global__ __launch_bounds__(NT, 4) void ds_row_bwd(Prob p, const typename T::S* __restrict__ x,
                                                 const void* __restrict__ teacher, const void* __restrict__ index,
                                                 const float4* __restrict__ stats, const float* __restrict__ g_loss,
                                                 typename T::S* __restrict__ g) {
  const unsigned block = block_from_end();
  const int64_t row = block / (unsigned)p.chunks;
  const int chunk = block - (unsigned)row * p.chunks;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const typename T::S* xr = x + row * p.V;
  typename T::S* gr = g + row * p.V;
  const int begin = chunk * p.chunk, end = min(p.V, begin + p.chunk);
  const Side z = side(p);
  const float4 st = stats[row];
  const float up = g_loss[row];
  const bool dead = up == 0.f || st.w == 0.f;
  const float gs = up * p.scale, rest_f = gs * st.y, member_f = gs * st.w;
  if (dead) {
    row_zero<T, NT>(gr, begin, end, lane, wave);
    return;
  }
  Entry e = load_entry(p, row, teacher, index, lane);
  float with = 0.f;
  {
    float qe = e.idx >= 0 ? exp_(e.value) : 0.f;
    float sum = qe;  // of all entries of this class
    for (int k = 0; k < p.k; ++k) {
      const int other = __builtin_amdgcn_readlane(e.idx, k);
      const float oq = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, qe), k));
      if (k != lane && other == e.idx && other >= 0) sum += oq;
    }
    if (e.idx >= 0) {
      const float v = T::up(xr[e.idx]);
      with = exp2_((v - st.z) * p.c) * member_f - gs * sum;
    }
    if (e.again) e.idx = -1;
  }
  walk_row<T, NT>(xr, begin, end, lane, wave, z.far(), [&](float (&v)[32], int base, int, bool full) {
#pragma unroll
    for (int u = 0; u < 32; ++u) {
      v[u] = exp2_((v[u] - st.x) * p.c) * rest_f;
      fence_schedule(u);
    }
    patch_tile<T>(v, base, lane, e.idx, with);
    row_put<T>(gr, base, end, lane, v, p.past, full);
  });
}

// ---- host side -----------------------------------------------------------------------------------------------
// Below 2^-120 a difference of two logits that leaves float32's range would not yet be a probability of 0; above 2^120
// the factor of the exponents, scale log2 e, and twice the scale come near its end.
constexpr float kLeastScale = 0x1p-120f, kMostScale = 0x1p120f;
// Bytes inside a row are counted in 32 bits (2^30 for float32), classes in an int, which also has to hold the ones a
// block would step to behind the last.
constexpr int64_t kMaxClasses = 1 << 28;
constexpr int64_t kMaxThreads = 0xffffffff; // of a launch
// Waves a launch should have, 8 a compute unit: long rows are split, and the waves of a tile's block share its classes, until
// there are so many.  For rows the second launch of a split is what decides (forward + backward, us; 1024 instead of 2048 in
// brackets): 64 x 32768 bf16 top 5 12.3 + 4.4 (12.4 + 4.5, 512: 12.8 + 5.3), 600 x 32768 bf16 13.0 + 15.5 (13.2 + 15.5, 4096:
// 17.2 + 14.2); it loses forward where 1024 leaves rows whole, 333 x 50001 bf16 17.3 + 16.9 (13.6 + 18.7),
// 1500 x 4096 bf16 12.3 + 7.2 (7.5 + 7.9).
constexpr int kWantWaves = 2048;
// A gradient from this size on is stored past the caches.  It would fill half of the 256 MB last-level cache or
// more, and what comes next would have to wait while that is written back: the next forward pass over 4096 x
// 32768 bf16 takes 54 us instead of 80, over 4 x 256 x 192 x 640 bf16 66 instead of 86; the backward pass
// itself 83 either way.  Smaller ones stay where the next operator finds them.  Where a wave writes half a line and
// the other half comes much later it costs more than it saves: planes take it only where 64 pixels are whole
// lines (255 bins of 131 x 641 pixels bf16: 165 us instead of 96), turned rows never (193 classes f16: 45 instead of 29).
// Flat tiles are written in one stretch.  So are rows, 1 KB at a time, and whether they begin and end with a line
// decides little (backward alone, then forward and backward in turn; ordinary stores in brackets): 2048 x 49984 bf16, whole
// lines, 85 (84), 115 (132); 2048 x 50001 95 (91), 130 (145); 1100 x 50001 f32 100 (97), 121 (146); 40000 x 3001 f16 109 (106),
// 159 (164); 40000 x 3008 92 (90), 146 (145).
constexpr int64_t kPastBytes = (int64_t)128 << 20;
constexpr size_t kLdsBudget = 152 * 1024;  // of a block, of the compute unit's 160 KB
constexpr int kMostFlat = 64 * 1024;       // of a flat tile

struct Plan {
  Prob p;
  bool tile, last;
  int layout;    // tile: kPlanes, kTurned, kFlat
  int nw;        // tile: waves a block
  int nt;        // row: threads a block
  unsigned grid;
  size_t ws;
};

int make_plan(const dw_dist_desc* d, bool distill, bool backward, Plan* out) {
  if (!d) return DW_ERR_NULL;
  if (d->outer < 0 || d->inner < 0 || d->classes < 1 || d->classes > kMaxClasses) return DW_ERR_SHAPE;
  if (d->entries < 0 || d->entries > kMaxEntries) return DW_ERR_SHAPE;
  if (distill ? d->entries < 1 : d->entries > d->classes) return DW_ERR_SHAPE;
  if (d->dtype < DW_DTYPE_F32 || d->dtype > DW_DTYPE_F16) return DW_ERR_ARG;
  const int known = distill ? DW_DIST_INDEX64 | DW_DIST_LAST | DW_DIST_RENORMALISE | DW_DIST_TEACHER_BF16 | DW_DIST_TEACHER_F16
                            : DW_DIST_INDEX64 | DW_DIST_LAST;
  if (d->flags & ~known) return DW_ERR_ARG;
  if ((d->flags & DW_DIST_TEACHER_BF16) && (d->flags & DW_DIST_TEACHER_F16)) return DW_ERR_ARG;
  if (!(fabsf(d->scale) >= kLeastScale && fabsf(d->scale) <= kMostScale)) return DW_ERR_ARG;  // (nor NaN)
  const int64_t limit = (int64_t)1 << 40;
  if (d->outer > limit || d->inner > limit || (d->inner > 0 && d->outer > limit / d->inner)) return DW_ERR_SHAPE;
  if (d->outer * d->inner > ((int64_t)1 << 48) / d->classes) return DW_ERR_SHAPE;

  Plan& P = *out;
  Prob& p = P.p;
  p = Prob{};
  p.outer = d->outer;
  p.inner = d->inner;
  p.rows = d->outer * d->inner;
  for (int i = 0; i < 3; ++i) p.es[i] = d->entry_stride[i];
  p.V = (int)d->classes;
  p.k = d->entries;
  p.scale = d->scale;
  p.c = d->scale * kLog2e;
  p.flags = d->flags;
  p.past = false;
  p.chunks = 1;
  p.chunk = p.V;
  P.ws = 0;
  P.last = (d->flags & DW_DIST_LAST) || d->inner == 1;
  const int64_t tiles = P.last ? (p.rows + 63) / 64 : d->outer * ((d->inner + 63) / 64);
  const int esize = d->dtype == DW_DTYPE_F32 ? 4 : 2;
  // Planes are tiles; so are rows of up to 2048 classes from 128 tiles on (forward + backward, us; the other family in
  // brackets).  8200 rows bf16: 40 classes 4.3 + 4.5 (12.4 + 11.5), with the top 8 6.1 + 4.5 (39.9 + 11.2), 512 classes 7.4 + 8.5 (12.5 + 12.1).
  // Rows of 3000 classes are not, 18.2 + 24.2 (21.8 + 40.7).  Between, the two are near each other forward and rows win backward: 16400 x
  // 1000 bf16 17.3 + 22.8 (19.9 + 19.5), x 2048 26.0 + 40.5 (20.8 + 26.5; with the top 8 53.9, 43.7; distillation 34.7 + 41.3, 29.2
  // + 29.2).  Nor are fewer rows, though those of up to 512 classes would be faster as tiles: 4100 x 40 8.2 + 7.8 (4.2 + 4.5),
  // top 8 24.4 (6.0), x 512 8.3 + 8.1 (7.0 + 7.4); 2100 x 1000 6.9 + 6.6 (10.1 + 11.2).
  P.tile = !P.last || (p.V <= 2048 && tiles * 4 >= kWantWaves / 4);
  if (P.tile) {
    const int row = p.V * esize;
    // Rows that are not whole lines lie in LDS as they do in memory, if 64 of them fit 64 KB (193 classes of 4 x 192 x 320
    // pixels f16: forward 32 us, turned 35; backward 40 and 70; distillation backward 54 and 64; f32, 250 classes,
    // half as many pixels: 37 and 45, 49 and 69, 55 and 76).  Not the distillation's forward pass, where one wave ends
    // the work of a block: 193 classes 44 and 40, f32 42 and 38, 50 classes 39 and 42.
    const bool flat = P.last && row % kSegBytes != 0 && flat_bytes(row) <= kMostFlat && (!distill || backward);
    P.layout = !P.last ? kPlanes : flat ? kFlat : kTurned;
    const int stage = P.layout == kTurned ? kSegBytes / esize : 32;
    const int stages = (p.V + stage - 1) / stage;
    const int most = distill || backward ? 16 : list_waves(P.last, p.k > 0);
    P.nw = 1;
    while (P.nw < most && tiles * P.nw < kWantWaves && P.nw * 2 <= stages) P.nw *= 2;
    const auto lds = [&](int nw) {
      return distill ? distill_stages(P.layout, nw, p.V, esize) + distill_lds(nw, p.k, false)
                     : (P.layout == kTurned ? (size_t)nw * kStageBytes : P.layout == kFlat ? flat_bytes(row) : 0) +
                           (size_t)nw * 64 * (backward ? 0 : 12 + (p.k ? 8 * 16 : 0));
    };
    const auto waves = [&](int nw) { return lds(nw) > kLdsBudget ? 0 : (int)(kLdsBudget / lds(nw)) * nw; };
    if (flat) {
      // The waves of a block share the tile; 16 or more should fit a compute unit (f16, 193 classes: 43 + 65 us with one
      // wave a block, 35 + 53 with two, 33 + 39 with 4 and with 8; 50 classes: 24 + 36 with one, 27 + 34 with two).
      while (P.nw * 2 <= (most < stages ? most : stages) && waves(P.nw) < 16) P.nw *= 2;
    } else if (distill) {
      // The list is the block's, a stage each wave's, so more waves a block are more waves in the LDS of a compute
      // unit.  The forward pass ends with one wave's work: it takes that only where fewer than 8 waves would fit
      // (channels_last f16, 128 classes, 8 entries: 35 us with one wave a block, 39 with two; bf16 planes, 256
      // classes, 64 entries: 210 and 116 with one and 8).  The backward pass does not (bf16 planes, 256 classes,
      // 8 entries: 118 us with one, 105 with two).
      for (int nw = P.nw * 2; nw <= 16 && nw <= stages; nw *= 2)
        if (waves(nw) > waves(P.nw) && waves(P.nw) < (backward ? 16 : 8)) P.nw = nw;
    }
    while (P.nw > 1 && lds(P.nw) > kLdsBudget) P.nw /= 2;
    // A flat tile's classes lie there already: its waves share them evenly, in whole pieces.  Not where a list is kept:
    // there a share is whole steps, so that a step has no places with the numbers of the next wave's classes.  (As many steps
    // either way; leaving such places out of the keys instead took 18.4 us for 40000 x 193 f32 top 4, 84.3 for top 64; so 17.1, 77.2.)
    p.cpw = P.layout == kFlat && (distill || backward || p.k == 0) ? (p.V + 8 * P.nw - 1) / (8 * P.nw) * 8
                                                                   : (stages + P.nw - 1) / P.nw * stage;
    if (tiles > kMaxThreads / (P.nw * 64)) return DW_ERR_SHAPE;
    P.grid = (unsigned)tiles;
    return DW_OK;
  }
  // One wave a row up to 4096 classes, four above (forward + backward, us; the other in brackets): 4000 rows bf16 of 4000 classes
  // 11.8 + 13.7 (17.5 + 17.5), 1000 rows 10.6 + 6.3 (7.8 + 7.9: one launch), 4000 of 8192 21.2 + 25.6 (18.3 + 27.1), f32
  // 27.7 + 49.1 (29.2 + 52.6), 16000 of 6000 bf16 63.9 + 68.8 (45.2 + 81.2).
  P.nt = p.V <= 2 * kWaveTile ? 64 : 256;
  const int64_t block_tile = (int64_t)P.nt * 32;
  // few rows: several blocks share one, until the chip has its waves or a block is down to one tile
  const int64_t most = (p.V + block_tile - 1) / block_tile;
  int64_t chunks = 1;
  if (p.rows > 0) chunks = (kWantWaves / (P.nt / 64) + p.rows - 1) / p.rows;
  if (chunks > most) chunks = most;
  if (!distill && !backward && p.k > 0 && chunks * p.k > kCand) chunks = kCand / p.k;
  if (chunks < 1) chunks = 1;
  const int64_t tiles_each = (most + chunks - 1) / chunks;
  p.chunk = (int)(tiles_each * block_tile < p.V ? tiles_each * block_tile : p.V);
  p.chunks = (int)((p.V + (int64_t)p.chunk - 1) / p.chunk);
  if (p.rows > kMaxThreads / P.nt / p.chunks) return DW_ERR_SHAPE;
  P.grid = (unsigned)(p.rows * p.chunks);
  if (!backward && p.chunks > 1) {
    P.ws = parts_bytes(p.rows, p.chunks);
    if (!distill) P.ws += ((size_t)p.rows * p.chunks * p.k * 8 + 255) / 256 * 256;
  }
  return DW_OK;
}
// g: where the gradient goes
void choose_stores(Plan& P, int esize, const void* g) {
  if (P.p.rows * P.p.V * esize < kPastBytes) return;
  P.p.past = P.tile ? (P.layout == kFlat || (P.layout == kPlanes && P.p.inner % 64 == 0)) && ((uintptr_t)g & 127) == 0 : true;
}
int check_ws(const Plan& P, const void* ws, size_t bytes) {
  if (P.ws == 0) return DW_OK;
  if (!ws) return DW_ERR_NULL;
  return (bytes < P.ws || ((uintptr_t)ws & 255)) ? DW_ERR_WORKSPACE : DW_OK;
}
int launched() { return hipGetLastError() == hipSuccess ? DW_OK : DW_ERR_LAUNCH; }

template <class F>
int allow_lds(F f, size_t bytes) {  // more than 64 KB of LDS has to be asked for
  if (bytes <= 64 * 1024) return DW_OK;
  return hipFuncSetAttribute((const void*)f, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) == hipSuccess
             ? DW_OK : DW_ERR_LAUNCH;
}

template <class T, int L, class KP, int K>
int lp_tile_launch(const Plan& P, const void* x, const void* index, const LpOut& o, hipStream_t st) {
  const size_t lds = (L == kTurned ? P.nw * kStageBytes : L == kFlat ? flat_bytes(P.p.V * (int)sizeof(typename T::S)) : 0) +
                     (P.nw > 1 ? P.nw * 64 * (12 + sizeof(typename KP::Key) * K) : 0);
  if (int rc = allow_lds(lp_tile_fwd<T, L, KP, K>, lds)) return rc;
  lp_tile_fwd<T, L, KP, K><<<P.grid, P.nw * 64, lds, st>>>(P.p, (const typename T::S*)x, index, o.log_prob, o.entropy,
                                                              o.top_lp, o.top_idx, o.stats);
  return launched();
}
// the list in registers: the smallest that holds all of it, or the largest there is, several times
template <class T, int L>
int lp_tile(const Plan& P, const void* x, const void* index, const LpOut& o, hipStream_t st) {
  const int k = P.p.k;
  if (k == 0) return lp_tile_launch<T, L, Wide, 0>(P, x, index, o, st);
  if constexpr (sizeof(typename T::S) == 2) {
    if (P.p.V <= Narrow::kClasses) {
      if (k <= 4) return lp_tile_launch<T, L, Narrow, 4>(P, x, index, o, st);
      if (k <= 8) return lp_tile_launch<T, L, Narrow, 8>(P, x, index, o, st);
      if (k <= 16) return lp_tile_launch<T, L, Narrow, 16>(P, x, index, o, st);
      return lp_tile_launch<T, L, Narrow, 32>(P, x, index, o, st);
    }
  }
  if constexpr (sizeof(typename T::S) == 4 || L == kPlanes) {  // (rows of that many classes do not come here)
    if (k <= 4) return lp_tile_launch<T, L, Wide, 4>(P, x, index, o, st);
    if (k <= 8) return lp_tile_launch<T, L, Wide, 8>(P, x, index, o, st);
    return lp_tile_launch<T, L, Wide, 16>(P, x, index, o, st);
  }
  return DW_ERR_SHAPE;
}
template <class T>
int lp_fwd(const Plan& P, const void* x, const void* index, const LpOut& o, void* ws, hipStream_t st) {
  const int k = P.p.k;
  if (P.tile)
    return P.layout == kPlanes  ? lp_tile<T, kPlanes>(P, x, index, o, st)
           : P.layout == kFlat ? lp_tile<T, kFlat>(P, x, index, o, st)
                               : lp_tile<T, kTurned>(P, x, index, o, st);
  Part* parts = (Part*)ws;
  unsigned long long* keys = (unsigned long long*)((char*)ws + parts_bytes(P.p.rows, P.p.chunks));
  const typename T::S* xs = (const typename T::S*)x;
  const int steps = (P.p.chunk + P.nt * 32 - 1) / (P.nt * 32), span = cell_span(steps);
  const size_t cells = k ? (size_t)(steps + span - 1) / span * P.nt * sizeof(float) : 0;
  if (P.nt == 64) {
    if (k) lp_row_fwd<T, 64, true><<<P.grid, 64, cells, st>>>(P.p, xs, index, o, parts, keys);
    else lp_row_fwd<T, 64, false><<<P.grid, 64, 0, st>>>(P.p, xs, index, o, parts, keys);
  } else {
    if (k) lp_row_fwd<T, 256, true><<<P.grid, 256, cells, st>>>(P.p, xs, index, o, parts, keys);
    else lp_row_fwd<T, 256, false><<<P.grid, 256, 0, st>>>(P.p, xs, index, o, parts, keys);
  }
  if (P.p.chunks > 1) lp_row_join<T><<<(unsigned)P.p.rows, 256, 0, st>>>(P.p, xs, index, o, parts, keys);
  return launched();
}
template <class T, bool ENT>
int lp_bwd(const Plan& P, const void* x, const void* index, const Stats3* stats, const float* g_lp,
           const float* g_ent, void* g, hipStream_t st) {
  using S = typename T::S;
  if (P.tile) {
    if (P.layout == kFlat) {
      const size_t lds = flat_bytes(P.p.V * (int)sizeof(S));
      if (int rc = allow_lds(lp_tile_bwd<T, kFlat, ENT>, lds)) return rc;
      lp_tile_bwd<T, kFlat, ENT><<<P.grid, P.nw * 64, lds, st>>>(P.p, (const S*)x, index, stats, g_lp, g_ent, (S*)g);
    } else if (P.layout == kTurned) {
      const size_t lds = P.nw * kStageBytes;
      if (int rc = allow_lds(lp_tile_bwd<T, kTurned, ENT>, lds)) return rc;
      lp_tile_bwd<T, kTurned, ENT><<<P.grid, P.nw * 64, lds, st>>>(P.p, (const S*)x, index, stats, g_lp, g_ent, (S*)g);
    } else {
      lp_tile_bwd<T, kPlanes, ENT><<<P.grid, P.nw * 64, 0, st>>>(P.p, (const S*)x, index, stats, g_lp, g_ent, (S*)g);
    }
  } else if (P.nt == 64) {
    lp_row_bwd<T, 64, ENT><<<P.grid, 64, 0, st>>>(P.p, (const S*)x, index, stats, g_lp, g_ent, (S*)g);
  } else {
    lp_row_bwd<T, 256, ENT><<<P.grid, 256, 0, st>>>(P.p, (const S*)x, index, stats, g_lp, g_ent, (S*)g);
  }
  return launched();
}
template <class T, int L>
int ds_tile_launch(const Plan& P, bool backward, const void* x, const void* teacher, const void* index, float* loss,
                   float4* stats, const float* g_loss, void* g, hipStream_t st) {
  using S = typename T::S;
  const size_t lds = distill_stages(L, P.nw, P.p.V, sizeof(S)) + distill_lds(P.nw, P.p.k, backward);
  if (backward) {
    if (int rc = allow_lds(ds_tile_bwd<T, L>, lds)) return rc;
    ds_tile_bwd<T, L><<<P.grid, P.nw * 64, lds, st>>>(P.p, (const S*)x, teacher, index, stats, g_loss, (S*)g);
  } else if constexpr (L != kFlat) {
    if (int rc = allow_lds(ds_tile_fwd<T, L>, lds)) return rc;
    ds_tile_fwd<T, L><<<P.grid, P.nw * 64, lds, st>>>(P.p, (const S*)x, teacher, index, loss, stats);
  }
  return launched();
}
template <class T>
int ds_run(const Plan& P, bool backward, const void* x, const void* teacher, const void* index, float* loss,
           float4* stats, const float* g_loss, void* g, void* ws, hipStream_t st) {
  using S = typename T::S;
  if (P.tile)
    return P.layout == kPlanes  ? ds_tile_launch<T, kPlanes>(P, backward, x, teacher, index, loss, stats, g_loss, g, st)
           : P.layout == kFlat ? ds_tile_launch<T, kFlat>(P, backward, x, teacher, index, loss, stats, g_loss, g, st)
                               : ds_tile_launch<T, kTurned>(P, backward, x, teacher, index, loss, stats, g_loss, g, st);
  const S* xs = (const S*)x;
  if (backward) {
    if (P.nt == 64) ds_row_bwd<T, 64><<<P.grid, 64, 0, st>>>(P.p, xs, teacher, index, stats, g_loss, (S*)g);
    else ds_row_bwd<T, 256><<<P.grid, 256, 0, st>>>(P.p, xs, teacher, index, stats, g_loss, (S*)g);
    return launched();
  }
  Part* parts = (Part*)ws;
  if (P.nt == 64) ds_row_fwd<T, 64><<<P.grid, 64, 0, st>>>(P.p, xs, teacher, index, loss, stats, parts);
  else ds_row_fwd<T, 256><<<P.grid, 256, 0, st>>>(P.p, xs, teacher, index, loss, stats, parts);
  if (P.p.chunks > 1) ds_row_join<T><<<(unsigned)P.p.rows, 64, 0, st>>>(P.p, xs, teacher, index, loss, stats, parts);
  return launched();
}
}  // namespace

extern "C" int64_t dw_log_probs_workspace_bytes(const dw_dist_desc* d) {
  Plan P;
  const int rc = make_plan(d, false, false, &P);
  return rc ? rc : (int64_t)P.ws;
}

extern "C" int dw_log_probs_fwd(const dw_dist_desc* d, const void* logits, const void* index, float* log_prob,
                                float* entropy, float* top_log_prob, int32_t* top_index, float* stats,
                                void* workspace, size_t workspace_bytes, void* stream) {
  Plan P;
  if (int rc = make_plan(d, false, false, &P)) return rc;
  if (P.p.rows == 0) return DW_OK;
  if (!logits || (log_prob && !index) || (P.p.k > 0 && (!top_log_prob || !top_index))) return DW_ERR_NULL;
  if (int rc = check_ws(P, workspace, workspace_bytes)) return rc;
  const LpOut o{log_prob, entropy, top_log_prob, top_index, (Stats3*)stats};
  hipStream_t st = (hipStream_t)stream;
  switch (d->dtype) {
    case DW_DTYPE_F32: return lp_fwd<F32>(P, logits, index, o, workspace, st);
    case DW_DTYPE_BF16: return lp_fwd<BF16>(P, logits, index, o, workspace, st);
    default: return lp_fwd<F16>(P, logits, index, o, workspace, st);
  }
}

extern "C" int dw_log_probs_bwd(const dw_dist_desc* d, const void* logits, const void* index, const float* stats,
                                const float* grad_log_prob, const float* grad_entropy, void* grad_logits,
                                void* stream) {
  Plan P;
  if (int rc = make_plan(d, false, true, &P)) return rc;
  if (P.p.rows == 0) return DW_OK;
  if (!logits || !stats || !grad_logits || (grad_log_prob && !index)) return DW_ERR_NULL;
  choose_stores(P, d->dtype == DW_DTYPE_F32 ? 4 : 2, grad_logits);
  const Stats3* s3 = (const Stats3*)stats;
  hipStream_t st = (hipStream_t)stream;
#define DW_LP_BWD(T)                                                                                     \
  return grad_entropy ? lp_bwd<T, true>(P, logits, index, s3, grad_log_prob, grad_entropy, grad_logits, st) \
                      : lp_bwd<T, false>(P, logits, index, s3, grad_log_prob, grad_entropy, grad_logits, st)
  switch (d->dtype) {
    case DW_DTYPE_F32: DW_LP_BWD(F32);
    case DW_DTYPE_BF16: DW_LP_BWD(BF16);
    default: DW_LP_BWD(F16);
  }
#undef DW_LP_BWD
}

extern "C" int64_t dw_distill_workspace_bytes(const dw_dist_desc* d) {
  Plan P;
  const int rc = make_plan(d, true, false, &P);
  return rc ? rc : (int64_t)P.ws;
}

extern "C" int dw_distill_fwd(const dw_dist_desc* d, const void* logits, const void* teacher, const void* teacher_index,
                              float* loss, float* stats, void* workspace, size_t workspace_bytes, void* stream) {
  Plan P;
  if (int rc = make_plan(d, true, false, &P)) return rc;
  if (P.p.rows == 0) return DW_OK;
  if (!logits || !teacher || !teacher_index || !loss) return DW_ERR_NULL;
  if (int rc = check_ws(P, workspace, workspace_bytes)) return rc;
  hipStream_t st = (hipStream_t)stream;
  switch (d->dtype) {
    case DW_DTYPE_F32: return ds_run<F32>(P, false, logits, teacher, teacher_index, loss, (float4*)stats, nullptr, nullptr, workspace, st);
    case DW_DTYPE_BF16: return ds_run<BF16>(P, false, logits, teacher, teacher_index, loss, (float4*)stats, nullptr, nullptr, workspace, st);
    default: return ds_run<F16>(P, false, logits, teacher, teacher_index, loss, (float4*)stats, nullptr, nullptr, workspace, st);
  }
}

extern "C" int dw_distill_bwd(const dw_dist_desc* d, const void* logits, const void* teacher, const void* teacher_index,
                              const float* stats, const float* grad_loss, void* grad_logits, void* stream) {
  Plan P;
  if (int rc = make_plan(d, true, true, &P)) return rc;
  if (P.p.rows == 0) return DW_OK;
  if (!logits || !teacher || !teacher_index || !stats || !grad_loss || !grad_logits) return DW_ERR_NULL;
  choose_stores(P, d->dtype == DW_DTYPE_F32 ? 4 : 2, grad_logits);
  float4* s4 = (float4*)const_cast<float*>(stats);
  hipStream_t st = (hipStream_t)stream;
  switch (d->dtype) {
    case DW_DTYPE_F32: return ds_run<F32>(P, true, logits, teacher, teacher_index, nullptr, s4, grad_loss, grad_logits, nullptr, st);
    case DW_DTYPE_BF16: return ds_run<BF16>(P, true, logits, teacher, teacher_index, nullptr, s4, grad_loss, grad_logits, nullptr, st);
    default: return ds_run<F16>(P, true, logits, teacher, teacher_index, nullptr, s4, grad_loss, grad_logits, nullptr, st);
  }
}
