// Distributions over classes (disparity bins, tokens): log-probabilities of given classes with the
// entropy and the top alternatives, and distillation from a teacher's listed classes; forward and
// backward, for float32, bfloat16 and float16 logits.
//
// Per row, with z_j = scale * x_j and everything in base 2 (c = |scale| * log2 e, v_j = sign(scale) * x_j):
//   m = max v_j,  t_j = (v_j - m) c,  e_j = 2^t_j,  s = sum e_j,  w = sum e_j t_j
//   log p_j = ln2 t_j - ln s,   entropy = ln s - ln2 w / s
// one pass over the data with a running (m, s, w): when the maximum moves by d = (m_old - m_new) c,
// s <- s 2^d and w <- 2^d (w + s d).  The difference v_j - m is taken before the product, so rows
// at the end of the float32 range (all classes at the type's lowest value) keep their meaning.
//
// Two families of kernels:
//   tile  one thread a row, 64 rows a wave; the waves of a block share the classes of their 64 rows.
//         The classes of a volume (B, V, inner) are read plane by plane (64 neighbouring pixels a
//         load); rows whose classes lie together are turned through LDS, 128 bytes of each row at
//         a time.  No cross-lane work at all, and the top classes stay sorted in registers.
//   row   a block (or a few, joined by a second kernel) for each row, for rows that are long or few.
#include <type_traits>

#include "dw_common.h"

namespace {
using namespace dw;

constexpr float kInf = __builtin_inff();
constexpr float kLn2 = 0x1.62e43p-1f;      // fl(ln 2)
constexpr float kLog2e = 0x1.715476p+0f;   // fl(log2 e)
constexpr float kFloor = -1e30f;           // stands in for an exponent of -inf where 0 * -inf would be NaN
constexpr int kMaxEntries = 64;

// mark(e): a NaN that names entry e of a teacher's list; marked(): that entry, 64 for any other value.
// (A NaN of the caller's may look the same: whoever reads a mark compares the entries' classes.)
// ---- element types -------------------------------------------------------------------------
struct F32 {
  using S = float;
  static constexpr int VEC = 4;
  static __device__ __forceinline__ float up(float v) { return v; }
  static __device__ __forceinline__ float down(float v) { return v; }
  static __device__ __forceinline__ float mark(int e) { return __builtin_bit_cast(float, 0xffc00000u | (unsigned)e); }
  static __device__ __forceinline__ int marked(float v) {
    const unsigned b = __builtin_bit_cast(unsigned, v);
    return (b & ~63u) == 0xffc00000u ? (int)(b & 63u) : 64;
  }
};
struct BF16 {
  using S = uint16_t;
  static constexpr int VEC = 8;
  static __device__ __forceinline__ float up(uint16_t v) { return __builtin_bit_cast(float, (unsigned)v << 16); }
  static __device__ __forceinline__ uint16_t down(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }
  static __device__ __forceinline__ uint16_t mark(int e) { return (uint16_t)(0xffc0 | e); }
  static __device__ __forceinline__ int marked(uint16_t v) { return (v & ~63) == 0xffc0 ? (v & 63) : 64; }
};
struct F16 {
  using S = uint16_t;
  static constexpr int VEC = 8;
  static __device__ __forceinline__ float up(uint16_t v) { return (float)__builtin_bit_cast(_Float16, v); }
  static __device__ __forceinline__ uint16_t down(float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }
  static __device__ __forceinline__ uint16_t mark(int e) { return (uint16_t)(0xff40 | e); }
  static __device__ __forceinline__ int marked(uint16_t v) { return (v & ~63) == 0xff40 ? (v & 63) : 64; }
};

// 16 bytes of elements at any element-aligned address (gfx950 loads and stores them unaligned)
template <class T>
struct Vec {
  typename T::S e[T::VEC];
};
template <class T>
__device__ __forceinline__ Vec<T> load_vec(const typename T::S* p) {
  Vec<T> r;
  __builtin_memcpy(&r, p, 16);
  return r;
}
template <class T>
__device__ __forceinline__ void store_vec(typename T::S* p, const Vec<T>& v) {
  __builtin_memcpy(p, &v, 16);
}

// v_max_f32 without the canonicalisation the compiler puts before fmaxf of loaded values; a quiet
// NaN operand gives the other one (the sum carries the NaN)
__device__ __forceinline__ float vmax(float a, float b) {
  float r;
  asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}
__device__ __forceinline__ float exp2_(float t) { return __builtin_amdgcn_exp2f(t); }

// ---- running soft-max ------------------------------------------------------------------------
struct Acc {
  float m, s, w;
};
using Stats3 = Acc;  // what the backward pass gets of a row; m is 0 in an empty one
// entropy = ln s - ln2 w / s: both terms are >= 0, nothing cancels
__device__ __forceinline__ float entropy_of(float s, float w, float ln_s) { return s == 0.f ? 0.f : ln_s - kLn2 * w / s; }
__device__ __forceinline__ Acc acc_empty() { return Acc{-kInf, 0.f, 0.f}; }

template <bool ENT, int N>
__device__ __forceinline__ void absorb(Acc& a, const float (&v)[N], float c) {
  float m = a.m;
#pragma unroll
  for (int i = 0; i < N; ++i) m = vmax(m, v[i]);
  const float b = m == -kInf ? 0.f : m;
  const float d = fmaxf((a.m - b) * c, kFloor), al = exp2_(d);
  if (ENT) a.w = al * fmaf(a.s, d, a.w);
  a.s *= al;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float t = (v[i] - b) * c, e = exp2_(t);
    a.s += e;
    if (ENT) a.w = fmaf(e, vmax(t, kFloor), a.w);
  }
  a.m = m;
}
__device__ __forceinline__ Acc acc_join(const Acc& a, const Acc& b, float c) {
  const float m = vmax(a.m, b.m), o = m == -kInf ? 0.f : m;
  const float da = fmaxf((a.m - o) * c, kFloor), db = fmaxf((b.m - o) * c, kFloor);
  const float ea = exp2_(da), eb = exp2_(db);
  return Acc{m, a.s * ea + b.s * eb, ea * fmaf(a.s, da, a.w) + eb * fmaf(b.s, db, b.w)};
}
__device__ __forceinline__ float shfl_xor(float v, int mask) { return __shfl_xor(v, mask, 64); }
__device__ __forceinline__ Acc acc_wave(Acc a, float c) {
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) {
    Acc b{shfl_xor(a.m, k), shfl_xor(a.s, k), shfl_xor(a.w, k)};
    // both lanes of a pair evaluate the same expression (lower lane's sums first): one result everywhere
    a = (threadIdx.x & k) ? acc_join(b, a, c) : acc_join(a, b, c);
  }
  return a;
}
__device__ __forceinline__ float wave_max_all(float v) {
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) v = vmax(v, shfl_xor(v, k));
  return v;
}
__device__ __forceinline__ float wave_sum_all(float v) {
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) v += shfl_xor(v, k);
  return v;
}

// log p of a class of value v in a row of (m, ln s): -inf for a masked class, also where the whole row
// is masked (ln s = -inf); NaN where the row holds NaN or +inf
// (in base e: in base 2 the log-probability of a class at float32's lowest value would overflow)
__device__ __forceinline__ float log_p(float v, float m, float ln_s, float scale) {
  return (v == -kInf && ln_s == ln_s) ? -kInf : fmaf(v - m, fabsf(scale), -ln_s);
}

// ---- order keys --------------------------------------------------------------------------------
// 64-bit whole number that orders classes by value, then by lowest index; NaN above everything
__device__ __forceinline__ unsigned long long key_u64(float v, int idx) {
  unsigned b = __builtin_bit_cast(unsigned, v + 0.f);
  b = v != v ? 0xffffffffu : (b ^ ((unsigned)((int)b >> 31) | 0x80000000u));
  return ((unsigned long long)b << 32) | (0xffffffffu - (unsigned)idx);
}
__device__ __forceinline__ float key_value(unsigned long long k) {
  const unsigned b = (unsigned)(k >> 32);
  if (b == 0xffffffffu) return __builtin_nanf("");
  return __builtin_bit_cast(float, (b >> 31) ? (b ^ 0x80000000u) : ~b);
}
__device__ __forceinline__ int key_index(unsigned long long k) { return (int)(0xffffffffu - (unsigned)k); }

// The same order as a float64, so that a comparator is one v_max_f64 and one v_min_f64 (full rate on
// this chip): the value in the upper bits, the index in the 29 mantissa bits a converted float32
// leaves empty, complemented for positive values.  Infinities and NaN become finite values beyond
// every float32.
constexpr double kKeyInf = 0x1p+200, kKeyNan = 0x1p+300, kKeyNone = -0x1p+400;
__device__ __forceinline__ double key_f64(float v, int idx) {
  double d = (double)(v + 0.f);
  if (!(fabsf(v) < kInf)) d = v != v ? kKeyNan : (v > 0.f ? kKeyInf : -kKeyInf);
  unsigned long long b = __builtin_bit_cast(unsigned long long, d);
  const unsigned low = (b >> 63) ? (unsigned)idx : (0x1fffffffu - (unsigned)idx);
  return __builtin_bit_cast(double, b | low);
}
__device__ __forceinline__ float key_f64_value(double k) {
  const unsigned long long b = __builtin_bit_cast(unsigned long long, k) & ~0x1fffffffull;
  const double d = __builtin_bit_cast(double, b);
  if (d >= kKeyNan) return __builtin_nanf("");
  if (d >= kKeyInf) return kInf;
  if (d <= -kKeyInf) return -kInf;
  return (float)d;
}
__device__ __forceinline__ int key_f64_index(double k) {
  const unsigned long long b = __builtin_bit_cast(unsigned long long, k);
  const int low = (int)(b & 0x1fffffffull);
  return (b >> 63) ? low : 0x1fffffff - low;
}
__device__ __forceinline__ double max64(double a, double b) {
  double r;
  asm("v_max_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}
__device__ __forceinline__ double min64(double a, double b) {
  double r;
  asm("v_min_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}
__device__ __forceinline__ void order2(double& hi, double& lo) {
  const double a = max64(hi, lo), b = min64(hi, lo);
  hi = a;
  lo = b;
}
// descending sort of K keys in registers: Batcher's odd-even merge network
template <int K>
__device__ __forceinline__ void sort_desc(double (&a)[K]) {
#pragma unroll
  for (int p = 1; p < K; p <<= 1)
#pragma unroll
    for (int k = p; k >= 1; k >>= 1)
#pragma unroll
      for (int j = k % p; j + k < K; j += 2 * k)
#pragma unroll
        for (int i = 0; i < k; ++i)
          if (i + j + k < K && (i + j) / (2 * p) == (i + j + k) / (2 * p)) order2(a[i + j], a[i + j + k]);
}
// top <- the K largest of two descending lists, descending
template <int K>
__device__ __forceinline__ void merge_desc(double (&top)[K], const double (&n)[K]) {
#pragma unroll
  for (int i = 0; i < K; ++i) top[i] = max64(top[i], n[K - 1 - i]);
#pragma unroll
  for (int h = K / 2; h >= 1; h >>= 1)
#pragma unroll
    for (int i = 0; i < K; ++i)
      if ((i & h) == 0) order2(top[i], top[i + h]);
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
};
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

// ---- tile kernels: where the 64 rows of a block are, and how their classes come in -----------------
struct Place {
  int64_t row;    // this lane's row, clamped to the last one
  int64_t o, i;   // its outer and inner index
  int64_t first;  // first row (LAST) or first pixel (planes) of the block
  int lane, wave;
  bool live;      // the row exists
};
template <bool LAST>
__device__ __forceinline__ Place place(const Prob& p) {
  Place q;
  q.lane = threadIdx.x & 63;
  q.wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (LAST) {
    q.first = (int64_t)blockIdx.x * 64;
    q.row = q.first + q.lane;
    q.live = q.row < p.rows;
    if (!q.live) q.row = p.rows - 1;
    q.o = p.inner == 1 ? q.row : q.row / p.inner;
    q.i = p.inner == 1 ? 0 : q.row - q.o * p.inner;
  } else {
    const unsigned tiles = (unsigned)((p.inner + 63) / 64);
    q.o = blockIdx.x / tiles;
    q.first = (int64_t)(blockIdx.x - (unsigned)q.o * tiles) * 64;
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
template <class T, bool LAST>
constexpr int stage_classes() { return LAST ? kSegBytes / (int)sizeof(typename T::S) : 32; }

// 64 row segments of classes [c0, c0 + n) into LDS (n <= stage_classes); 8 lanes a row
template <class T>
__device__ __forceinline__ void stage_in(const typename T::S* x, const Prob& p, const Place& q, int c0, int n,
                                         char* lds) {
  constexpr int PER = kSegBytes / 16;
  const int seg = q.lane % PER, j = seg * T::VEC;
  Vec<T> v[PER];
#pragma unroll
  for (int it = 0; it < PER; ++it) {
    const int64_t row = min(q.first + it * (64 / PER) + q.lane / PER, p.rows - 1);
    const typename T::S* src = x + row * p.V + c0 + j;
    if (j + T::VEC <= n) {
      v[it] = load_vec<T>(src);
    } else {
#pragma unroll
      for (int e = 0; e < T::VEC; ++e) v[it].e[e] = j + e < n ? src[e] : typename T::S(0);
    }
  }
#pragma unroll
  for (int it = 0; it < PER; ++it)
    *(Vec<T>*)(lds + (it * (64 / PER) + q.lane / PER) * kRowBytes + seg * 16) = v[it];
}
template <class T>
__device__ __forceinline__ void stage_out(typename T::S* g, const Prob& p, const Place& q, int c0, int n,
                                          const char* lds) {
  constexpr int PER = kSegBytes / 16;
  const int seg = q.lane % PER, j = seg * T::VEC;
#pragma unroll
  for (int it = 0; it < PER; ++it) {
    const int r = it * (64 / PER) + q.lane / PER;
    if (q.first + r >= p.rows) continue;
    const Vec<T> v = *(const Vec<T>*)(lds + r * kRowBytes + seg * 16);
    typename T::S* dst = g + (q.first + r) * p.V + c0 + j;
    if (j + T::VEC <= n) {
      store_vec<T>(dst, v);
    } else {
#pragma unroll
      for (int e = 0; e < T::VEC; ++e)
        if (j + e < n) dst[e] = v.e[e];
    }
  }
}
// 32 classes of this lane's row from the stage, from class h of the segment on
template <class T>
__device__ __forceinline__ void stage_read(const char* lds, int lane, int h, float (&v)[32]) {
#pragma unroll
  for (int u = 0; u < 32 / T::VEC; ++u) {
    const Vec<T> w = *(const Vec<T>*)(lds + lane * kRowBytes + h * (int)sizeof(typename T::S) + u * 16);
#pragma unroll
    for (int e = 0; e < T::VEC; ++e) v[u * T::VEC + e] = T::up(w.e[e]);
  }
}
template <class T>
__device__ __forceinline__ void stage_write(char* lds, int lane, int h, const float (&v)[32]) {
#pragma unroll
  for (int u = 0; u < 32 / T::VEC; ++u) {
    Vec<T> w;
#pragma unroll
    for (int e = 0; e < T::VEC; ++e) w.e[e] = T::down(v[u * T::VEC + e]);
    *(Vec<T>*)(lds + lane * kRowBytes + h * (int)sizeof(typename T::S) + u * 16) = w;
  }
}
// 32 planes from class c0 on; the planes behind the n-th repeat it
template <class T>
__device__ __forceinline__ void planes_in(const typename T::S* x, const Prob& p, const Place& q, int c0, int n,
                                          float (&v)[32]) {
  const typename T::S* base = x + (q.o * p.V + c0) * p.inner + q.first;
  const unsigned at = (unsigned)(q.i - q.first);
#pragma unroll
  for (int u = 0; u < 32; ++u) v[u] = T::up((base + (int64_t)min(u, n - 1) * p.inner)[at]);
}
// z's sign, and -inf behind the n-th class
__device__ __forceinline__ void settle(float (&v)[32], bool neg, int n) {
  if (neg) {
#pragma unroll
    for (int u = 0; u < 32; ++u) v[u] = -v[u];
  }
  if (n < 32) {
#pragma unroll
    for (int u = 0; u < 32; ++u) v[u] = u < n ? v[u] : -kInf;
  }
}

// ---- log-probabilities, forward, tile ---------------------------------------------------------------
// K: top classes kept in registers (0: none).  More than K wanted: further passes over the data, each
// for the next K below the last key of the pass before.
template <class T, bool LAST, int K>
__global__ void lp_tile_fwd(Prob p, const typename T::S* __restrict__ x, const void* __restrict__ index,
                            float* __restrict__ log_prob, float* __restrict__ entropy, float* __restrict__ top_lp,
                            int32_t* __restrict__ top_idx, Stats3* __restrict__ stats) {
  extern __shared__ __align__(16) char smem[];
  const Place q = place<LAST>(p);
  const int nw = blockDim.x >> 6;
  char* stage = smem + q.wave * kStageBytes;                       // LAST only
  char* joint = smem + (LAST ? nw * kStageBytes : 0);
  float* red = (float*)joint;                                      // [3][nw][64]
  double* keys = (double*)(joint + 3 * nw * 64 * sizeof(float));   // [nw][K][64]
  const bool neg = p.scale < 0.f;
  const int c_lo = q.wave * p.cpw, c_hi = min(p.V, c_lo + p.cpw);

  Acc a = acc_empty();
  double limit = 0.0;
  float ln_s = 0.f, base = 0.f;
  for (int done = 0; done == 0 || done < p.k; done += (K ? K : 1)) {
    double top[K ? K : 1];
#pragma unroll
    for (int i = 0; i < K; ++i) top[i] = kKeyNone;
    for (int c0 = c_lo; c0 < c_hi; c0 += stage_classes<T, LAST>()) {
      const int n = min(stage_classes<T, LAST>(), c_hi - c0);
      if (LAST) {
        wave_sync();
        stage_in<T>(x, p, q, c0, n, stage);
        wave_sync();
      }
      for (int h = 0; h < n; h += 32) {
        float v[32];
        if (LAST)
          stage_read<T>(stage, q.lane, h, v);
        else
          planes_in<T>(x, p, q, c0, n, v);
        settle(v, neg, n - h);
        if (done == 0) absorb<true>(a, v, p.c);
        if constexpr (K > 0) {
#pragma unroll
          for (int g = 0; g < 32; g += K) {
            double nk[K];
#pragma unroll
            for (int i = 0; i < K; ++i) {
              nk[i] = key_f64(v[g + i], c0 + h + g + i);
              if (done > 0 && !(nk[i] < limit)) nk[i] = kKeyNone;
            }
            sort_desc<K>(nk);
            merge_desc<K>(top, nk);
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
          a = acc_join(a, Acc{red[w * 64 + q.lane], red[(nw + w) * 64 + q.lane], red[(2 * nw + w) * 64 + q.lane]}, p.c);
      }
      if constexpr (K > 0) {
#pragma unroll
        for (int i = 0; i < K; ++i) top[i] = keys[i * 64 + q.lane];
        for (int w = 1; w < nw; ++w) {
          double other[K];
#pragma unroll
          for (int i = 0; i < K; ++i) other[i] = keys[(w * K + i) * 64 + q.lane];
          merge_desc<K>(top, other);
        }
      }
      __syncthreads();
    }
    if (done == 0) {
      base = a.m == -kInf ? 0.f : a.m;
      ln_s = logf(a.s);
      if (q.wave == 0 && q.live) {
        const int t = index ? valid_index(load_index(index, q.row, p.flags), p.V) : -1;
        float lp = 0.f;
        if (t >= 0) {
          const float v = T::up(x[element<LAST>(p, q, t)]);
          lp = log_p(neg ? -v : v, base, ln_s, p.scale);
        }
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
            const float v = key_f64_value(top[i]);
            const int64_t at = LAST ? q.row * p.k + done + i : (q.o * p.k + done + i) * p.inner + q.i;
            top_lp[at] = log_p(v, base, ln_s, p.scale);
            top_idx[at] = key_f64_index(top[i]);
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
  return fmaf(e, ENT ? fmaf(vmax(t, kFloor), r.k1, r.k0) : r.k0, add);
}

template <class T, bool LAST, bool ENT>
__global__ void lp_tile_bwd(Prob p, const typename T::S* __restrict__ x, const void* __restrict__ index,
                            const Stats3* __restrict__ stats, const float* __restrict__ g_lp, const float* __restrict__ g_ent,
                            typename T::S* __restrict__ g) {
  extern __shared__ __align__(16) char smem[];
  const Place q = place<LAST>(p);
  char* stage = smem + q.wave * kStageBytes;
  const bool neg = p.scale < 0.f;
  const int c_lo = q.wave * p.cpw, c_hi = min(p.V, c_lo + p.cpw);
  const LpCoef r = lp_coef<ENT>(p, q.row, index, stats, g_lp, g_ent);
  const bool any_dead = __any(r.dead);
  for (int c0 = c_lo; c0 < c_hi; c0 += stage_classes<T, LAST>()) {
    const int n = min(stage_classes<T, LAST>(), c_hi - c0);
    if (LAST) {
      wave_sync();
      stage_in<T>(x, p, q, c0, n, stage);
      wave_sync();
    }
    for (int h = 0; h < n; h += 32) {
      float v[32];
      if (LAST)
        stage_read<T>(stage, q.lane, h, v);
      else
        planes_in<T>(x, p, q, c0, n, v);
      settle(v, neg, n - h);
      const int rel = r.target - c0 - h;
#pragma unroll
      for (int u = 0; u < 32; ++u) v[u] = lp_grad<ENT>(r, v[u], p.c, rel == u ? r.hit : 0.f);
      if (any_dead) {
#pragma unroll
        for (int u = 0; u < 32; ++u) v[u] = r.dead ? 0.f : v[u];
      }
      if (LAST) {
        stage_write<T>(stage, q.lane, h, v);
      } else {
        typename T::S* dst = g + (q.o * p.V + c0) * p.inner + q.first;
        const unsigned at = (unsigned)(q.i - q.first);
        if (q.live) {
#pragma unroll
          for (int u = 0; u < 32; ++u)
            if (u < n) (dst + (int64_t)u * p.inner)[at] = T::down(v[u]);
        }
      }
    }
    if (LAST) {
      wave_sync();
      stage_out<T>(g, p, q, c0, n, stage);
    }
  }
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
  const float lp = fmaf(r.m_r - r.b, fabsf(scale), logf(r.s_r) - r.ln_s);
  return rr > 0.f ? rr * (logf(rr) - lp) : 0.f;
}
__device__ __forceinline__ float4 distill_stats(const RowSums& r, float c, float mass, float rr, bool alive) {
  float4 st = make_float4(0.f, 0.f, r.b, 0.f);
  if (!alive || r.s == 0.f) return st;
  if (r.s_r != 0.f) {
    st.x = r.m_r;
    st.y = mass * exp2_((r.m_r - r.b) * c) / r.s - rr / r.s_r;
  }
  st.w = mass / r.s;
  return st;
}

// Column of this lane's row inside the stage: planes [class][64] float32, or the row's own bytes
template <class T, bool LAST>
struct Column {
  using S = std::conditional_t<LAST, typename T::S, float>;
  using M = std::conditional_t<LAST, T, F32>;
  char* lds;
  int lane;
  __device__ __forceinline__ S* at(int u) const {
    return LAST ? (S*)(lds + lane * kRowBytes) + u : (S*)lds + u * 64 + lane;
  }
};
constexpr int kPlaneStage = 32 * 64 * 4;
template <bool LAST>
constexpr int distill_stage_bytes() { return LAST ? kStageBytes : kPlaneStage; }

// ---- distillation, forward, tile ------------------------------------------------------------------------
// Each listed class is taken out of its column before the running soft-max sees the column, so the
// unlisted classes are summed on their own (1 - sum of the listed would cancel where the list holds
// nearly everything).  A class listed twice is taken out once: a mark left in the column shows it.
template <class T, bool LAST>
__global__ void ds_tile_fwd(Prob p, const typename T::S* __restrict__ x, const void* __restrict__ teacher,
                            const void* __restrict__ index, float* __restrict__ loss, float4* __restrict__ stats) {
  extern __shared__ __align__(16) char smem[];
  const Place q = place<LAST>(p);
  const int nw = blockDim.x >> 6, K = p.k;
  char* stage = smem + q.wave * distill_stage_bytes<LAST>();
  char* rest = smem + nw * distill_stage_bytes<LAST>();
  int* idx = (int*)rest + q.lane;                  // [K][64]
  float* xk = (float*)rest + K * 64 + q.lane;      // value of the entry's class
  float* xs = (float*)rest + 2 * K * 64 + q.lane;  // the same, -inf where the class was listed before
  float* red = (float*)rest + 3 * K * 64 + q.lane; // [2][nw][64]
  const Column<T, LAST> col{stage, q.lane};
  using C = Column<T, LAST>;
  const bool neg = p.scale < 0.f;
  const int c_lo = q.wave * p.cpw, c_hi = min(p.V, c_lo + p.cpw);
  const int64_t t0 = q.o * p.es[0] + q.i * p.es[2];

  for (int e = q.wave; e < K; e += nw) {
    idx[e * 64] = valid_index(load_index(index, t0 + e * p.es[1], p.flags), p.V);
    xk[e * 64] = -kInf;
    xs[e * 64] = -kInf;
  }
  __syncthreads();
  bool alive = false;
  for (int e = 0; e < K; ++e) alive |= idx[e * 64] >= 0;
  Acc a = acc_empty();
  if (__any(alive)) {  // the same in every wave of the block
    for (int c0 = c_lo; c0 < c_hi; c0 += stage_classes<T, LAST>()) {
      const int n = min(stage_classes<T, LAST>(), c_hi - c0);
      float v[32];
      wave_sync();
      if (LAST) {
        stage_in<T>(x, p, q, c0, n, stage);
      } else {
        planes_in<T>(x, p, q, c0, n, v);
#pragma unroll
        for (int u = 0; u < 32; ++u) *(float*)col.at(u) = v[u];
      }
      wave_sync();
      for (int e = 0; e < K; ++e) {
        const int rel = idx[e * 64] - c0;
        if ((unsigned)rel < (unsigned)n) {
          const typename C::S raw = *col.at(rel);
          const int before = C::M::marked(raw);
          if (before < e && idx[before * 64] == idx[e * 64]) {
            xk[e * 64] = xk[before * 64];
          } else {
            const float f = neg ? -C::M::up(raw) : C::M::up(raw);
            xk[e * 64] = f;
            xs[e * 64] = f;
            *col.at(rel) = C::M::mark(e);
          }
        }
      }
      for (int e = 0; e < K; ++e) {
        const int rel = idx[e * 64] - c0;
        if ((unsigned)rel < (unsigned)n) *col.at(rel) = C::M::down(neg ? kInf : -kInf);
      }
      wave_sync();
      for (int h = 0; h < n; h += 32) {
        if (LAST) {
          stage_read<T>(stage, q.lane, h, v);
        } else {
#pragma unroll
          for (int u = 0; u < 32; ++u) v[u] = *(const float*)col.at(u);
        }
        settle(v, neg, n - h);
        absorb<false>(a, v, p.c);
      }
    }
  }
  red[q.wave * 64] = a.m;
  red[(nw + q.wave) * 64] = a.s;
  __syncthreads();
  if (q.wave != 0 || !q.live) return;
  a = Acc{red[0], red[nw * 64], 0.f};
  for (int w = 1; w < nw; ++w) a = acc_join(a, Acc{red[w * 64], red[(nw + w) * 64], 0.f}, p.c);

  RowSums r;
  r.m_r = a.m;
  r.s_r = a.s;
  float m = a.m, tm = -kInf;
  for (int e = 0; e < K; ++e) {
    m = vmax(m, xs[e * 64]);
    if ((p.flags & kRenorm) && idx[e * 64] >= 0) tm = fmaxf(tm, load_teacher(teacher, t0 + e * p.es[1], p.flags));
  }
  r.b = m == -kInf ? 0.f : m;
  r.s = a.s * exp2_((a.m - r.b) * p.c);
  float ts = 0.f;
  for (int e = 0; e < K; ++e) {
    r.s += exp2_((xs[e * 64] - r.b) * p.c);
    if ((p.flags & kRenorm) && idx[e * 64] >= 0)
      ts += expf(load_teacher(teacher, t0 + e * p.es[1], p.flags) - (tm == -kInf ? 0.f : tm));
  }
  r.ln_s = logf(r.s);
  const float shift = (p.flags & kRenorm) ? (ts == 0.f ? 0.f : tm + logf(ts)) : 0.f;
  float mass = 0.f, l = 0.f;
  for (int e = 0; e < K; ++e) {
    if (idx[e * 64] < 0) continue;
    const float lq = load_teacher(teacher, t0 + e * p.es[1], p.flags) - shift, qe = expf(lq);
    mass += qe;
    if (qe != 0.f) l = fmaf(qe, lq - log_p(xk[e * 64], r.b, r.ln_s, p.scale), l);
  }
  const float rr = (alive && !(p.flags & kRenorm) && r.s_r != 0.f) ? fmaxf(1.f - mass, 0.f) : 0.f;
  if (rr > 0.f) l += rest_term(r, p.scale, rr);
  loss[q.row] = alive ? l : 0.f;
  if (stats) stats[q.row] = distill_stats(r, p.c, mass + rr, rr, alive);
}

// ---- distillation, backward, tile -------------------------------------------------------------------------
template <class T, bool LAST>
__global__ void ds_tile_bwd(Prob p, const typename T::S* __restrict__ x, const void* __restrict__ teacher,
                            const void* __restrict__ index, const float4* __restrict__ stats,
                            const float* __restrict__ g_loss, typename T::S* __restrict__ g) {
  extern __shared__ __align__(16) char smem[];
  const Place q = place<LAST>(p);
  const int nw = blockDim.x >> 6, K = p.k;
  char* stage = smem + q.wave * distill_stage_bytes<LAST>();
  char* rest = smem + nw * distill_stage_bytes<LAST>();
  int* idx = (int*)rest + q.lane;
  float* gq = (float*)rest + K * 64 + q.lane;      // upstream gradient * scale * teacher's probability
  float* xk = (float*)rest + 2 * K * 64 + q.lane;  // gradient of a listed class before gq
  unsigned long long again = 0;                    // entries whose class this wave has met in an earlier entry
  const Column<T, LAST> col{stage, q.lane};
  using C = Column<T, LAST>;
  const bool neg = p.scale < 0.f, renorm = p.flags & kRenorm;
  const int c_lo = q.wave * p.cpw, c_hi = min(p.V, c_lo + p.cpw);
  const int64_t t0 = q.o * p.es[0] + q.i * p.es[2];
  const float4 st = stats[q.row];
  const float up = g_loss[q.row];
  const bool dead = up == 0.f || st.w == 0.f;
  const float gs = up * p.scale, rest_f = gs * st.y, member_f = gs * st.w;

  float shift = 0.f;
  if (renorm && !dead) {
    float tm = -kInf, ts = 0.f;
    for (int e = 0; e < K; ++e)
      if (valid_index(load_index(index, t0 + e * p.es[1], p.flags), p.V) >= 0)
        tm = fmaxf(tm, load_teacher(teacher, t0 + e * p.es[1], p.flags));
    for (int e = 0; e < K; ++e)
      if (valid_index(load_index(index, t0 + e * p.es[1], p.flags), p.V) >= 0)
        ts += expf(load_teacher(teacher, t0 + e * p.es[1], p.flags) - (tm == -kInf ? 0.f : tm));
    shift = ts == 0.f ? 0.f : tm + logf(ts);
  }
  for (int e = q.wave; e < K; e += nw) {
    const int i = dead ? -1 : valid_index(load_index(index, t0 + e * p.es[1], p.flags), p.V);
    idx[e * 64] = i;
    gq[e * 64] = i >= 0 ? gs * expf(load_teacher(teacher, t0 + e * p.es[1], p.flags) - shift) : 0.f;
  }
  __syncthreads();
  const bool any_dead = __any(dead);
  for (int c0 = c_lo; c0 < c_hi; c0 += stage_classes<T, LAST>()) {
    const int n = min(stage_classes<T, LAST>(), c_hi - c0);
    float v[32];
    wave_sync();
    if (LAST) {
      stage_in<T>(x, p, q, c0, n, stage);
    } else {
      planes_in<T>(x, p, q, c0, n, v);
#pragma unroll
      for (int u = 0; u < 32; ++u) *(float*)col.at(u) = v[u];
    }
    wave_sync();
    // listed classes: their soft-max gradient, the rest of it later; a class listed again adds its share to the first entry
    for (int e = 0; e < K; ++e) {
      const int rel = idx[e * 64] - c0;
      if ((unsigned)rel < (unsigned)n) {
        const typename C::S raw = *col.at(rel);
        const int before = C::M::marked(raw);
        if (before < e && idx[before * 64] == idx[e * 64]) {
          gq[before * 64] += gq[e * 64];
          again |= 1ull << e;
        } else {
          const float f = neg ? -C::M::up(raw) : C::M::up(raw);
          xk[e * 64] = exp2_((f - st.z) * p.c) * member_f;
          *col.at(rel) = C::M::mark(e);
        }
      }
    }
    wave_sync();
    for (int h = 0; h < n; h += 32) {
      if (LAST) stage_read<T>(stage, q.lane, h, v);
      settle(v, neg, n - h);
#pragma unroll
      for (int u = 0; u < 32; ++u) v[u] = exp2_((v[u] - st.x) * p.c) * rest_f;
      if (any_dead) {
#pragma unroll
        for (int u = 0; u < 32; ++u) v[u] = dead ? 0.f : v[u];
      }
      if (LAST) {
        stage_write<T>(stage, q.lane, h, v);
      } else {
#pragma unroll
        for (int u = 0; u < 32; ++u) *(float*)col.at(u) = v[u];
      }
    }
    wave_sync();
    for (int e = 0; e < K; ++e) {
      const int rel = idx[e * 64] - c0;
      if ((unsigned)rel < (unsigned)n && !(again >> e & 1))
        *col.at(rel) = C::M::down(xk[e * 64] - gq[e * 64]);
    }
    wave_sync();
    if (LAST) {
      stage_out<T>(g, p, q, c0, n, stage);
    } else if (q.live) {
      typename T::S* dst = g + (q.o * p.V + c0) * p.inner + q.first;
      const unsigned at = (unsigned)(q.i - q.first);
#pragma unroll
      for (int u = 0; u < 32; ++u)
        if (u < n) (dst + (int64_t)u * p.inner)[at] = T::down(*(const float*)col.at(u));
    }
  }
}

// ---- row kernels -------------------------------------------------------------------------------------------
// A wave takes 2048 neighbouring classes at a time, 32 a lane in 16-byte pieces.
constexpr int kWaveTile = 64 * 32;
template <class T>
__device__ __forceinline__ int tile_class(int lane, int u) {  // class of a lane's u-th value inside the wave's tile
  return (u / T::VEC) * 64 * T::VEC + lane * T::VEC + u % T::VEC;
}
template <class T>
__device__ __forceinline__ void row_in(const typename T::S* row, int base, int end, int lane, bool neg, float (&v)[32]) {
  if (base + kWaveTile <= end) {
    Vec<T> w[32 / T::VEC];
#pragma unroll
    for (int u = 0; u < 32 / T::VEC; ++u) w[u] = load_vec<T>(row + base + tile_class<T>(lane, u * T::VEC));
#pragma unroll
    for (int u = 0; u < 32; ++u) v[u] = T::up(w[u / T::VEC].e[u % T::VEC]);
  } else {
#pragma unroll
    for (int u = 0; u < 32 / T::VEC; ++u) {
      const int j = base + tile_class<T>(lane, u * T::VEC);
      if (j + T::VEC <= end) {
        const Vec<T> w = load_vec<T>(row + j);
#pragma unroll
        for (int e = 0; e < T::VEC; ++e) v[u * T::VEC + e] = T::up(w.e[e]);
      } else {
#pragma unroll
        for (int e = 0; e < T::VEC; ++e)
          v[u * T::VEC + e] = j + e < end ? T::up(row[j + e]) : (neg ? kInf : -kInf);
      }
    }
  }
  if (neg) {
#pragma unroll
    for (int u = 0; u < 32; ++u) v[u] = -v[u];
  }
}
template <class T>
__device__ __forceinline__ void row_out(typename T::S* row, int base, int end, int lane, const float (&v)[32]) {
#pragma unroll
  for (int u = 0; u < 32 / T::VEC; ++u) {
    const int j = base + tile_class<T>(lane, u * T::VEC);
    Vec<T> w;
#pragma unroll
    for (int e = 0; e < T::VEC; ++e) w.e[e] = T::down(v[u * T::VEC + e]);
    if (j + T::VEC <= end) {
      store_vec<T>(row + j, w);
    } else {
#pragma unroll
      for (int e = 0; e < T::VEC; ++e)
        if (j + e < end) row[j + e] = w.e[e];
    }
  }
}
template <int NT>
__device__ __forceinline__ Acc acc_block(Acc a, float c, Acc* red) {
  a = acc_wave(a, c);
  if (NT == 64) return a;
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = a;
  __syncthreads();
  a = red[0];
#pragma unroll
  for (int w = 1; w < NT / 64; ++w) a = acc_join(a, red[w], c);
  return a;
}

// ---- top classes of a stretch of a row ---------------------------------------------------------------------
// The k-th largest of the threads' own maxima is a bound that at least k classes reach; few others do, and
// only the threads whose maximum reaches it look at their classes again.  What reaches the bound is
// collected in LDS and ranked by counting.  Where more classes tie at the bound than LDS holds, the ones
// above it are collected and the ties are filled in from the first on.  Rows with NaN, and rows with
// more classes above the bound than fit, take k rounds of "largest below the last".
constexpr int kCand = 1024;
struct TopShared {
  unsigned long long cand[kCand];
  float maxima[256];
  unsigned long long best[4];
  int count, total[4];
  float bound;
};
template <class T, int NT>
__device__ void row_top(const typename T::S* row, int begin, int end, int k, bool neg, float my_max, bool bad,
                        unsigned long long* out, TopShared& sh) {
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int want = min(k, end - begin);
  if (tid == 0) sh.count = 0;
  sh.maxima[tid] = my_max;
  __syncthreads();
  {
    int rank = 0;
    for (int j = 0; j < NT; ++j) {
      const float o = sh.maxima[j];
      rank += (o > my_max || (o == my_max && j < tid)) ? 1 : 0;
    }
    if (rank == min(k, NT) - 1) sh.bound = my_max;
  }
  __syncthreads();
  const float bound = sh.bound;
  bool slow = bad;
  int n = 0;
  if (!slow) {
    for (int pass = 0; pass < 2; ++pass) {  // 0: all that reach the bound; 1: the ones above it
      if (my_max >= bound) {
        for (int base = begin + wave * kWaveTile; base < end; base += NT * 32) {
          if (pass == 0 && *(volatile int*)&sh.count > kCand) break;
          float v[32];
          row_in<T>(row, base, end, lane, neg, v);
#pragma unroll
          for (int u = 0; u < 32; ++u) {
            const int j = base + tile_class<T>(lane, u);
            if ((pass == 0 ? v[u] >= bound : v[u] > bound) && j < end) {
              const int at = atomicAdd(&sh.count, 1);
              if (at < kCand) sh.cand[at] = key_u64(v[u], j);
            }
          }
        }
      }
      __syncthreads();
      n = sh.count;
      if (n <= kCand) {
        if (pass == 1 && n < want) {  // ties, lowest index first
          __syncthreads();
          for (int base = begin; base < end && n < want; base += NT) {
            const int j = base + tid;
            const float v = j < end ? T::up(row[j]) : 0.f;
            const bool tie = j < end && (neg ? -v : v) == bound;
            const unsigned long long b = __ballot(tie);
            if (lane == 0) sh.total[wave] = __popcll(b);
            __syncthreads();
            int at = n + __popcll(b & ((1ull << lane) - 1));
            for (int w = 0; w < wave; ++w) at += sh.total[w];
            if (tie && at < want) sh.cand[at] = key_u64(neg ? -v : v, j);
            for (int w = 0; w < NT / 64; ++w) n += sh.total[w];
            __syncthreads();
          }
          n = min(n, want);
        }
        break;
      }
      if (pass == 1) slow = true;
      __syncthreads();
      if (tid == 0) sh.count = 0;
      __syncthreads();
    }
  }
  if (!slow) {
    __syncthreads();
    for (int i = tid; i < n; i += NT) {
      const unsigned long long mine = sh.cand[i];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += sh.cand[j] > mine ? 1 : 0;
      if (rank < want) out[rank] = mine;
    }
  } else {
    unsigned long long last = ~0ull;
    for (int r = 0; r < want; ++r) {
      unsigned long long best = 0;
      for (int j = begin + tid; j < end; j += NT) {
        const float v = T::up(row[j]);
        const unsigned long long key = key_u64(neg ? -v : v, j);
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
  for (int i = want + tid; i < k; i += NT) out[i] = 0;  // shorter than k: nothing
  __syncthreads();
}

struct LpOut {
  float *log_prob, *entropy, *top_lp;
  int32_t* top_idx;
  Stats3* stats;
};
template <class T>
__device__ __forceinline__ void lp_row_write(const Prob& p, int64_t row, const typename T::S* xr, const void* index,
                                             const Acc& a, const LpOut& o) {
  const bool neg = p.scale < 0.f;
  const float base = a.m == -kInf ? 0.f : a.m, ln_s = logf(a.s);
  const int t = index ? valid_index(load_index(index, row, p.flags), p.V) : -1;
  float lp = 0.f;
  if (t >= 0) {
    const float v = T::up(xr[t]);
    lp = log_p(neg ? -v : v, base, ln_s, p.scale);
  }
  if (o.log_prob) o.log_prob[row] = lp;
  if (o.entropy) o.entropy[row] = entropy_of(a.s, a.w, ln_s);
  if (o.stats) o.stats[row] = Stats3{base, a.s, a.w};
}
__device__ __forceinline__ void lp_row_top_write(const Prob& p, int64_t row, int rank, unsigned long long key,
                                                 const Acc& a, const LpOut& o) {
  const float base = a.m == -kInf ? 0.f : a.m;
  o.top_lp[row * p.k + rank] = log_p(key_value(key), base, logf(a.s), p.scale);
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
__global__ __launch_bounds__(NT) void lp_row_fwd(Prob p, const typename T::S* __restrict__ x,
                                                 const void* __restrict__ index, LpOut o, Part* __restrict__ parts,
                                                 unsigned long long* __restrict__ part_keys) {
  __shared__ Acc red[NT / 64];
  const int64_t row = blockIdx.x / (unsigned)p.chunks;
  const int chunk = blockIdx.x - (unsigned)row * p.chunks;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const typename T::S* xr = x + row * p.V;
  const int begin = chunk * p.chunk, end = min(p.V, begin + p.chunk);
  const bool neg = p.scale < 0.f;
  Acc a = acc_empty();
  for (int base = begin + wave * kWaveTile; base < end; base += NT * 32) {
    float v[32];
    row_in<T>(xr, base, end, lane, neg, v);
    absorb<true>(a, v, p.c);
  }
  const float my_max = a.m;
  a = acc_block<NT>(a, p.c, red);
  if (p.chunks == 1) {
    if (threadIdx.x == 0) lp_row_write<T>(p, row, xr, index, a, o);
  } else if (threadIdx.x == 0) {
    parts[row * p.chunks + chunk] = Part{a.m, a.s, a.w, 0.f};
  }
  if constexpr (TOP) {
    __shared__ TopShared sh;
    __shared__ unsigned long long best[kMaxEntries];
    row_top<T, NT>(xr, begin, end, p.k, neg, my_max, a.s != a.s, best, sh);
    if ((int)threadIdx.x < p.k) {
      if (p.chunks == 1)
        lp_row_top_write(p, row, threadIdx.x, best[threadIdx.x], a, o);
      else
        part_keys[(row * p.chunks + chunk) * p.k + threadIdx.x] = best[threadIdx.x];
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
  Acc a = acc_empty();
  for (int i = 0; i < p.chunks; ++i) {
    const Part q = parts[row * p.chunks + i];
    a = acc_join(a, Acc{q.m, q.s, q.w}, p.c);
  }
  if (threadIdx.x == 0) lp_row_write<T>(p, row, x + row * p.V, index, a, o);
  const int n = p.chunks * p.k;  // at most kCand
  for (int i = threadIdx.x; i < n; i += 256) keys[i] = part_keys[row * n + i];
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += 256) {
    const unsigned long long mine = keys[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += keys[j] > mine ? 1 : 0;
    if (mine != 0 && rank < p.k) lp_row_top_write(p, row, rank, mine, a, o);
  }
}

template <class T, int NT, bool ENT>
__global__ __launch_bounds__(NT) void lp_row_bwd(Prob p, const typename T::S* __restrict__ x,
                                                 const void* __restrict__ index, const Stats3* __restrict__ stats,
                                                 const float* __restrict__ g_lp,
                                                 const float* __restrict__ g_ent, typename T::S* __restrict__ g) {
  const int64_t row = blockIdx.x / (unsigned)p.chunks;
  const int chunk = blockIdx.x - (unsigned)row * p.chunks;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const typename T::S* xr = x + row * p.V;
  typename T::S* gr = g + row * p.V;
  const int begin = chunk * p.chunk, end = min(p.V, begin + p.chunk);
  const bool neg = p.scale < 0.f;
  const LpCoef r = lp_coef<ENT>(p, row, index, stats, g_lp, g_ent);
  for (int base = begin + wave * kWaveTile; base < end; base += NT * 32) {
    float v[32];
    if (r.dead) {
#pragma unroll
      for (int u = 0; u < 32; ++u) v[u] = 0.f;
    } else {
      row_in<T>(xr, base, end, lane, neg, v);
#pragma unroll
      for (int u = 0; u < 32; ++u) v[u] = lp_grad<ENT>(r, v[u], p.c, 0.f);
      const int rel = r.target - base;
      if ((unsigned)rel < (unsigned)kWaveTile) {
#pragma unroll
        for (int u = 0; u < 32; ++u) v[u] += tile_class<T>(lane, u) == rel ? r.hit : 0.f;
      }
    }
    row_out<T>(gr, base, end, lane, v);
  }
}

// ---- distillation over long rows: every wave holds the whole list, one entry a lane --------------------
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
      const float ts = wave_sum_all(expf(e.value - (tm == -kInf ? 0.f : tm)));
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
__device__ __forceinline__ void ds_row_write(const Prob& p, int64_t row, const typename T::S* xr, const Entry& e,
                                             const Acc& a, float* loss, float4* stats) {
  const bool neg = p.scale < 0.f;
  float v = -kInf;
  if (e.idx >= 0) v = neg ? -T::up(xr[e.idx]) : T::up(xr[e.idx]);
  const float first = e.again ? -kInf : v;
  RowSums r;
  r.m_r = a.m;
  r.s_r = a.s;
  const float m = vmax(a.m, wave_max_all(first));
  r.b = m == -kInf ? 0.f : m;
  r.s = fmaf(a.s, exp2_((a.m - r.b) * p.c), wave_sum_all(exp2_((first - r.b) * p.c)));
  r.ln_s = logf(r.s);
  const bool alive = __any(e.idx >= 0);
  const float qe = e.idx >= 0 ? expf(e.value) : 0.f;
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
__global__ __launch_bounds__(NT) void ds_row_fwd(Prob p, const typename T::S* __restrict__ x,
                                                 const void* __restrict__ teacher, const void* __restrict__ index,
                                                 float* __restrict__ loss, float4* __restrict__ stats,
                                                 Part* __restrict__ parts) {
  __shared__ Acc red[NT / 64];
  const int64_t row = blockIdx.x / (unsigned)p.chunks;
  const int chunk = blockIdx.x - (unsigned)row * p.chunks;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const typename T::S* xr = x + row * p.V;
  const int begin = chunk * p.chunk, end = min(p.V, begin + p.chunk);
  const bool neg = p.scale < 0.f;
  const Entry e = load_entry(p, row, p.chunks == 1 ? teacher : nullptr, index, lane);
  Acc a = acc_empty();
  if (__any(e.idx >= 0)) {  // the same in every wave
    for (int base = begin + wave * kWaveTile; base < end; base += NT * 32) {
      float v[32];
      row_in<T>(xr, base, end, lane, neg, v);
      patch_tile<T>(v, base, lane, e.idx, -kInf);
      absorb<false>(a, v, p.c);
    }
  }
  a = acc_block<NT>(a, p.c, red);
  if (p.chunks > 1) {
    if (threadIdx.x == 0) parts[row * p.chunks + chunk] = Part{a.m, a.s, 0.f, 0.f};
  } else if (wave == 0) {
    ds_row_write<T>(p, row, xr, e, a, loss, stats);
  }
}
template <class T>
__global__ __launch_bounds__(64) void ds_row_join(Prob p, const typename T::S* __restrict__ x,
                                                  const void* __restrict__ teacher, const void* __restrict__ index,
                                                  float* __restrict__ loss, float4* __restrict__ stats,
                                                  const Part* __restrict__ parts) {
  const int64_t row = blockIdx.x;
  const Entry e = load_entry(p, row, teacher, index, threadIdx.x);
  Acc a = acc_empty();
  for (int i = threadIdx.x; i < p.chunks; i += 64) {
    const Part q = parts[row * p.chunks + i];
    a = acc_join(a, Acc{q.m, q.s, 0.f}, p.c);
  }
  a = acc_wave(a, p.c);
  ds_row_write<T>(p, row, x + row * p.V, e, a, loss, stats);
}

template <class T, int NT>
__global__ __launch_bounds__(NT) void ds_row_bwd(Prob p, const typename T::S* __restrict__ x,
                                                 const void* __restrict__ teacher, const void* __restrict__ index,
                                                 const float4* __restrict__ stats, const float* __restrict__ g_loss,
                                                 typename T::S* __restrict__ g) {
  const int64_t row = blockIdx.x / (unsigned)p.chunks;
  const int chunk = blockIdx.x - (unsigned)row * p.chunks;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const typename T::S* xr = x + row * p.V;
  typename T::S* gr = g + row * p.V;
  const int begin = chunk * p.chunk, end = min(p.V, begin + p.chunk);
  const bool neg = p.scale < 0.f;
  const float4 st = stats[row];
  const float up = g_loss[row];
  const bool dead = up == 0.f || st.w == 0.f;
  const float gs = up * p.scale, rest_f = gs * st.y, member_f = gs * st.w;
  Entry e{-1, 0.f, false};
  float with = 0.f;
  if (!dead) {
    e = load_entry(p, row, teacher, index, lane);
    float qe = e.idx >= 0 ? expf(e.value) : 0.f;
    float sum = qe;  // of all entries of this class
    for (int k = 0; k < p.k; ++k) {
      const int other = __builtin_amdgcn_readlane(e.idx, k);
      const float oq = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, qe), k));
      if (k != lane && other == e.idx && other >= 0) sum += oq;
    }
    if (e.idx >= 0) {
      const float v = neg ? -T::up(xr[e.idx]) : T::up(xr[e.idx]);
      with = exp2_((v - st.z) * p.c) * member_f - gs * sum;
    }
    if (e.again) e.idx = -1;
  }
  for (int base = begin + wave * kWaveTile; base < end; base += NT * 32) {
    float v[32];
    if (dead) {
#pragma unroll
      for (int u = 0; u < 32; ++u) v[u] = 0.f;
    } else {
      row_in<T>(xr, base, end, lane, neg, v);
#pragma unroll
      for (int u = 0; u < 32; ++u) v[u] = exp2_((v[u] - st.x) * p.c) * rest_f;
      patch_tile<T>(v, base, lane, e.idx, with);
    }
    row_out<T>(gr, base, end, lane, v);
  }
}

// ---- host side -----------------------------------------------------------------------------------------------
constexpr int64_t kMaxClasses = 1 << 28;   // the order keys hold 29 bits of index
constexpr int kWantWaves = 2048;           // 8 a compute unit: enough loads in flight
constexpr size_t kLdsBudget = 152 * 1024;  // of a block, of the compute unit's 160 KB

struct Plan {
  Prob p;
  bool tile, last;
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
  if (!(d->scale != 0.f) || !(d->scale - d->scale == 0.f)) return DW_ERR_ARG;  // zero, NaN, infinite
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
  p.c = (d->scale < 0.f ? -d->scale : d->scale) * kLog2e;
  p.flags = d->flags;
  p.chunks = 1;
  p.chunk = p.V;
  P.ws = 0;
  P.last = (d->flags & DW_DIST_LAST) || d->inner == 1;
  const int64_t tiles = P.last ? (p.rows + 63) / 64 : d->outer * ((d->inner + 63) / 64);
  const int esize = d->dtype == DW_DTYPE_F32 ? 4 : 2;
  P.tile = !P.last || (p.V <= 2048 && tiles * 4 >= kWantWaves / 4);
  if (P.tile) {
    const int stage = P.last ? kSegBytes / esize : 32;
    const int stages = (p.V + stage - 1) / stage;
    P.nw = 1;
    while (P.nw < 16 && tiles * P.nw < kWantWaves && P.nw * 2 <= stages) P.nw *= 2;
    const size_t per_wave = kStageBytes + (distill ? 512 : 64 * (12 + 8 * 16)), shared = distill ? p.k * 768 : 0;
    while (P.nw > 1 && P.nw * per_wave + shared > kLdsBudget) P.nw /= 2;
    p.cpw = (stages + P.nw - 1) / P.nw * stage;
    if (tiles > 0x7fffffff) return DW_ERR_SHAPE;
    P.grid = (unsigned)tiles;
    return DW_OK;
  }
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
  if (p.rows > 0x7fffffff / p.chunks) return DW_ERR_SHAPE;
  P.grid = (unsigned)(p.rows * p.chunks);
  if (!backward && p.chunks > 1) {
    P.ws = parts_bytes(p.rows, p.chunks);
    if (!distill) P.ws += ((size_t)p.rows * p.chunks * p.k * 8 + 255) / 256 * 256;
  }
  return DW_OK;
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

template <class T, bool LAST, int K>
int lp_tile_launch(const Plan& P, const void* x, const void* index, const LpOut& o, hipStream_t st) {
  const size_t lds = (LAST ? P.nw * kStageBytes : 0) + (P.nw > 1 ? P.nw * 64 * (12 + 8 * K) : 0);
  if (int rc = allow_lds(lp_tile_fwd<T, LAST, K>, lds)) return rc;
  lp_tile_fwd<T, LAST, K><<<P.grid, P.nw * 64, lds, st>>>(P.p, (const typename T::S*)x, index, o.log_prob, o.entropy,
                                                          o.top_lp, o.top_idx, o.stats);
  return launched();
}
template <class T>
int lp_fwd(const Plan& P, const void* x, const void* index, const LpOut& o, void* ws, hipStream_t st) {
  const int k = P.p.k;
  if (P.tile) {
    if (P.last) {
      if (k == 0) return lp_tile_launch<T, true, 0>(P, x, index, o, st);
      if (k <= 4) return lp_tile_launch<T, true, 4>(P, x, index, o, st);
      if (k <= 8) return lp_tile_launch<T, true, 8>(P, x, index, o, st);
      return lp_tile_launch<T, true, 16>(P, x, index, o, st);
    }
    if (k == 0) return lp_tile_launch<T, false, 0>(P, x, index, o, st);
    if (k <= 4) return lp_tile_launch<T, false, 4>(P, x, index, o, st);
    if (k <= 8) return lp_tile_launch<T, false, 8>(P, x, index, o, st);
    return lp_tile_launch<T, false, 16>(P, x, index, o, st);
  }
  Part* parts = (Part*)ws;
  unsigned long long* keys = (unsigned long long*)((char*)ws + parts_bytes(P.p.rows, P.p.chunks));
  const typename T::S* xs = (const typename T::S*)x;
  if (P.nt == 64) {
    if (k) lp_row_fwd<T, 64, true><<<P.grid, 64, 0, st>>>(P.p, xs, index, o, parts, keys);
    else lp_row_fwd<T, 64, false><<<P.grid, 64, 0, st>>>(P.p, xs, index, o, parts, keys);
  } else {
    if (k) lp_row_fwd<T, 256, true><<<P.grid, 256, 0, st>>>(P.p, xs, index, o, parts, keys);
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
    if (P.last) {
      const size_t lds = P.nw * kStageBytes;
      if (int rc = allow_lds(lp_tile_bwd<T, true, ENT>, lds)) return rc;
      lp_tile_bwd<T, true, ENT><<<P.grid, P.nw * 64, lds, st>>>(P.p, (const S*)x, index, stats, g_lp, g_ent, (S*)g);
    } else {
      lp_tile_bwd<T, false, ENT><<<P.grid, P.nw * 64, 0, st>>>(P.p, (const S*)x, index, stats, g_lp, g_ent, (S*)g);
    }
  } else if (P.nt == 64) {
    lp_row_bwd<T, 64, ENT><<<P.grid, 64, 0, st>>>(P.p, (const S*)x, index, stats, g_lp, g_ent, (S*)g);
  } else {
    lp_row_bwd<T, 256, ENT><<<P.grid, 256, 0, st>>>(P.p, (const S*)x, index, stats, g_lp, g_ent, (S*)g);
  }
  return launched();
}
template <class T, bool LAST>
int ds_tile_launch(const Plan& P, bool backward, const void* x, const void* teacher, const void* index, float* loss,
                   float4* stats, const float* g_loss, void* g, hipStream_t st) {
  using S = typename T::S;
  const size_t lds = P.nw * (size_t)distill_stage_bytes<LAST>() + (size_t)P.p.k * 768 + P.nw * 512;
  if (backward) {
    if (int rc = allow_lds(ds_tile_bwd<T, LAST>, lds)) return rc;
    ds_tile_bwd<T, LAST><<<P.grid, P.nw * 64, lds, st>>>(P.p, (const S*)x, teacher, index, stats, g_loss, (S*)g);
  } else {
    if (int rc = allow_lds(ds_tile_fwd<T, LAST>, lds)) return rc;
    ds_tile_fwd<T, LAST><<<P.grid, P.nw * 64, lds, st>>>(P.p, (const S*)x, teacher, index, loss, stats);
  }
  return launched();
}
template <class T>
int ds_run(const Plan& P, bool backward, const void* x, const void* teacher, const void* index, float* loss,
           float4* stats, const float* g_loss, void* g, void* ws, hipStream_t st) {
  using S = typename T::S;
  if (P.tile)
    return P.last ? ds_tile_launch<T, true>(P, backward, x, teacher, index, loss, stats, g_loss, g, st)
                  : ds_tile_launch<T, false>(P, backward, x, teacher, index, loss, stats, g_loss, g, st);
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
  float4* s4 = (float4*)const_cast<float*>(stats);
  hipStream_t st = (hipStream_t)stream;
  switch (d->dtype) {
    case DW_DTYPE_F32: return ds_run<F32>(P, true, logits, teacher, teacher_index, nullptr, s4, grad_loss, grad_logits, nullptr, st);
    case DW_DTYPE_BF16: return ds_run<BF16>(P, true, logits, teacher, teacher_index, nullptr, s4, grad_loss, grad_logits, nullptr, st);
    default: return ds_run<F16>(P, true, logits, teacher, teacher_index, nullptr, s4, grad_loss, grad_logits, nullptr, st);
  }
}
