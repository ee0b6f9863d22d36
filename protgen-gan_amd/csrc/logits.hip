// Operators over rows of vocabulary logits: a teacher's top entries with the log-mass of the rest, distillation from such
// records (loss, gradient, both in one call), and sampling under temperature / top-k / top-p / min-p from given noise.
//
// Entries of a row are ordered by value, ties by the lower index: one 64-bit key per entry, (value bits made monotone) << 32 |
// ~index, is unique, so "the first n entries of a row" is always "the entries whose key is at least B" for one key B.
// NaN counts as -inf, -0 as +0.
#include "../../include/protgen_hip.h"
#include "pg_common.h"
#include <float.h>
#include <math.h>

namespace {

constexpr int MAX_K = 1024;
constexpr int MAX_VOCAB = 1 << 24;  // sampling: one less, so that a row of weights of 2^40 each sums to less than 2^64
constexpr float MIN_TAU = 1e-30f, MAX_TAU = 1e30f;
constexpr double LOG2E = 1.4426950408889634074;
constexpr double LN2 = 0.69314718055994530942;

__device__ __forceinline__ float no_nan(float x) { return x == x ? x : -INFINITY; }
__device__ __forceinline__ uint32_t value_key(float x) {
  x = x + 0.0f;  // -0 -> +0
  if (x != x) x = -INFINITY;
  const uint32_t b = __float_as_uint(x);
  return b ^ (((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k);
}
__device__ __forceinline__ uint64_t entry_key(float x, uint32_t i) { return ((uint64_t)value_key(x) << 32) | (uint32_t)~i; }

__device__ __forceinline__ void unpack(uint4 d, float (&o)[4]) {
  o[0] = __uint_as_float(d.x); o[1] = __uint_as_float(d.y); o[2] = __uint_as_float(d.z); o[3] = __uint_as_float(d.w);
}
__device__ __forceinline__ void unpack(uint4 d, float (&o)[8]) {
  o[0] = __uint_as_float(d.x << 16); o[1] = __uint_as_float(d.x & 0xffff0000u);
  o[2] = __uint_as_float(d.y << 16); o[3] = __uint_as_float(d.y & 0xffff0000u);
  o[4] = __uint_as_float(d.z << 16); o[5] = __uint_as_float(d.z & 0xffff0000u);
  o[6] = __uint_as_float(d.w << 16); o[7] = __uint_as_float(d.w & 0xffff0000u);
}
// f(index, value) over the n elements at p: elements up to the first 16-byte boundary and behind the last whole 16 bytes one by
// one, the rest in 16-byte loads, four in flight per thread (with one, a pass over a row is sixteen memory latencies in a row).
template <typename T, int NT, typename F> __device__ __forceinline__ void each(const T* p, int n, F f) {
  constexpr int E = 16 / (int)sizeof(T);
  int head = (int)((16 - ((uintptr_t)p & 15)) & 15) / (int)sizeof(T);
  if (head > n) head = n;
  const int nv = (n - head) / E, tail = head + nv * E;
  const uint4* vec = reinterpret_cast<const uint4*>(p + head);
  if ((int)threadIdx.x < nv) {
    uint4 d[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) d[u] = vec[min((int)threadIdx.x + u * NT, nv - 1)];
#pragma unroll 1
    for (int v = threadIdx.x; v < nv; v += NT) {
      float o[E];
      unpack(d[0], o);
      d[0] = d[1]; d[1] = d[2]; d[2] = d[3];
      d[3] = vec[min(v + 4 * NT, nv - 1)];
#pragma unroll
      for (int e = 0; e < E; ++e) f(head + v * E + e, o[e]);
    }
  }
#pragma unroll 1
  for (int i = (int)threadIdx.x < head ? (int)threadIdx.x : tail + (int)threadIdx.x - head; i < n; i += i < head ? n : NT)
    f(i, to_f32<T>(p[i]));
}

template <int NT, typename T, typename Op> __device__ __forceinline__ T block_all(T v, T* lds, Op op) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = op(v, __shfl_xor(v, o, 64));
  if (NT == 64) return v;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  v = lds[0];
#pragma unroll
  for (int w = 1; w < NT / 64; ++w) v = op(v, lds[w]);
  return v;
}
template <int NT> __device__ __forceinline__ double block_sum(double v, double* lds) {
  return block_all<NT>(v, lds, [](double a, double b) { return a + b; });
}
template <int NT> __device__ __forceinline__ float block_max(float v, float* lds) {
  return block_all<NT>(v, lds, [](float a, float b) { return fmaxf(a, b); });
}

// A sum of exponentials held as m, s: sum = s * 2^(m c).  m starts at the lowest finite value, so that neither an empty sum nor
// entries of -inf ever form inf - inf.
struct ExpSum { float m, s; };
__device__ __forceinline__ void exp_sum_add(ExpSum& a, float x, float c) {
  if (x > a.m) {
    a.s *= __builtin_amdgcn_exp2f((a.m - x) * c);
    a.m = x;
  }
  a.s += __builtin_amdgcn_exp2f((x - a.m) * c);
}
__device__ __forceinline__ ExpSum exp_sum_join(ExpSum a, ExpSum b, float c) {
  const float m = fmaxf(a.m, b.m);
  return {m, a.s * __builtin_amdgcn_exp2f((a.m - m) * c) + b.s * __builtin_amdgcn_exp2f((b.m - m) * c)};
}
// N such sums over the workgroup at once: each wave's by shuffles, the waves' through LDS (4 * N words per wave) behind one barrier.
template <int NT, int N> __device__ __forceinline__ void block_exp_sums(ExpSum (&a)[N], float c, float2* lds) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float m = a[i].m;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    float s = a[i].s * __builtin_amdgcn_exp2f((a[i].m - m) * c);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    a[i] = {m, s};
    if (NT > 64 && (threadIdx.x & 63) == 0) lds[(threadIdx.x >> 6) * N + i] = make_float2(m, s);
  }
  if (NT == 64) return;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    ExpSum t = {lds[i].x, lds[i].y};
#pragma unroll
    for (int w = 1; w < NT / 64; ++w) t = exp_sum_join(t, {lds[w * N + i].x, lds[w * N + i].y}, c);
    a[i] = t;
  }
}
template <int NT> __device__ __forceinline__ ExpSum block_exp_sum(ExpSum a, float c, float* lds) {
  const float m = block_max<NT>(a.m, lds);
  const float s = block_all<NT>(a.s * __builtin_amdgcn_exp2f((a.m - m) * c), lds, [](float x, float y) { return x + y; });
  return {m, s};
}

// 2^t in 64 bits, 2^-1022 for every t below: 2^t = 2^n 2^f, |f| <= 1/2, the Taylor series of 2^f to degree 9 (remainder below 8e-12).
__device__ __forceinline__ double exp2_f64(double t) {
  t = fmax(t, -1022.0);
  const double n = rint(t), f = t - n;
  double p = 1.01780860092396959520e-7;           // ln(2)^9 / 9!
  p = fma(p, f, 1.32154867901443052734e-6);
  p = fma(p, f, 1.52527338040598376946e-5);
  p = fma(p, f, 1.54035303933816060656e-4);
  p = fma(p, f, 1.33335581464284411157e-3);
  p = fma(p, f, 9.61812910762847687873e-3);
  p = fma(p, f, 5.55041086648215761801e-2);
  p = fma(p, f, 2.40226506959100694072e-1);
  p = fma(p, f, 6.93147180559945286227e-1);
  p = fma(p, f, 1.0);
  return ldexp(p, (int)n);
}

// NaN kept (exp2_f64 takes it for -1022)
__device__ __forceinline__ double exp2_or_nan(double t) { return t == t ? exp2_f64(t) : t; }

// log s in 64 bits for s > 0: the fp32 logarithm y and what is left, s e^-y - 1 (below 2^-20: its own logarithm to 2^-40).
__device__ __forceinline__ double log_f64(double s) {
  const double y = (double)logf((float)s);
  const double e = s * exp2_f64(-y * LOG2E) - 1.0;
  return s > 0.0 && s < (double)INFINITY ? y + e : y;  // (0, infinite, NaN: as logf)
}

// ------------------------------------------------------------------ the largest entries of a segment of a row, kept in registers
// A row is cut into segments of NT * VPT 16-byte vectors; a workgroup loads one whole segment into registers (all its loads in
// flight at once) and reads it once.  The K-th largest of the threads' maxima is a lower bound of the segment's K-th largest entry
// and not far below it (64 of 256 maxima leave about 75 entries above the bound, 128 about 180; above that each thread's vectors
// form four groups), found by eight rounds of counting on the upper 16 bits of their keys.  Vectors with an entry above the bound go to
// LDS, all others into the sum of exponentials.  Where too many entries tie at the bound, the K-th key's digits are found by
// counting over the segment instead.
constexpr int MERGE = 4096;  // keys of all segments of one row in LDS
constexpr int MAX_SEG_K = 512;
constexpr int max_cap(int K) { return K > 128 ? 1088 : 512; }  // keys a segment may leave

// The largest of three.  Quiet NaN is passed over, but a signalling one makes its first maximum a quiet NaN, with which the other
// operand is lost: only for operands that are none, or where a NaN decides the result anyway.  The compiler forms the same
// instruction from two fmaxf, so raw entries do not go through those either.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
// The largest of three, NaN if one is.
__device__ __forceinline__ float maximum3(float a, float b, float c) {
  float r;
  asm("v_maximum3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
// The largest entry of a vector.  STICKY: NaN if one is NaN; else for vectors without NaN, and for sums that keep NaN, where any
// largest will do beside one.
template <int E, bool STICKY = false> __device__ __forceinline__ float vec_max(const float (&o)[E]) {
  float m = -INFINITY;
#pragma unroll
  for (int e = 0; e + 1 < E; e += 2) m = STICKY ? maximum3(m, o[e], o[e + 1]) : max3(m, o[e], o[e + 1]);
  return m;
}
// The exponentials of E entries of which vm is the largest, with one rescaling for all of them.  NaN as -inf (looked for in the
// sum, not entry by entry), or (KEEP_NAN) kept.
template <int E, bool KEEP_NAN = false> __device__ __forceinline__ void exp_sum_vec(ExpSum& a, const float (&o)[E], float vm, float c) {
  const float m = max3(a.m, a.m, vm);
  float s = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) s += __builtin_amdgcn_exp2f((o[e] - m) * c);
  if (!KEEP_NAN && s != s) {
    s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) s += o[e] == o[e] ? __builtin_amdgcn_exp2f((o[e] - m) * c) : 0.f;
  }
  a.s = a.s * __builtin_amdgcn_exp2f((a.m - m) * c) + s;
  a.m = m;
}
// The same sum for entries of one set with a fixed reference m, an entry of the set: one multiply-add, one exponential and one
// addition per entry.  m c is rounded once (mc) and the sum corrected by the difference at the end.  Entries far above m make it
// large: past 2^90 a join with a sum whose m is 2^126 larger would flush its factor, and lose more than 2^-36 of the whole.  Past
// 2^29 the rounding of m c (half an ulp: above 16) could do as much.  Then ok() is false and the caller takes the way above, as
// where there is no usable m.
struct FixedSum {
  float m, mc, s, c;
  __device__ __forceinline__ FixedSum(float reference, float scale) : m(reference), mc(reference * scale), s(0.f), c(scale) {}
  __device__ __forceinline__ bool ok() const { return fabsf(mc) < 0x1p29f && s < 0x1p90f; }  // (false for NaN)
  template <int E> __device__ __forceinline__ void add(const float (&o)[E]) {
    float t[2] = {0.f, 0.f};
#pragma unroll
    for (int e = 0; e < E; ++e) t[e & 1] += __builtin_amdgcn_exp2f(fmaf(o[e], c, -mc));
    s += t[0] + t[1];
  }
  __device__ __forceinline__ ExpSum end() const { return {m, s * __builtin_amdgcn_exp2f(-fmaf(m, c, -mc))}; }
};
// 16 bytes of a row that is read once: past the caches (1024 x 131072 bf16, k 64: 91 us against 95 with ordinary loads; loss and
// gradient of 4096 x 32768 bf16: 133 against 144).
__device__ __forceinline__ uint4 load_once(const void* p) {
  typedef __attribute__((ext_vector_type(4))) uint32_t u4;
  const u4 v = __builtin_nontemporal_load(reinterpret_cast<const u4*>(p));
  return make_uint4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void exp_sum_one(ExpSum& a, float x, float c) {
  const float o[1] = {x};
  exp_sum_vec<1>(a, o, no_nan(x), c);
}

// exp((x - m) / temperature) for x <= m in whole multiples of 2^-40: sums of these are the same in any order.
__device__ __forceinline__ uint64_t fixed_weight(float x, float m, float c) {
  return x == m ? 1ull << 40 : (uint64_t)(__builtin_amdgcn_exp2f((x - m) * c) * 0x1p40f);
}

// The largest multiple B of 2^lo with at least K of the workgroup's keys k[r], r < used, at B or above (0: there are fewer), two
// bits a round; a wave's three counts share a word.
template <int NT, int R, typename Key>
__device__ __forceinline__ Key kth_bound(const Key (&k)[R], int used, int K, int hi, int lo, uint64_t (*counts)[16]) {
  constexpr int NW = NT / 64;
  Key bound = 0;
  for (int b = hi; b >= lo; b -= 2) {
    uint64_t cnt = 0;
#pragma unroll
    for (int g = 0; g < R; ++g) {
      if (g >= used) break;
#pragma unroll
      for (int i = 0; i < 3; ++i) cnt += (uint64_t)__popcll(__ballot(k[g] >= (bound | ((Key)(i + 1) << b)))) << (20 * i);
    }
    if (NW > 1) {  // (two buffers: a round's counts are read while the next round's are written)
      uint64_t* w = counts[(b >> 1) & 1];
      if ((threadIdx.x & 63) == 0) w[threadIdx.x >> 6] = cnt;
      __syncthreads();
      cnt = 0;
#pragma unroll
      for (int j = 0; j < NW; ++j) cnt += w[j];
    }
    const int c1 = (int)cnt & 0xfffff, c2 = (int)(cnt >> 20) & 0xfffff, c3 = (int)(cnt >> 40);
    bound |= (Key)(c3 >= K ? 3 : c2 >= K ? 2 : c1 >= K ? 1 : 0) << b;
  }
  return bound;
}

// The first i < n at which get(0) + ... + get(i) reaches need, and the sum before it; i = n, the sum of all, if none does.
struct CutAt { int i; uint64_t before; };
template <int NT, typename L, typename F> __device__ __forceinline__ CutAt find_cut(int n, uint64_t need, L& l, F get) {
  const int per = (n + NT - 1) / NT, a = min((int)threadIdx.x * per, n), b = min(a + per, n);
  uint64_t sum = 0;
  for (int i = a; i < b; ++i) sum += get(i);
  uint64_t upto = sum;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint64_t v = __shfl_up(upto, o, 64);
    if ((int)(threadIdx.x & 63) >= o) upto += v;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 63) l.wave[threadIdx.x >> 6] = upto;
  if (threadIdx.x == 0) l.cut = n;
  __syncthreads();
  uint64_t all = 0, off = 0;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) {
    if (w < (int)(threadIdx.x >> 6)) off += l.wave[w];
    all += l.wave[w];
  }
  upto += off;
  uint64_t before = upto - sum;
  if (before < need && upto >= need) {
    int i = a;
    for (uint64_t g; i < b && before + (g = get(i)) < need; ++i) before += g;
    l.cut = i;
    l.cut_before = before;
  }
  __syncthreads();
  return l.cut < n ? CutAt{l.cut, l.cut_before} : CutAt{n, all};
}

template <int NT, bool MANY> struct SegLds {  // MANY: for K above 128
  uint64_t wave[16];
  static constexpr int STAGE = MANY ? 1024 : 256;  // vectors that may hold an entry above the bound (k 512: about 700)
  static constexpr int LIST = MANY ? 2048 : 512;  // keys (a power of two of at least max_cap)
  __align__(16) uint64_t list[LIST];
  uint4 vec[STAGE];
  int at[STAGE];
  uint32_t n_vec, n;
  uint64_t counts[2][16];
  uint64_t cut_before;
  int cut;
  float red[16];
};
struct SegHead {      // what a segment leaves for the merge
  uint64_t level;     // every entry of the segment with at least this key is in its list
  float m, s;         // the sum over its other entries
  uint32_t n, pad[3];
};

// A word of one or two entries, those marked in `in` replaced by -inf.
template <typename T> __device__ __forceinline__ uint32_t without(uint32_t d, uint32_t in) {
  if (sizeof(T) == 4) return in & 1 ? 0xff800000u : d;
  d = in & 1 ? (d & 0xffff0000u) | 0xff80u : d;
  return in & 2 ? (d & 0xffffu) | 0xff800000u : d;
}

template <typename T, int NT, int VPT> struct Segment {
  static constexpr int E = 16 / (int)sizeof(T), VECS = NT * VPT;
  uint4 d[VPT];
  float ends[2];     // this thread's entry of those before the first / behind the last whole vector
  int end_at[2];     // their indexes, -1: none
  int base, nv;

  __device__ __forceinline__ int index(int j) const { return base + (j * NT + (int)threadIdx.x) * E; }
  __device__ __forceinline__ bool has(int j) const { return j * NT + (int)threadIdx.x < nv; }
  __device__ __forceinline__ void place(const T* row, int V, int seg, int nseg) {
    int head = (int)((16 - ((uintptr_t)row & 15)) & 15) / (int)sizeof(T);
    if (head > V) head = V;
    const int all = (V - head) / E, tail = head + all * E;
    base = head + seg * VECS * E;
    nv = all - seg * VECS;
    nv = nv < 0 ? 0 : nv > VECS ? VECS : nv;
    end_at[0] = seg == 0 && (int)threadIdx.x < head ? (int)threadIdx.x : -1;
    end_at[1] = seg == nseg - 1 && (int)threadIdx.x < V - tail ? tail + (int)threadIdx.x : -1;
  }
  __device__ __forceinline__ void load(const T* row, int V, int seg, int nseg) {
    place(row, V, seg, nseg);
    const uint32_t none = sizeof(T) == 2 ? 0xff80ff80u : 0xff800000u;  // -inf
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      d[j] = make_uint4(none, none, none, none);
      if (has(j)) d[j] = load_once(row + index(j));
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) ends[i] = end_at[i] >= 0 ? to_f32<T>(row[end_at[i]]) : -INFINITY;
  }
  // Unpacked anew in every phase: kept from one to the next, the fp32 values of a bf16 segment would not fit the registers.
  __device__ __forceinline__ void fresh() {
#pragma unroll
    for (int j = 0; j < VPT; ++j) asm volatile("" : "+v"(d[j].x), "+v"(d[j].y), "+v"(d[j].z), "+v"(d[j].w));
  }
  // Vector j without the entries marked in `in`, one bit each.
  __device__ __forceinline__ void remove(int j, uint32_t in) {
    d[j].x = without<T>(d[j].x, in);
    d[j].y = without<T>(d[j].y, in >> E / 4);
    d[j].z = without<T>(d[j].z, in >> E / 2);
    d[j].w = without<T>(d[j].w, in >> E * 3 / 4);
  }
  // f(value, index) over this thread's entries of segments seg .. seg + count - 1, read again from memory
  template <typename F> static __device__ __forceinline__ void entries(const T* row, int V, int seg, int count, int nseg, F f) {
#pragma unroll 1
    for (int s = seg; s < seg + count; ++s) {
      Segment at;
      at.place(row, V, s, nseg);
#pragma unroll 1
      for (int j = 0; j < VPT && at.has(j); ++j) {
        float o[E];
        unpack(*reinterpret_cast<const uint4*>(row + at.index(j)), o);
#pragma unroll
        for (int e = 0; e < E; ++e) f(o[e], at.index(j) + e);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (at.end_at[i] >= 0) f(to_f32<T>(row[at.end_at[i]]), at.end_at[i]);
    }
  }
};

// Leaves the keys of the largest entries of segments seg .. seg + count - 1 (of nseg in the row) in l.list (n of them, at most cap,
// in no order; at least K if there are as many), the sum over the other entries in rest (per thread), and the level.  FINITE:
// entries of -inf are never listed.  Over several segments the threads' maxima, and with them the bound, run on.
template <typename T, int NT, int VPT, bool FINITE, bool MANY>
__device__ __forceinline__ int collect(const T* row, int V, int seg, int count, int nseg, int K, int cap, float c, SegLds<NT, MANY>& l,
                                       uint64_t& level, ExpSum& rest) {
  typedef Segment<T, NT, VPT> Seg;
  constexpr int E = Seg::E, STAGE = SegLds<NT, MANY>::STAGE, LIST = SegLds<NT, MANY>::LIST;
  uint64_t* list = l.list;
  constexpr int GROUPS = MANY ? 4 : 1;  // of a thread's vectors
  Seg sg;
  sg.load(row, V, seg, nseg);
  float gm[GROUPS], thr = -INFINITY;
#pragma unroll
  for (int g = 0; g < GROUPS; ++g) gm[g] = -INFINITY;
  rest = {-FLT_MAX, 0.f};
  bool over = false;
  if (threadIdx.x == 0) l.n = 0;
#pragma unroll 1
  for (int s = 0;; ++s) {
    float low = INFINITY, sm[GROUPS], nan = 0.f;
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) sm[g] = -INFINITY;
    sg.fresh();
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      float o[E];
      unpack(sg.d[j], o);
      const float vm = vec_max<E, true>(o);
      sm[j % GROUPS] = maximum3(sm[j % GROUPS], sm[j % GROUPS], vm);
      low = sg.has(j) && vm < low ? vm : low;
    }
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) nan = maximum3(nan, nan, sm[g]);
    if (nan != nan) {  // a NaN among this thread's entries: -inf from here on
      sg.fresh();
      low = INFINITY;
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) sm[g] = -INFINITY;
#pragma unroll
      for (int j = 0; j < VPT; ++j) {
        float o[E];
        unpack(sg.d[j], o);
        uint32_t in = 0;
        float vm = -INFINITY;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          in |= (o[e] != o[e]) << e;
          vm = o[e] > vm ? o[e] : vm;
        }
        sg.remove(j, in);
        sm[j % GROUPS] = vm > sm[j % GROUPS] ? vm : sm[j % GROUPS];
        low = sg.has(j) && vm < low ? vm : low;
        __builtin_amdgcn_sched_barrier(0);
      }
    }
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) gm[g] = fmaxf(gm[g], sm[g]);
#pragma unroll
    for (int i = 0; i < 2; ++i) gm[0] = sg.ends[i] > gm[0] ? sg.ends[i] : gm[0];
    uint32_t mk[GROUPS];
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) mk[g] = gm[g] > -INFINITY ? value_key(gm[g]) : 0;
    if (threadIdx.x == 0) l.n_vec = 0;
    const uint32_t bound = kth_bound<NT>(mk, GROUPS, K, 30, 16, l.counts);
    thr = bound > 0x007fffffu ? key_value(bound) : -INFINITY;
    __syncthreads();
    sg.fresh();
    // the sum over vectors without an entry above the bound: against the smallest of the vectors' maxima if that is one of them
    FixedSum sum(low < thr && low > -INFINITY ? low : INFINITY, c);
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      float o[E];
      unpack(sg.d[j], o);
      const float vm = vec_max<E>(o);
      if (vm >= thr && (!FINITE || vm > -INFINITY) && sg.has(j)) {
        const uint32_t p = atomicAdd(&l.n_vec, 1u);
        if (p < STAGE) {
          l.vec[p] = sg.d[j];
          l.at[p] = sg.index(j);
        }
      } else {
        sum.template add<E>(o);
      }
    }
    ExpSum part = sum.end();
    if (!sum.ok()) {  // (vectors without an entry above -inf or all with one above the bound, entries far apart)
      part = {-FLT_MAX, 0.f};
      sg.fresh();
#pragma unroll
      for (int j = 0; j < VPT; ++j) {
        float o[E];
        unpack(sg.d[j], o);
        const float vm = vec_max<E>(o);
        if (!(vm >= thr && (!FINITE || vm > -INFINITY) && sg.has(j))) exp_sum_vec<E>(part, o, vm, c);
      }
    }
    rest = s == 0 ? part : exp_sum_join(rest, part, c);
    auto take = [&](float x, int i) {
      x = no_nan(x);
      const bool in = x >= thr && (!FINITE || x > -INFINITY);
      if (in) {
        const uint32_t p = atomicAdd(&l.n, 1u);
        if (p < LIST) list[p] = entry_key(x, i);
      }
      return in;
    };
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (sg.end_at[i] >= 0 && !take(sg.ends[i], sg.end_at[i])) exp_sum_one(rest, sg.ends[i], c);
    if (s + 1 < count) sg.load(row, V, seg + s + 1, nseg);  // (on its way while the staged vectors are looked through)
    __syncthreads();
    const int n_vec = l.n_vec, staged = n_vec < STAGE ? n_vec : STAGE;
    float most = -INFINITY;  // the largest entry that a vector with a listed one brings along
    for (int i = threadIdx.x; i < staged; i += NT) {
      float o[E];
      unpack(l.vec[i], o);
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (!take(o[e], l.at[i] + e) && o[e] > most) most = o[e];
    }
    most = block_max<NT>(most, l.red);
    if (most > -INFINITY) {  // the staged vectors are in no fixed order: their sum is one of whole multiples of 2^-40 of the largest
      uint64_t sum = 0;
      for (int i = threadIdx.x; i < staged; i += NT) {
        float o[E];
        unpack(l.vec[i], o);
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (o[e] < thr) sum += fixed_weight(o[e], most, c);
      }
      sum = block_all<NT>(sum, l.wave, [](uint64_t a, uint64_t b) { return a + b; });
      if (threadIdx.x == 0) rest = exp_sum_join(rest, {most, (float)sum * 0x1p-40f}, c);
    }
    __syncthreads();
    over = over || n_vec > STAGE;
    if (s + 1 == count) break;
  }
  int n = l.n;
  level = thr > -INFINITY ? (uint64_t)value_key(thr) << 32 : 0;
  if (over || n > cap) {  // too many at the bound: the K-th key by its digits, ten bits at a time, until at most cap keys are left
    uint32_t* bins = reinterpret_cast<uint32_t*>(l.vec);
    uint64_t prefix = 0;
    int above = 0;
    for (int shift = 54, last = 64;; last = shift, shift = shift > 10 ? shift - 10 : 0) {
      __syncthreads();
      for (int i = threadIdx.x; i < 1024; i += NT) bins[i] = 0;
      __syncthreads();
      Seg::entries(row, V, seg, count, nseg, [&](float x, int i) {
        const uint64_t k = entry_key(x, i);
        if ((last == 64 || k >> last == prefix) && (!FINITE || x > -INFINITY))
          atomicAdd(&bins[(int)(k >> shift) & ((1 << (last - shift)) - 1)], 1u);
      });
      __syncthreads();
      const int digits = 1 << (last - shift);
      const CutAt at = find_cut<NT>(digits, K - above, l, [&](int i) { return (uint64_t)bins[digits - 1 - i]; });
      const int digit = digits - 1 - min(at.i, digits - 1);
      above += (int)at.before;
      prefix = prefix << (last - shift) | digit;
      level = prefix << shift;
      if (above + (int)bins[digit] <= cap || shift == 0) break;
    }
    rest = {-FLT_MAX, 0.f};
    __syncthreads();
    if (threadIdx.x == 0) l.n = 0;
    __syncthreads();
    Seg::entries(row, V, seg, count, nseg, [&](float x, int i) {
      const uint64_t k = entry_key(x, i);
      if (k >= level && (!FINITE || x > -INFINITY)) list[atomicAdd(&l.n, 1u)] = k;
      else exp_sum_one(rest, x, c);
    });
    __syncthreads();
    n = l.n;
  }
  return n;
}

// list[0..n) in LDS, largest first; at least P = the next power of two of room
template <int NT> __device__ __forceinline__ void sort_keys(uint64_t* list, int n) {
  if (n <= NT && n <= 504) {  // few: each key's rank by counting, two barriers instead of one per step of a network
    const uint64_t mine = (int)threadIdx.x < n ? list[threadIdx.x] : 0;
    const int padded = (n + 7) & ~7;
    if (n + (int)threadIdx.x < padded) list[n + threadIdx.x] = 0;
    __syncthreads();
    int rank = 0;
    if ((int)(threadIdx.x & ~63u) < n)  // (whole waves)
#pragma unroll 1
      for (int j = 0; j < padded; j += 8) {  // (four reads in flight: one at a time, each step waits for LDS)
        ulonglong2 d[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) d[u] = *reinterpret_cast<const ulonglong2*>(list + j + 2 * u);
#pragma unroll
        for (int u = 0; u < 4; ++u) rank += (d[u].x > mine) + (d[u].y > mine);
      }
    __syncthreads();
    if ((int)threadIdx.x < n) list[rank] = mine;
    __syncthreads();
    return;
  }
  int P = 1;
  while (P < n) P <<= 1;
  for (int i = n + threadIdx.x; i < P; i += NT) list[i] = 0;
  for (int size = 2; size <= P; size <<= 1)
    for (int stride = size >> 1; stride > 0; stride >>= 1) {
      __syncthreads();
      for (int i = threadIdx.x; i < P / 2; i += NT) {
        const int a = 2 * i - (i & (stride - 1)), b = a + stride;
        const uint64_t x = list[a], y = list[b];
        if ((x < y) == ((a & size) == 0)) { list[a] = y; list[b] = x; }
      }
    }
  __syncthreads();
}

template <typename T, int NT>
__device__ __forceinline__ void top_finish(uint64_t* list, int n, int K, float tau, float c, ExpSum rest, float* red, T* values,
                                           int32_t* ids, float* rest_out) {
  sort_keys<NT>(list, n);
  for (int i = threadIdx.x; i < n; i += NT) {
    const float x = key_value((uint32_t)(list[i] >> 32));
    if (i < K) {
      values[i] = from_f32<T>(x);
      ids[i] = (int32_t)~(uint32_t)list[i];
    } else {
      exp_sum_one(rest, x, c);
    }
  }
  rest = block_exp_sum<NT>(rest, c, red);
  if (threadIdx.x == 0)
    *rest_out = rest.m == INFINITY ? INFINITY : rest.s > 0.f ? (float)((double)rest.m / tau + log((double)rest.s)) : -INFINITY;
}

// 1024 rows of 131072 bf16, k 64: 91 us (268 MB; reading alone 45), whole rows by one workgroup of 256, four a CU.  A segment's load, the
// rounds that count for the bound, and the sum follow one another, and four workgroups overlap them only in part; a fifth does
// not fit beside 128 registers a thread (the next segment's loads straight into LDS, which would take none, were not tried).  16 rows
// of 50021 fp32, k 100, in 13 segments each: 8.8 us.
template <typename T, int NT, int VPT, bool MANY>
__global__ __launch_bounds__(NT, 4) void top_segment_kernel(const T* __restrict__ logits, int64_t ld, int V, int K, int cap, int count, float tau,
                                                         T* __restrict__ values, int32_t* __restrict__ ids, float* __restrict__ rest_out,
                                                         SegHead* __restrict__ heads, uint64_t* __restrict__ lists) {
  __shared__ SegLds<NT, MANY> l;
  const int64_t t = blockIdx.x;
  const int seg = blockIdx.y, nseg = gridDim.y;
  const float c = (float)(LOG2E / (double)tau);
  const T* row = logits + t * ld;
  uint64_t level;
  ExpSum rest;
  const int n = collect<T, NT, VPT, false, MANY>(row, V, seg * count, count, nseg * count, K, cap, c, l, level, rest);
  if (nseg == 1) {
    top_finish<T, NT>(l.list, n, K, tau, c, rest, l.red, values + t * K, ids + t * K, rest_out + t);
    return;
  }
  rest = block_exp_sum<NT>(rest, c, l.red);
  const int64_t at = t * nseg + seg;
  for (int i = threadIdx.x; i < n; i += NT) lists[at * cap + i] = l.list[i];
  if (threadIdx.x == 0) heads[at] = {level, rest.m, rest.s, (uint32_t)n, {0, 0, 0}};
}

// The segments' keys of one row, at most MERGE, R = MERGE / NT to a thread (0: none).
constexpr int MAX_SEGS = 64;
template <int NT> struct RowKeys {
  static constexpr int R = MERGE / NT;
  uint64_t k[R];
  uint64_t level;  // complete down to here
  ExpSum rest;     // this thread's share of the entries that no segment listed
  int n;
  __device__ __forceinline__ void load(const SegHead* heads, const uint64_t* lists, int64_t t, int nseg, int cap, uint32_t* ends) {
    rest = {-FLT_MAX, 0.f};
    const bool mine = (int)threadIdx.x < nseg;
    SegHead h = {};
    if (mine) {
      h = heads[t * nseg + threadIdx.x];
      rest = {h.m, h.s};
    }
    __syncthreads();
    if (threadIdx.x < 64) {  // (nseg <= 64: one wave)
      uint32_t end = mine ? h.n : 0;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const uint32_t up = __shfl_up(end, o, 64);
        if ((int)threadIdx.x >= o) end += up;
      }
      uint64_t lv = mine ? h.level : 0;
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) {
        const uint64_t v = __shfl_xor(lv, o, 64);
        lv = v > lv ? v : lv;
      }
      ends[threadIdx.x] = end;
      if (threadIdx.x == 0) {
        ends[64] = (uint32_t)lv;
        ends[65] = (uint32_t)(lv >> 32);
      }
    }
    __syncthreads();
    n = ends[nseg - 1];
    level = ((uint64_t)ends[65] << 32) | ends[64];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int i = r * NT + threadIdx.x;
      k[r] = 0;
      if (r * NT < n && i < n) {
        int s = 0;
        while ((int)ends[s] <= i) ++s;
        k[r] = lists[(t * nseg + s) * cap + i - (s ? (int)ends[s - 1] : 0)];
      }
    }
  }
  // The keys that can be among the first K, unsorted, into list; the sum over the others joins rest.  More than `room` of them
  // (ties at the bound): the exact K-th key as the bound.  The others come in no fixed order: their sum is one of whole multiples
  // of 2^-40 of the largest.
  template <typename L> __device__ __forceinline__ int first(int K, int room, uint64_t* list, float c, L& l) {
    uint64_t bound = 0;
    const int used = (n + NT - 1) / NT;
    if (n > 2 * K) {  // by the upper half of the values' bits, nearly always enough
      uint32_t hi[R];
#pragma unroll
      for (int r = 0; r < R; ++r) hi[r] = (uint32_t)(k[r] >> 32);
      bound = (uint64_t)kth_bound<NT>(hi, used, K, 30, 16, l.counts) << 32;
    }
    for (int round = 0;; ++round) {
      int m = 0;
      uint64_t most = 0;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (r >= used) break;
        m += k[r] != 0 && k[r] >= bound;
        if (k[r] < bound && k[r] > most) most = k[r];
      }
      m = block_all<NT>(m, reinterpret_cast<int*>(l.red), [](int a, int b) { return a + b; });
      if (m > room && round == 0) {
        bound = kth_bound<NT>(k, used, K, 62, 0, l.counts);
        continue;
      }
      if (bound) {
        most = block_all<NT>(most, l.wave, [](uint64_t a, uint64_t b) { return a > b ? a : b; });
        const float x0 = key_value((uint32_t)(most >> 32));
        uint64_t sum = 0;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          if (r >= used) break;
          if (k[r] != 0 && k[r] < bound) sum += fixed_weight(key_value((uint32_t)(k[r] >> 32)), x0, c);
        }
        sum = block_all<NT>(sum, l.wave, [](uint64_t a, uint64_t b) { return a + b; });
        if (threadIdx.x == 0 && most && x0 > -INFINITY) rest = exp_sum_join(rest, {x0, (float)sum * 0x1p-40f}, c);
      }
      __syncthreads();
      if (threadIdx.x == 0) l.n = 0;
      __syncthreads();
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (r >= used) break;
        if (k[r] != 0 && k[r] >= bound) list[atomicAdd(&l.n, 1u)] = k[r];
      }
      __syncthreads();
      level = bound > level ? bound : level;
      return m;
    }
  }
};

struct MergeLds {
  __align__(16) uint64_t list[2 * MAX_SEG_K];
  uint64_t wave[16], counts[2][16];
  float red[16];
  uint32_t n, ends[66];
};

// One workgroup a row, bound by latency: the lists' lengths, their keys, the bound and the sort wait for memory and LDS one after
// the other, and the bound's eight rounds read the keys from scratch memory (160 bytes a lane: loops over RowKeys::k end at a run-time
// count).  16 rows of 13 lists, k 100: 19 us; 1000 rows of 4 lists, k 512: 58 us.
template <typename T, int NT>
__global__ __launch_bounds__(NT) void top_merge_kernel(int nseg, int K, int cap, float tau, T* __restrict__ values,
                                                       int32_t* __restrict__ ids, float* __restrict__ rest_out,
                                                       const SegHead* __restrict__ heads, const uint64_t* __restrict__ lists) {
  __shared__ MergeLds l;
  const int64_t t = blockIdx.x;
  const float c = (float)(LOG2E / (double)tau);
  RowKeys<NT> rk;
  rk.load(heads, lists, t, nseg, cap, l.ends);
  const int n = rk.first(K, 2 * MAX_SEG_K, l.list, c, l);
  top_finish<T, NT>(l.list, n, K, tau, c, rk.rest, l.red, values + t * K, ids + t * K, rest_out + t);
}

// How a call is cut: threads and vectors per thread of a segment, workgroups per row, keys a workgroup may leave, K above 128,
// segments a workgroup takes one after the other.
struct Cut { int nt, vpt, nseg, cap; bool many; int count; };
Cut cut_rows(int dtype, int T, int V, int K) {
  const Cut none = {0, 0, 0, 0, false, 1};
  if (K > MAX_SEG_K || V <= 64) return none;
  const bool many = K > 128;
  const int vecs = V / (dtype == PG_F32 ? 4 : 8);
  // (64 threads leave 64 maxima: for K above that there is no bound, all entries are listed, and rows of more than `cap` of them go
  // by digits; 4096 x 1000 bf16: k 32 14 us, k 100 34)
  const int shapes[3][2] = {{64, 4}, {256, 4}, {256, 16}};
  for (int i = many ? 1 : 0; i < 3; ++i) {
    const int per = shapes[i][0] * shapes[i][1], nseg = vecs <= per ? 1 : (vecs + per - 1) / per;
    if (nseg > 1 && i < 2) {
      // few rows: small segments, to spread them over the chip; many: the next larger ones
      if (i == 0 || (int64_t)T * nseg > 1024) continue;
    }
    // rows enough for four workgroups a CU: one takes the whole row and joins nothing (1024 x 131072 bf16, k 64: 87 us,
    // against 105 with four workgroups a row and a launch that joins their lists).  Its
    // list grows by about 1.2 K / s in segment s
    if (nseg > 1 && i == 2 && T >= 1024 && 1.4 * K * (1.0 + log((double)nseg)) <= 400.0) return {256, 16, 1, max_cap(K), many, nseg};
    if (nseg > MAX_SEGS) continue;
    int cap = 2 * K + 64;
    if (cap > max_cap(K)) cap = max_cap(K);
    if (cap > MERGE / nseg) cap = MERGE / nseg;
    if (nseg == 1 || cap >= K + K / 2 + 32) return {shapes[i][0], shapes[i][1], nseg, cap, many, 1};
  }
  return none;
}
template <int N> struct Int { static constexpr int value = N; };
template <bool B> struct Bool { static constexpr bool value = B; };
template <typename F> void by_cut(const Cut& c, F f) {
  if (c.nt == 64) f(Int<64>(), Int<4>(), Bool<false>());
  else if (c.vpt == 4 && c.many) f(Int<256>(), Int<4>(), Bool<true>());
  else if (c.vpt == 4) f(Int<256>(), Int<4>(), Bool<false>());
  else if (c.many) f(Int<256>(), Int<16>(), Bool<true>());
  else f(Int<256>(), Int<16>(), Bool<false>());
}

// ------------------------------------------------------------------ sampling
struct RowFilter {
  float temperature, top_p, min_p;
  int top_k;
  // w >= min_p, as x >= max + temperature ln(min_p): no exponential's rounding decides it
  __device__ __forceinline__ bool above_min_p(float x, float m) const {
    if (!(min_p > 0.f) || x == m) return true;
    return min_p < 1.f && (double)x >= (double)m + (double)temperature * log((double)min_p);
  }
};
struct SampleArgs {
  float temperature, top_p, min_p;
  int top_k, empty;  // empty: the token of a row with nothing above -inf
  const float* temps; const int32_t* ks; const float* ps; const float* mins;
  // (positive temperatures within MIN_TAU .. MAX_TAU, where no scale or product of a scale leaves fp32's range; a row's negative
  // top_k is 0, off)
  __device__ __forceinline__ RowFilter row(int64_t t) const {
    const float given = temps ? temps[t] : temperature;
    return {given > 0.f ? fminf(fmaxf(given, MIN_TAU), MAX_TAU) : 0.f, ps ? ps[t] : top_p, mins ? mins[t] : min_p,
            ks ? max(ks[t], 0) : top_k};
  }
};
// ------------------------------------------------------------------ one row by a whole workgroup, any boundary
constexpr int BINS = 2048, POOL = 2048;
constexpr double MASS_ONE = 1099511627776.0;  // 2^40: weights are at most 1, their sums whole multiples of 2^-40 in any order
// Six digits of an entry's key from the top: 11 + 11 + 10 bits of the value, 11 + 11 + 10 of ~index.
__device__ __constant__ const int SEL_SHIFT[6] = {53, 42, 32, 21, 10, 0};
__device__ __constant__ const int SEL_BITS[6] = {11, 11, 10, 11, 11, 10};

struct PackedEntry { float x; int i; };
template <int NT> struct RowLds {
  __align__(16) uint64_t list[POOL];
  union {
    uint64_t mass[BINS];
    PackedEntry pack[NT / 64 * 512];
  };
  uint64_t wave[16], counts[2][16];
  uint64_t cut_before;
  double redd[16];
  float red[16];
  int cut;
  uint32_t n, ends[66];
};

// Bins of equal width in m - x, m the largest entry: an entry's bin never decreases with m - x, so bins are ranges of the order.
struct Bins {
  float m, per;
  __device__ __forceinline__ Bins(float largest, float per_unit) : m(fminf(largest, FLT_MAX)), per(per_unit) {}
  __device__ __forceinline__ int of(float x) const { return (int)fminf((m - fminf(x, FLT_MAX)) * per, (float)(BINS - 1)); }
};
// Where a filter's kept entries end: at a key of bin `bin` whose digits under `mask` are `prefix`; n such entries are in the list,
// sorted, of which the first `kept` are kept, down to key B.
struct Border {
  int bin, n, kept;
  float lo, hi;  // the bin's values
  uint64_t prefix, mask, B;
};
// The smallest value whose bin is at most b (b < 0: none, NaN), by bisection over the values' keys.
__device__ __forceinline__ float lowest_of(const Bins& bins, int b) {
  uint32_t lo = 0x007fffffu, hi = 0xff800000u;  // -inf .. +inf
  if (b < 0) return NAN;
  while (lo < hi) {
    const uint32_t mid = lo + (hi - lo) / 2;
    if (bins.of(key_value(mid)) <= b) hi = mid;
    else lo = mid + 1;
  }
  return key_value(lo);
}

__device__ __forceinline__ uint64_t fixed(double w) {  // w <= 1 in multiples of 2^-40
  return (uint64_t)(__double_as_longlong(w + 4096.0) - 0x40b0000000000000ll);  // (in 4096..8192 one unit in the last place is 2^-40)
}

// The border after which `need_count` entries (by_mass: the share `part` of the mass) of those with key >= floor lie.  2048 bins are
// counted (weighed) first; the border's bin is listed by gather(at) and sorted.  One that does not fit the list (many equal values,
// entries far below the largest) is divided by the key's bits first.
template <typename T, int NT, typename W, typename G>
__device__ __forceinline__ Border border(const T* row, int V, Bins bins, uint64_t floor, bool by_mass, int need_count, double part, W weight,
                                         RowLds<NT>& l, G gather) {
  uint32_t* count = reinterpret_cast<uint32_t*>(l.mass);
  const float floor_x = floor ? key_value((uint32_t)(floor >> 32)) : -INFINITY;
  auto below = [&](float x, int i) { return x <= floor_x && (x < floor_x || entry_key(x, i) < floor); };
  uint64_t need = need_count;
  Border at = {0, 0, 0, INFINITY, -INFINITY, 0, 0, 0};
#pragma unroll 1
  for (int d = -1;; ++d) {
    if (need_count >= 0) {
      const int shift = d < 0 ? 0 : SEL_SHIFT[d], n_bins = d < 0 ? BINS : 1 << SEL_BITS[d];
      __syncthreads();
      for (int i = threadIdx.x; i < n_bins; i += NT) l.mass[i] = 0;
      __syncthreads();
      auto put = [&](int b, float x) {
        if (by_mass) atomicAdd((unsigned long long*)&l.mass[b], (unsigned long long)fixed(weight(x)));
        else atomicAdd(&count[b], 1u);
      };
      if (d < 0)
        each<T, NT>(row, V, [&](int i, float x) {
          x = no_nan(x);
          if (!below(x, i)) put(bins.of(x), x);
        });
      else
        for (int i = threadIdx.x; i < V; i += NT) {
          const float x = no_nan(to_f32<T>(row[i]));
          const uint64_t k = entry_key(x, i);
          if (k >= floor && bins.of(x) == at.bin && (k & at.mask) == at.prefix) put(n_bins - 1 - ((int)(k >> shift) & (n_bins - 1)), x);
        }
      __syncthreads();
      auto get = [&](int i) { return by_mass ? l.mass[i] : (uint64_t)count[i]; };
      if (by_mass && d < 0) {
        const double all = (double)find_cut<NT>(n_bins, ~0ull, l, get).before;
        need = (uint64_t)fmin(fmax(ceil(part * all), 1.0), all);
      }
      const CutAt c = find_cut<NT>(n_bins, need, l, get);
      const int b = min(c.i, n_bins - 1);  // (fewer than asked for: down to the last)
      need = c.i < n_bins ? need - c.before : ~0ull;
      if (d < 0) {
        at.bin = b;
        at.lo = lowest_of(bins, b);
        const float next = lowest_of(bins, b - 1);
        at.hi = b > 0 ? key_value(value_key(next) - 1) : INFINITY;
      } else {
        at.prefix |= (uint64_t)(n_bins - 1 - b) << shift;
        at.mask |= (uint64_t)(n_bins - 1) << shift;
      }
    } else {
      at.bin = BINS;  // (no border to look for: every entry above -inf is before it, lo > hi)
    }
    __syncthreads();
    if (threadIdx.x == 0) l.n = 0;
    __syncthreads();
    gather(at);
    __syncthreads();
    if (l.n <= POOL || d == 5) break;
  }
  at.n = l.n;
  if (at.n == 0) return at;
  sort_keys<NT>(l.list, at.n);
  const CutAt c = find_cut<NT>(at.n, need, l, [&](int i) { return by_mass ? fixed(weight(key_value((uint32_t)(l.list[i] >> 32)))) : (uint64_t)1; });
  at.kept = min(c.i + 1, at.n);
  at.B = l.list[at.kept - 1];
  return at;
}

// exp((x - m) / temperature) in 64 bits (scale = log2(e) / temperature); the largest entry has 1, an infinite one too.
struct Weight {
  float m;
  double scale;
  __device__ __forceinline__ double operator()(float x) const { return x == m ? 1.0 : exp2_f64(((double)x - (double)m) * scale); }
};

// The entries of the border's bin into the list.
template <typename T, int NT>
__device__ __forceinline__ void gather_bin(const T* row, int V, uint64_t floor, const Border& at, RowLds<NT>& l) {
  each<T, NT>(row, V, [&](int i, float x) {
    x = no_nan(x);
    if (x < at.lo || x > at.hi) return;
    const uint64_t k = entry_key(x, i);
    if (k < floor || (k & at.mask) != at.prefix) return;
    const uint32_t p = atomicAdd(&l.n, 1u);
    if (p < POOL) l.list[p] = k;
  });
}

// A thread's share of the race: the best w / noise, in 64 bits where an fp32 quotient (off by less than 2^-20) says it can win.
struct Race {
  double best = -1.0, total = 0.0;
  float screen = -1.f, x = 0.f;
  uint64_t at = ~0ull;
  __device__ __forceinline__ void add(double w, float value, float q, uint32_t i) {
    total += w;
    const float r = (float)w * __builtin_amdgcn_rcpf(q);
    if (r < screen) return;
    const double e = w > 0.0 ? w / (double)q : 0.0;
    if (e > best || (e == best && i < at)) {
      best = e;
      at = i;
      x = value;
      screen = (float)e < FLT_MAX ? (float)e * (1.f - 0x1p-16f) : FLT_MAX;
    }
  }
};

struct ListLds {
  __align__(16) uint64_t list[POOL];
  uint64_t mass[POOL];
  uint64_t wave[16], counts[2][16];
  double redd[16];
  float red[16];
  int cut;
  uint32_t n, ends[66];
};

// Ends a row's race over the whole workgroup or its first wave: token and probability.
template <int NT, typename L, typename W>
__device__ __forceinline__ void finish(const Race& race, double kept_mass, uint32_t arg, W weight, L& l, int64_t* pred,
                                       float* conf) {
  const double best = block_all<NT>(race.best, l.redd, [](double a, double b) { return fmax(a, b); });
  const uint64_t mine = race.best == best ? race.at : (uint64_t)~0ull;
  const uint64_t at = block_all<NT>(mine, l.wave, [](uint64_t a, uint64_t b) { return a < b ? a : b; });
  if (at == ~0ull) {  // (noise without a usable draw)
    if (threadIdx.x == 0) *pred = arg, *conf = (float)(1.0 / kept_mass);
  } else if (mine == at) {
    *pred = (int64_t)at;
    *conf = (float)(weight(race.x) / kept_mass);
  }
}

// From the segments' lists, if the end of the kept entries lies within them.  A row where it does not is left to
// sample_row_kernel: pred = -2 - (index of its largest entry), conf = that entry.  Bound as the merge, its keys in scratch memory too
// (1024 rows write 39 MiB of it): 13 us a row, 19 us for 256 rows of 4 lists.
template <typename T, int NT>
__global__ __launch_bounds__(NT) void sample_list_kernel(const float* __restrict__ noise, int64_t ld_noise, int V, SampleArgs args,
                                                         int nseg, int cap, const SegHead* __restrict__ heads,
                                                         const uint64_t* __restrict__ lists, int64_t* __restrict__ pred,
                                                         float* __restrict__ conf, uint64_t* __restrict__ split, int64_t split_words) {
  __shared__ ListLds l;
  const int64_t t = blockIdx.x;
  const float* q = noise + t * ld_noise;
  const RowFilter f = args.row(t);
  const bool greedy = !(f.temperature > 0.f);
  const double scale = LOG2E / (double)f.temperature;
  const float c = greedy ? 0.f : (float)scale;
  RowKeys<NT> rk;
  rk.load(heads, lists, t, nseg, cap, l.ends);
  const int want = f.top_k > 0 && f.top_k <= MAX_SEG_K ? f.top_k : 192;  // (what 256 threads sort by counting)
  const int n = rk.first(want, POOL, l.list, c, l);
  if (n == 0) {
    if (threadIdx.x == 0) pred[t] = args.empty, conf[t] = 0.f;
    return;
  }
  sort_keys<NT>(l.list, n);
  const float m = key_value((uint32_t)(l.list[0] >> 32));
  const uint32_t arg = ~(uint32_t)l.list[0];
  if (greedy) {
    if (threadIdx.x == 0) pred[t] = arg, conf[t] = 1.f;
    return;
  }
  const Weight weight = {m, scale};
  // l.mass[i]: the weights of the entries 0..i; nv, na: entries down to which the list is complete / that min_p leaves
  const int per = (n + NT - 1) / NT, a0 = min((int)threadIdx.x * per, n), a1 = min(a0 + per, n);
  uint64_t sum = 0;
  int both = 0;
  for (int i = a0; i < a1; ++i) {
    const uint64_t k = l.list[i];
    const float x = key_value((uint32_t)(k >> 32));
    sum += fixed(weight(x));
    l.mass[i] = sum;
    both += (k >= rk.level) + (f.above_min_p(x, m) << 16);
  }
  uint64_t upto = sum;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint64_t v = __shfl_up(upto, o, 64);
    if ((int)(threadIdx.x & 63) >= o) upto += v;
  }
  float out_m = rk.rest.m, out_s = rk.rest.s;  // (the segments' sums: in the first wave's lanes)
  if (threadIdx.x < 64) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const ExpSum j = exp_sum_join({out_m, out_s}, {__shfl_xor(out_m, o, 64), __shfl_xor(out_s, o, 64)}, c);
      out_m = j.m; out_s = j.s;
    }
    if (threadIdx.x == 0) l.red[0] = out_m, l.red[1] = out_s;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) both += __shfl_xor(both, o, 64);
  if ((threadIdx.x & 63) == 63) l.wave[threadIdx.x >> 6] = upto, l.counts[0][threadIdx.x >> 6] = (uint64_t)(uint32_t)both;
  if (threadIdx.x == 0) l.cut = n;
  __syncthreads();
  uint64_t off = upto - sum;
  int nv = 0, na = 0;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) {
    if (w < (int)(threadIdx.x >> 6)) off += l.wave[w];
    nv += (int)l.counts[0][w] & 0xffff;
    na += (int)l.counts[0][w] >> 16;
  }
  for (int i = a0; i < a1; ++i) l.mass[i] += off;
  const double left = (double)l.red[1] * (double)__builtin_amdgcn_exp2f((l.red[0] - m) * c);  // the mass outside the list
  __syncthreads();
  const bool whole = rk.level == 0;  // (every entry above -inf is in the list)
  const int nk = f.top_k > 0 && f.top_k < V ? f.top_k : V;
  const bool nk_in = nk <= nv || whole;
  int keep = nk_in ? min(nk, nv) : V;
  bool sure = true;
  if (f.top_p < 1.f) {
    if (nk_in || nk == V) {
      // the mass outside: fp32 sums of up to 2^7 terms per thread and a tree, their relative error below 2^-15, of masses that are
      // not rounded to multiples of 2^-40 (each off by less than half a multiple, and by less than itself)
      const double rest = nk_in ? 0.0 : left * MASS_ONE, err = rest * 0x1p-15 + fmin(rest, 0.5 * (V - n));
      const double share = (double)f.top_p * ((double)l.mass[(nk_in ? keep : n) - 1] + rest), need = fmax(1.0, ceil(share));
      for (int i = a0; i < a1; ++i)
        if ((i == 0 || (double)l.mass[i - 1] < need) && (double)l.mass[i] >= need) l.cut = i;
      __syncthreads();
      const int at = l.cut;  // (n: beyond the list)
      const double before = at > 0 ? (double)l.mass[min(at, nv) - 1] : 0.0;
      if (at < nv) {
        if (err > 0.0) sure = before < fmax(1.0, share - err) && (double)l.mass[at] >= fmax(1.0, share + err);
        keep = min(keep, at + 1);
      } else if (!nk_in) {
        sure = before < fmax(1.0, share - err);
      }
    } else {
      sure = false;  // (the mass of the first k is not known)
    }
    if (m == INFINITY && !nk_in) sure = false;  // (infinite entries outside the list have no mass in it)
  }
  if (f.min_p > 0.f && (na < nv || whole)) keep = min(keep, na);
  if (!sure || keep > nv) {
    if (threadIdx.x == 0) pred[t] = -2 - (int64_t)arg, conf[t] = m;
    if (split)
      for (int i = threadIdx.x; i < split_words; i += NT) split[t * split_words + i] = 0;
    return;
  }
  const double kept_mass = (double)l.mass[keep - 1] * 0x1p-40;
  Race race;
  for (int i = threadIdx.x; i < keep; i += NT) {
    const uint32_t at = ~(uint32_t)l.list[i];
    const float x = key_value((uint32_t)(l.list[i] >> 32));
    race.add(weight(x), x, q[at], at);
  }
  if (keep <= 64) {  // the first wave's alone
    if (threadIdx.x < 64) finish<64>(race, kept_mass, arg, weight, l, pred + t, conf + t);
  } else {
    finish<NT>(race, kept_mass, arg, weight, l, pred + t, conf + t);
  }
}

// min_p as the smallest value it leaves; -inf and NaN never race
__device__ __forceinline__ float least_value(const RowFilter& f, float m) {
  if (!(f.min_p > 0.f)) return -FLT_MAX;
  const double x = (double)m + (double)f.temperature * log((double)fminf(f.min_p, 1.f));
  float least = fmaxf((float)x, -FLT_MAX);
  if ((double)least < x) least = key_value(value_key(least) + 1);
  return fminf(least, m);
}
__device__ __forceinline__ Bins row_bins(const RowFilter& f, float m) { return Bins(m, (float)BINS / fminf(40.f * f.temperature, 32.f)); }

// The n entries at p, the first of them entry i0 of its row: those before the border race, those at it go to push(key).  A wave
// first packs a vector's racing entries (each wave its own part of `packs`), so that a few among many do not take the 64-bit work
// of all; four vectors per thread are on their way meanwhile, and noise is read for the racing entries alone.
template <typename T, int NT, typename P>
__device__ __forceinline__ void sweep(const T* p, int n, int i0, const float* q, uint64_t floor, const Border& at, float least, const Weight& weight,
                                      Race& race, PackedEntry* packs, P push) {
  constexpr int E = 16 / (int)sizeof(T);
  PackedEntry* pack = packs + (threadIdx.x >> 6) * 512;
  int packed = 0;
  auto look = [&](float x, int i) {  // (by whole waves)
    bool go = x >= least;
    if (!(x > at.hi)) {
      const bool near = x >= at.lo;
      go = go && near;
      if (near) {
        const uint64_t k = entry_key(x, i), digits = k & at.mask;
        go = go && k >= floor && digits > at.prefix;
        if (k >= floor && digits == at.prefix) push(k);
      }
    }
    const uint64_t lanes = __ballot(go);
    if (go) pack[packed + __builtin_amdgcn_mbcnt_hi((uint32_t)(lanes >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)lanes, 0))] = {x, i};
    packed += __popcll(lanes);
  };
  auto run = [&]() {
    if (packed == 0) return;
    race.screen = wave_max(race.screen);  // (alone, some lane of a wave nearly always has a new best of its own to divide for)
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll 1
    for (int j = threadIdx.x & 63; j < packed; j += 256) {
      PackedEntry e[4];
      float z[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        e[u] = pack[min(j + 64 * u, packed - 1)];
        z[u] = q[e[u].i];
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (j + 64 * u < packed) race.add(weight(e[u].x), e[u].x, z[u], e[u].i);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    packed = 0;
  };
  int head = (int)((16 - ((uintptr_t)p & 15)) & 15) / (int)sizeof(T);
  if (head > n) head = n;
  const int nv = (n - head) / E, tail = head + nv * E;
  const uint4* vec = reinterpret_cast<const uint4*>(p + head);
  uint4 d[4] = {};
  if (nv)
#pragma unroll
    for (int u = 0; u < 4; ++u) d[u] = vec[min((int)threadIdx.x + u * NT, nv - 1)];
#pragma unroll 1
  for (int r0 = 0; r0 < nv; r0 += NT) {
    const int v = r0 + threadIdx.x;
    float o[E];
    unpack(d[0], o);
    d[0] = d[1]; d[1] = d[2]; d[2] = d[3];
    d[3] = vec[min(v + 4 * NT, nv - 1)];
#pragma unroll
    for (int e = 0; e < E; ++e) look(v < nv ? o[e] : NAN, i0 + head + v * E + e);
    run();
  }
  const int end = (int)threadIdx.x < head ? (int)threadIdx.x : tail + (int)threadIdx.x - head;  // (both ends: less than 2 E entries)
  look(end < n && (int)threadIdx.x < head + n - tail ? to_f32<T>(p[end]) : NAN, i0 + end);
  run();
}

// From the whole row: every row (all), or those sample_list_kernel left.  The border of top-k, then of top-p among those, then
// the race.  One workgroup a row, bound by the 64-bit exponentials of its CU, one for every entry: 1024 rows of 32768 bf16 (normal
// logits) without a filter 135 us, at top_p 0.95, which the lists do not hold, 220 us.
template <typename T, int NT>
__global__ __launch_bounds__(NT, 2) void sample_row_kernel(const T* __restrict__ logits, int64_t ld, const float* __restrict__ noise,
                                                        int64_t ld_noise, int V, SampleArgs args, bool all, int64_t* __restrict__ pred,
                                                        float* __restrict__ conf) {
  __shared__ RowLds<NT> l;
  const int64_t t = blockIdx.x;
  const T* row = logits + t * ld;
  const float* q = noise + t * ld_noise;
  const RowFilter f = args.row(t);
  float m;
  uint32_t arg;
  if (all) {
    float most = -INFINITY;
    int first = -1;
    each<T, NT>(row, V, [&](int i, float x) {
      if (x > most || (x == most && (uint32_t)i < (uint32_t)first)) most = x, first = i;  // (the row's odd ends come last)
    });
    uint64_t top = first < 0 ? entry_key(-INFINITY, ~0u) : entry_key(most, first);
    top = block_all<NT>(top, l.wave, [](uint64_t a, uint64_t b) { return a > b ? a : b; });
    m = key_value((uint32_t)(top >> 32));
    arg = ~(uint32_t)top;
    if (m == -INFINITY || !(f.temperature > 0.f)) {
      if (threadIdx.x == 0) pred[t] = m == -INFINITY ? (int64_t)args.empty : (int64_t)arg, conf[t] = m == -INFINITY ? 0.f : 1.f;
      return;
    }
  } else {
    const int64_t left = pred[t];
    if (left > -2) return;
    arg = (uint32_t)(-2 - left);
    m = conf[t];
    __syncthreads();
  }
  const Weight weight = {m, LOG2E / (double)f.temperature};
  const Bins bins = row_bins(f, m);
  const bool by_k = f.top_k > 0 && f.top_k < V, by_p = f.top_p < 1.f;
  const float least = least_value(f, m);
  Race race;
  Border at = {BINS, 0, 0, INFINITY, -INFINITY, 0, 0, 0};
#pragma unroll 1
  for (int last = by_k && by_p ? 0 : 1; last < 2; ++last) {  // one copy of the code for both filters
    const uint64_t floor = at.B;
    auto gather = [&](const Border& a) {
      if (last) {
        race = Race();
        sweep<T, NT>(row, V, 0, q, floor, a, least, weight, race, l.pack, [&](uint64_t k) {
          const uint32_t p = atomicAdd(&l.n, 1u);
          if (p < POOL) l.list[p] = k;
        });
      } else {
        gather_bin<T, NT>(row, V, floor, a, l);
      }
    };
    at = border<T, NT>(row, V, bins, floor, last && by_p, by_k || by_p ? f.top_k : -1, (double)f.top_p, weight, l, gather);
  }
  for (int i = threadIdx.x; i < at.kept; i += NT) {
    const float x = key_value((uint32_t)(l.list[i] >> 32));
    const uint32_t j = ~(uint32_t)l.list[i];
    if (x >= least) race.add(weight(x), x, q[j], j);
  }
  const double kept_mass = block_sum<NT>(race.total, l.redd);
  finish<NT>(race, kept_mass, arg, weight, l, pred + t, conf + t);
}

// The rows sample_list_kernel left, where there are few rows: each cut into parts for several CUs, in three launches (bins of the
// parts added up; the race of the parts, the border's entries listed; the border and the race joined).  For rows with one border or
// none; a row with both filters open, or with more entries in the border's bin than the list holds, stays for sample_row_kernel.
// The parts are counted from all rows of the call: where the lists leave only a few, most workgroups return at once and as few CUs
// work.  256 rows of 32768 bf16, normal logits, top_p 0.95 (all left): bins 15 us, race 49, join 10; one row: 5, 19, 8; 256 of 131072
// of which the lists leave about one in twenty: 40, 45, 24.
struct SplitPart { double best, total; uint64_t at; float x; int pad; };
struct SplitRow {  // one per row, in the workspace
  uint64_t mass[BINS], list[POOL];
  uint64_t need;   // of the border's bin
  uint32_t n, pad;
  SplitPart part[16];
};
__device__ __forceinline__ bool split_row(const SampleArgs& args, int64_t t, int V, const int64_t* pred, RowFilter& f, bool& by_k, bool& by_p) {
  if (pred[t] > -2) return false;
  f = args.row(t);
  by_k = f.top_k > 0 && f.top_k < V;
  by_p = f.top_p < 1.f;
  return !(by_k && by_p);
}
struct PartOf { int i0, n; };
__device__ __forceinline__ PartOf part_of(int V, int part, int parts) {
  const int per = (V + parts - 1) / parts, i0 = min(part * per, V);
  return {i0, min(per, V - i0)};
}

template <typename T, int NT>
__global__ __launch_bounds__(NT) void sample_bins_kernel(const T* __restrict__ logits, int64_t ld, int V, SampleArgs args,
                                                         const int64_t* __restrict__ pred, const float* __restrict__ conf,
                                                         SplitRow* __restrict__ split) {
  __shared__ uint64_t mass[BINS];
  const int64_t t = blockIdx.x;
  RowFilter f;
  bool by_k, by_p;
  if (!split_row(args, t, V, pred, f, by_k, by_p) || !(by_k || by_p)) return;
  const float m = conf[t];
  const Weight weight = {m, LOG2E / (double)f.temperature};
  const Bins bins = row_bins(f, m);
  const PartOf at = part_of(V, blockIdx.y, gridDim.y);
  for (int i = threadIdx.x; i < BINS; i += NT) mass[i] = 0;
  __syncthreads();
  each<T, NT>(logits + t * ld + at.i0, at.n, [&](int, float x) {
    x = no_nan(x);
    atomicAdd((unsigned long long*)&mass[bins.of(x)], by_p ? (unsigned long long)fixed(weight(x)) : 1ull);
  });
  __syncthreads();
  for (int i = threadIdx.x; i < BINS; i += NT)
    if (mass[i]) atomicAdd((unsigned long long*)&split[t].mass[i], (unsigned long long)mass[i]);
}

template <typename T, int NT>
__global__ __launch_bounds__(NT, 2) void sample_part_kernel(const T* __restrict__ logits, int64_t ld, const float* __restrict__ noise,
                                                         int64_t ld_noise, int V, SampleArgs args, const int64_t* __restrict__ pred,
                                                         const float* __restrict__ conf, SplitRow* __restrict__ split) {
  __shared__ RowLds<NT> l;
  const int64_t t = blockIdx.x;
  RowFilter f;
  bool by_k, by_p;
  if (!split_row(args, t, V, pred, f, by_k, by_p)) return;
  const float m = conf[t];
  const Weight weight = {m, LOG2E / (double)f.temperature};
  const Bins bins = row_bins(f, m);
  SplitRow& w = split[t];
  Border at = {BINS, 0, 0, INFINITY, -INFINITY, 0, 0, 0};
  if (by_k || by_p) {
    for (int i = threadIdx.x; i < BINS; i += NT) l.mass[i] = w.mass[i];
    __syncthreads();
    auto get = [&](int i) { return l.mass[i]; };
    uint64_t need = f.top_k;
    if (by_p) {
      const double all = (double)find_cut<NT>(BINS, ~0ull, l, get).before;
      need = (uint64_t)fmin(fmax(ceil((double)f.top_p * all), 1.0), all);
    }
    const CutAt c = find_cut<NT>(BINS, need, l, get);
    at.bin = min(c.i, BINS - 1);
    at.lo = lowest_of(bins, at.bin);
    const float next = lowest_of(bins, at.bin - 1);
    at.hi = at.bin > 0 ? key_value(value_key(next) - 1) : INFINITY;
    if (blockIdx.y == 0 && threadIdx.x == 0) w.need = c.i < BINS ? need - c.before : ~0ull;
    __syncthreads();
  }
  const PartOf part = part_of(V, blockIdx.y, gridDim.y);
  Race race;
  sweep<T, NT>(logits + t * ld + part.i0, part.n, part.i0, noise + t * ld_noise, 0, at, least_value(f, m), weight, race, l.pack, [&](uint64_t k) {
    const uint32_t p = atomicAdd(&w.n, 1u);
    if (p < POOL) w.list[p] = k;
  });
  const double total = block_sum<NT>(race.total, l.redd);
  const double best = block_all<NT>(race.best, l.redd, [](double a, double b) { return fmax(a, b); });
  const uint64_t mine = race.best == best ? race.at : (uint64_t)~0ull;
  const uint64_t first = block_all<NT>(mine, l.wave, [](uint64_t a, uint64_t b) { return a < b ? a : b; });
  if (first == ~0ull ? threadIdx.x == 0 : mine == first) w.part[blockIdx.y] = {best, total, first, race.x, 0};
}

template <int NT>
__global__ __launch_bounds__(NT) void sample_join_kernel(const float* __restrict__ noise, int64_t ld_noise, int V, SampleArgs args, int parts,
                                                         int64_t* __restrict__ pred, float* __restrict__ conf,
                                                         const SplitRow* __restrict__ split) {
  __shared__ RowLds<NT> l;
  const int64_t t = blockIdx.x;
  RowFilter f;
  bool by_k, by_p;
  if (!split_row(args, t, V, pred, f, by_k, by_p)) return;
  const SplitRow& w = split[t];
  const int n = (int)w.n;
  if (n > POOL) return;
  const uint32_t arg = (uint32_t)(-2 - pred[t]);
  const float m = conf[t], least = least_value(f, m);
  const Weight weight = {m, LOG2E / (double)f.temperature};
  int kept = 0;
  if (n) {
    for (int i = threadIdx.x; i < n; i += NT) l.list[i] = w.list[i];
    __syncthreads();
    sort_keys<NT>(l.list, n);
    const CutAt c = find_cut<NT>(n, w.need, l, [&](int i) { return by_p ? fixed(weight(key_value((uint32_t)(l.list[i] >> 32)))) : (uint64_t)1; });
    kept = min(c.i + 1, n);
  }
  Race race;
  for (int i = threadIdx.x; i < kept; i += NT) {
    const float x = key_value((uint32_t)(l.list[i] >> 32));
    const uint32_t j = ~(uint32_t)l.list[i];
    if (x >= least) race.add(weight(x), x, noise[t * ld_noise + j], j);
  }
  double kept_mass = block_sum<NT>(race.total, l.redd);
  for (int p = 0; p < parts; ++p) kept_mass += w.part[p].total;
  if ((int)threadIdx.x < parts) {
    const SplitPart s = w.part[threadIdx.x];
    if (s.at != ~0ull && (s.best > race.best || (s.best == race.best && s.at < race.at))) {
      race.best = s.best;
      race.at = s.at;
      race.x = s.x;
    }
  }
  __syncthreads();  // (pred and conf are read by all before one writes)
  finish<NT>(race, kept_mass, arg, weight, l, pred + t, conf + t);
}

// 256 rows of 131072 bf16: 28 us (67 MB, 2.4 TB/s; phases as in top_segment_kernel); one row of 65537: 10 us.
template <typename T, int NT, int VPT, bool MANY>
__global__ __launch_bounds__(NT, 4) void sample_segment_kernel(const T* __restrict__ logits, int64_t ld, int V, SampleArgs args, int K,
                                                               int cap, int count, SegHead* __restrict__ heads, uint64_t* __restrict__ lists) {
  __shared__ SegLds<NT, MANY> l;
  const int64_t t = blockIdx.x;
  const int seg = blockIdx.y, nseg = gridDim.y;
  const float temp = args.row(t).temperature;
  const float c = temp > 0.f ? (float)(LOG2E / (double)temp) : 0.f;
  const T* row = logits + t * ld;
  uint64_t level;
  ExpSum rest;
  const int n = collect<T, NT, VPT, true, MANY>(row, V, seg * count, count, nseg * count, K, cap, c, l, level, rest);
  rest = block_exp_sum<NT>(rest, c, l.red);
  const int64_t at = t * nseg + seg;
  for (int i = threadIdx.x; i < n; i += NT) lists[at * cap + i] = l.list[i];
  if (threadIdx.x == 0) heads[at] = {level, rest.m, rest.s, (uint32_t)n, {0, 0, 0}};
}

// ------------------------------------------------------------------ top entries, any k and vocabulary
// For k above MAX_SEG_K, and where lists of k do not fit one merge: the row three to four times through the caches.  1024 rows of
// 131072 bf16, k 1024: 276 us for normal logits, 342 with a few entries far above the rest.
template <typename T, int NT>
__global__ __launch_bounds__(NT) void top_kernel(const T* __restrict__ logits, int64_t ld, int V, int K, float tau,
                                                 T* __restrict__ values, int32_t* __restrict__ ids, float* __restrict__ rest) {
  __shared__ RowLds<NT> l;
  const int64_t t = blockIdx.x;
  const T* row = logits + t * ld;
  const float c = (float)(LOG2E / (double)tau);
  float m = -INFINITY;
  each<T, NT>(row, V, [&](int, float x) { m = x > m ? x : m; });
  m = block_max<NT>(m, l.red);
  const Bins bins(m, BINS / 32.f);
  const uint64_t B = border<T, NT>(row, V, bins, 0, false, K, 0.0, [](float) { return 0.0; }, l,
                                              [&](const Border& at) { gather_bin<T, NT>(row, V, 0, at, l); }).B;
  __syncthreads();
  if (threadIdx.x == 0) l.n = 0;
  __syncthreads();
  ExpSum out = {-FLT_MAX, 0.f};
  each<T, NT>(row, V, [&](int i, float x) {
    const uint64_t k = entry_key(x, i);
    if (k >= B) l.list[atomicAdd(&l.n, 1u)] = k;
    else exp_sum_one(out, x, c);
  });
  __syncthreads();
  top_finish<T, NT>(l.list, K, K, tau, c, out, l.red, values + t * K, ids + t * K, rest + t);
}

// ------------------------------------------------------------------ distillation
// Per row kept between forward and backward, all fp32: with c = log2(e)/tau,
//   student probability of entry v:  exp2((x_v - [0]) c) [1]
//   gradient (before tau, weight and upstream) of an entry outside the teacher's list:  [3] exp2((x_v - [2]) c)
//   teacher probability of entry e:  exp2((v_e - [4]) c) [5]
//   [6]: 1 if the row counts, [7]: 1 if an id may occur twice
constexpr int STASH = 8;

struct DistillArgs {
  const void* values; const int32_t* ids; const float* rest; const float* weights;
  int K; float tau;
};

template <typename T> __device__ __forceinline__ bool valid_entry(const T* values, const int32_t* ids, int e, int V) {
  return (uint32_t)ids[e] < (uint32_t)V && to_f32<T>(values[e]) > -INFINITY;
}

// Is entry e the first of its id in the list?
template <typename T> __device__ __forceinline__ bool first_of_id(const T* values, const int32_t* ids, int e, int V) {
  for (int j = 0; j < e; ++j)
    if (ids[j] == ids[e] && valid_entry(values, ids, j, V)) return false;
  return true;
}

// Segment `seg` of `nseg` of a row: its whole 16-byte vectors [v0, v1); the elements before the first vector of the row belong to
// the first segment, those behind the last one to the last.
template <typename T> struct Span {
  static constexpr int E = 16 / (int)sizeof(T);
  int head, tail, v0, v1;  // head: elements before the row's first vector; tail: first element behind its last
  bool first, last;
  __device__ __forceinline__ Span(const T* row, int V, int seg, int nseg) {
    head = (int)((16 - ((uintptr_t)row & 15)) & 15) / (int)sizeof(T);
    if (head > V) head = V;
    const int nv = (V - head) / E, per = (nv + nseg - 1) / nseg;
    tail = head + nv * E;
    v0 = min(seg * per, nv);
    v1 = min(v0 + per, nv);
    first = seg == 0;
    last = seg == nseg - 1;
  }
  __device__ __forceinline__ bool owns(int i) const {
    return i < head ? first : i >= tail ? last : i >= head + v0 * E && i < head + v1 * E;
  }
  // vec(o, v) over the vectors, one(i) over the odd elements.  A wave takes 4 KB at a time, four vectors a lane from one address;
  // the next four are on their way while these are worked on (begin() sends the first off).
  static constexpr int U = 4;
  __device__ __forceinline__ int vector(int tile, int u) const { return v0 + tile * U + (int)(threadIdx.x & ~63u) * U + u * 64 + (int)(threadIdx.x & 63); }
  template <bool ONCE> static __device__ __forceinline__ uint4 get(const uint4* p) { return ONCE ? load_once(p) : *p; }
  template <int NT, bool ONCE> __device__ __forceinline__ void begin(const T* row, uint4 (&d)[U]) const {
    const uint4* p = reinterpret_cast<const uint4*>(row + head);
    if ((v1 - v0) >= NT * U)
#pragma unroll
      for (int u = 0; u < U; ++u) d[u] = get<ONCE>(p + vector(0, u));
  }
  template <int NT, bool ONCE, typename F, typename G> __device__ __forceinline__ void each(const T* row, int V, uint4 (&d)[U], F vec, G one) const {
    const uint4* p = reinterpret_cast<const uint4*>(row + head);
    const int tiles = (v1 - v0) / (NT * U);
    uint4 n[U];
    auto work = [&](const uint4 (&x)[U], int tile) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float o[E];
        unpack(x[u], o);
        vec(o, vector(tile, u));
      }
    };
#pragma unroll 1
    for (int i = 0; i < tiles; i += 2) {
      if (i + 1 < tiles)
#pragma unroll
        for (int u = 0; u < U; ++u) n[u] = get<ONCE>(p + vector((i + 1) * NT, u));
      work(d, i * NT);
      if (i + 2 < tiles)
#pragma unroll
        for (int u = 0; u < U; ++u) d[u] = get<ONCE>(p + vector((i + 2) * NT, u));
      if (i + 1 < tiles) work(n, (i + 1) * NT);
    }
#pragma unroll 1
    for (int v = v0 + tiles * NT * U + threadIdx.x; v < v1; v += NT) {
      float o[E];
      unpack(get<ONCE>(p + v), o);
      vec(o, v);
    }
    if (first && (int)threadIdx.x < head) one((int)threadIdx.x);
    if (last && tail + (int)threadIdx.x < V) one(tail + (int)threadIdx.x);
  }
};

// Which tokens are in the teacher's list: one bit per element of a segment in LDS, a vector's bits together (a byte for bf16, half
// of one for fp32), so that the pass over the row looks at one byte per vector.  MAX_MEMBER bits; longer rows are cut.
constexpr int MAX_MEMBER = 1 << 17;

template <typename T, int NT>
__device__ __forceinline__ ExpSum distill_sum(const T* row, int V, const Span<T>& sp, const T* values, const int32_t* ids, int K, bool tail,
                                              float c, uint32_t* member, int* repeated) {
  constexpr int E = Span<T>::E;
  uint4 d[Span<T>::U];
  sp.template begin<NT, false>(row, d);
  const int start = sp.head + sp.v0 * E - E;  // element of bit 0: a vector's worth before the segment, for the odd elements in front
  if (tail) {
    const int bits = (sp.v1 - sp.v0 + 2) * E;
    for (int i = threadIdx.x; i < (bits + 31) / 32; i += NT) member[i] = 0;
    if (threadIdx.x == 0) *repeated = 0;
    __syncthreads();
    for (int e = threadIdx.x; e < K; e += NT)
      if (valid_entry(values, ids, e, V) && sp.owns(ids[e])) {
        const int b = ids[e] - start;
        if (atomicOr(&member[b >> 5], 1u << (b & 31)) >> (b & 31) & 1) *repeated = 1;
      }
    __syncthreads();
  }
  const uint8_t* bytes = reinterpret_cast<const uint8_t*>(member);
  auto outside = [&](const float (&x)[E], int v, float (&y)[E]) {  // the vector without the list's tokens
    const int at = v - sp.v0 + 1;
    const uint32_t in = tail ? (E == 8 ? bytes[at] : bytes[at >> 1] >> (at & 1) * 4 & 15) : 0;
#pragma unroll
    for (int e = 0; e < E; ++e) y[e] = x[e];
    if (in)
#pragma unroll
      for (int e = 0; e < E; ++e) y[e] = in >> e & 1 ? -INFINITY : x[e];
  };
  // the reference of the thread's sum: its first vector's largest entry outside the list
  float m = INFINITY;
  if (sp.v1 - sp.v0 >= NT * Span<T>::U) {
    float x[E], y[E];
    unpack(d[0], x);
    outside(x, sp.vector(0, 0), y);
    m = vec_max<E>(y);
  }
  FixedSum sum(m, c);
  ExpSum ends = {-FLT_MAX, 0.f};
  auto one = [&](int i) {
    const int b = i - start;
    if (!tail || !(member[b >> 5] >> (b & 31) & 1)) exp_sum_add(ends, to_f32<T>(row[i]), c);
  };
  sp.template each<NT, false>(row, V, d, [&](const float (&x)[E], int v) {
    float y[E];
    outside(x, v, y);
    sum.template add<E>(y);
  }, one);
  ExpSum o = sum.end();
  if (!sum.ok()) {  // short segments, entries far apart, NaN
    o = {-FLT_MAX, 0.f};
    sp.template begin<NT, false>(row, d);
    sp.template each<NT, false>(row, V, d, [&](const float (&x)[E], int v) {
      float y[E];
      outside(x, v, y);
      exp_sum_vec<E, true>(o, y, vec_max<E>(y), c);
    }, [](int) {});
  }
  return ends.s == 0.f ? o : exp_sum_join(o, ends, c);
}

// One entry of the teacher's list per thread, loaded before the pass over the row (longer lists: the rest in loops).
struct ListEntry { int id; float v, x; };  // id -1: absent
template <typename T> __device__ __forceinline__ ListEntry list_entry(const T* row, int V, const T* values, const int32_t* ids, int e, int K) {
  if (e >= K || !valid_entry(values, ids, e, V)) return {-1, -INFINITY, 0.f};
  return {ids[e], to_f32<T>(values[e]), to_f32<T>(row[ids[e]])};
}
struct DistillLds {
  float2 sums[16 * 3];
  double redd[16];
  int repeated;
};

// The entries of the teacher's list, this thread's: f(entry, its place).
template <typename T, int NT, typename F>
__device__ __forceinline__ void own_entries(const T* row, int V, const T* values, const int32_t* ids, int K, ListEntry mine, F f) {
  if (mine.id >= 0) f(mine, (int)threadIdx.x);
  for (int e = threadIdx.x + NT; e < K; e += NT) {
    const ListEntry n = list_entry(row, V, values, ids, e, K);
    if (n.id >= 0) f(n, e);
  }
}
// The teacher's weights are taken relative to the largest of the list's entries and the rest, in 64 bits: the rest is in units of
// x / tau, and in fp32 its conversion would move it by whole probabilities where logits are far from 0.  An infinite entry or rest,
// or a rest of NaN, makes the sum of the weights NaN, and with it the row's loss and gradient.
struct Teacher {
  double per, scale, rest_x, m;  // 1 / tau, log2(e) / tau, rest tau, the reference
  bool has_rest;
  __device__ __forceinline__ Teacher(float list_max, const DistillArgs& a, int64_t t) {
    const float rest = a.rest ? a.rest[t] : -INFINITY;
    per = 1.0 / (double)a.tau;
    scale = per * LOG2E;
    rest_x = (double)rest * (double)a.tau;
    has_rest = !(rest == -INFINITY);
    m = has_rest ? fmax((double)list_max, rest_x) : (double)list_max;
  }
};
struct RowSums {
  ExpSum out, all, list;  // student: outside the list, all tokens; teacher: the list's entries
  bool live;
};

// The row's sums and stash from each thread's sum over the tokens outside the list (tail) or over all of them.  Every thread of the
// workgroup returns with them.
template <typename T, int NT>
__device__ __forceinline__ RowSums distill_sums(const T* row, int V, const T* values, const int32_t* ids, const DistillArgs& a, int64_t t,
                                                ListEntry mine, ExpSum own, bool repeated, DistillLds& l, float (&st)[STASH]) {
  const float c = (float)(LOG2E / (double)a.tau);
  const bool tail = a.rest != nullptr;
  ExpSum sums[3] = {own, {-FLT_MAX, 0.f}, {-FLT_MAX, 0.f}};  // outside, inside the list; the teacher's
  own_entries<T, NT>(row, V, values, ids, a.K, mine, [&](ListEntry n, int e) {
    exp_sum_add(sums[2], n.v, c);
    if (tail && (!repeated || first_of_id(values, ids, e, V))) exp_sum_add(sums[1], n.x, c);
  });
  block_exp_sums<NT, 3>(sums, c, l.sums);
  const ExpSum o = sums[0], all = tail ? exp_sum_join(o, sums[1], c) : o;
  const bool live = sums[2].s != 0.f && all.s != 0.f;  // (NaN lives)
  const Teacher te(sums[2].m, a, t);
  const float share = __builtin_amdgcn_exp2f((float)(((double)sums[2].m - te.m) * te.scale));
  const float rest = te.has_rest ? __builtin_amdgcn_exp2f((float)((te.rest_x - te.m) * te.scale)) : 0.f;
  const float weight = sums[2].s * share + rest;
  const float sr = tail ? o.s * __builtin_amdgcn_exp2f((o.m - all.m) * c) / all.s : 1.f;
  st[0] = all.m; st[1] = live ? 1.f / all.s : 0.f;
  st[2] = o.m; st[3] = live && o.s != 0.f ? (sr - rest / weight) / o.s : 0.f;
  st[4] = sums[2].m; st[5] = live ? share / weight : 0.f;
  st[6] = live ? 1.f : 0.f;
  st[7] = !tail || repeated ? 1.f : 0.f;  // (without the tail nobody looked)
  return {o, all, sums[2], live};
}
// Its loss, a small difference of large terms where student and teacher agree (it falls with tau^2 before it is scaled by it): the
// teacher's weights, the terms and their sums in 64 bits; the student's sums are fp32 as they come.
template <typename T, int NT>
__device__ __forceinline__ void distill_loss(const T* row, int V, const T* values, const int32_t* ids, const DistillArgs& a, int64_t t, float w,
                                             ListEntry mine, const RowSums& r, DistillLds& l, float* loss) {
  const Teacher te(r.list.m, a, t);
  double weight = 0.0, part = 0.0;
  if (r.live)
    own_entries<T, NT>(row, V, values, ids, a.K, mine, [&](ListEntry n, int) {
      const double v = (double)n.v - te.m, p = exp2_or_nan(v * te.scale);
      weight += p;
      if (p > 1e-300) part += p * (v - ((double)n.x - (double)r.all.m)) * te.per;
    });
  weight = block_sum<NT>(weight, l.redd);
  part = block_sum<NT>(part, l.redd);
  if (threadIdx.x != 0) return;
  if (r.live) {
    const double v = te.rest_x - te.m, p = te.has_rest ? exp2_or_nan(v * te.scale) : 0.0;
    weight += p;
    if (p > 1e-300) part += p * ((v - ((double)r.out.m - (double)r.all.m)) * te.per - log_f64((double)r.out.s));
    part = part / weight + (log_f64((double)r.all.s) - log_f64(weight));
  }
  *loss = r.live ? (float)((double)w * a.tau * a.tau * part) : 0.f;
}
template <typename T, int NT>
__device__ __forceinline__ void distill_row(const T* row, int V, const T* values, const int32_t* ids, const DistillArgs& a, int64_t t, float w,
                                            ListEntry mine, ExpSum own, bool repeated, DistillLds& l, float (&st)[STASH], float* loss) {
  const RowSums r = distill_sums<T, NT>(row, V, values, ids, a, t, mine, own, repeated, l, st);
  distill_loss<T, NT>(row, V, values, ids, a, t, w, mine, r, l, loss);
}

// The gradient of one segment: the tokens outside the list in one pass of 16-byte loads and stores, then those in the list.
template <typename T, int NT>
__device__ __forceinline__ void distill_grad(const T* row, int V, const Span<T>& sp, const T* values, const int32_t* ids,
                                             const DistillArgs& a, const float (&st)[STASH], float f, T* out) {
  constexpr int E = Span<T>::E;
  const float c = (float)(LOG2E / (double)a.tau);
  const bool together = (((uintptr_t)out ^ (uintptr_t)row) & 15) == 0;  // (vectors of the gradient are vectors of the logits)
  const float mo = st[2], co = st[3] * f;
  if (st[6] == 0.f) {  // (the logits are not read: they may hold anything)
    const float zero[E] = {};
    for (int v = sp.v0 + threadIdx.x; v < sp.v1; v += NT) {
      T* p = out + sp.head + v * E;
      if (together) VecIO<T, E>::store(p, zero);
      else
        for (int e = 0; e < E; ++e) p[e] = from_f32<T>(0.f);
    }
    if (sp.first && (int)threadIdx.x < sp.head) out[threadIdx.x] = from_f32<T>(0.f);
    if (sp.last && sp.tail + (int)threadIdx.x < V) out[sp.tail + threadIdx.x] = from_f32<T>(0.f);
    return;
  }
  auto grad = [&](float x) { return __builtin_amdgcn_exp2f((x - mo) * c) * co; };
  uint4 d[Span<T>::U];
  sp.template begin<NT, true>(row, d);
  sp.template each<NT, true>(row, V, d, [&](const float (&x)[E], int v) {
    float g[E];
#pragma unroll
    for (int e = 0; e < E; ++e) g[e] = grad(x[e]);
    T* p = out + sp.head + v * E;
    if (together) VecIO<T, E>::store(p, g);
    else
#pragma unroll
      for (int e = 0; e < E; ++e) p[e] = from_f32<T>(g[e]);
  }, [&](int i) { out[i] = from_f32<T>(grad(to_f32<T>(row[i]))); });
  __threadfence_block();  // (the list's tokens are written again, by other threads)
  __syncthreads();
  for (int e = threadIdx.x; e < a.K; e += NT) {
    if (!valid_entry(values, ids, e, V) || !sp.owns(ids[e])) continue;
    bool mine = true;
    float te = 0.f;
    const bool single = st[7] == 0.f;
    for (int j = single ? e : 0; j < (single ? e + 1 : a.K) && mine; ++j)
      if (ids[j] == ids[e] && valid_entry(values, ids, j, V)) {
        mine = j >= e;
        te += __builtin_amdgcn_exp2f((to_f32<T>(values[j]) - st[4]) * c) * st[5];
      }
    if (mine) out[ids[e]] = from_f32<T>((__builtin_amdgcn_exp2f((to_f32<T>(row[ids[e]]) - st[0]) * c) * st[1] - te) * f);
  }
}

// LOSS: loss and, without GRAD, the stash; GRAD: the gradient, from this pass's numbers or (not LOSS) the stash.  LOSS takes whole
// rows (grid n x 1), GRAD alone may have them cut (grid n x nseg).  Bound by memory: 2048 rows of 131072 bf16, k 64, loss 129-165 us
// (537 MB), gradient 178 us (1074 MB, 6.0 TB/s).
template <typename T, int NT, bool LOSS, bool GRAD>
__global__ __launch_bounds__(NT) void distill_kernel(const T* __restrict__ logits, int64_t ld, int V, DistillArgs a,
                                                     float* __restrict__ loss, float* __restrict__ stash,
                                                     const float* __restrict__ upstream, T* __restrict__ grad, int64_t ld_grad) {
  extern __shared__ uint32_t member[];
  __shared__ DistillLds l;
  const int64_t t = blockIdx.x;
  const float w = a.weights ? a.weights[t] : 1.f, c = (float)(LOG2E / (double)a.tau);
  const T* row = logits + t * ld;
  const T* values = (const T*)a.values + t * a.K;
  const int32_t* ids = a.ids + t * a.K;
  const Span<T> sp(row, V, blockIdx.y, gridDim.y);
  float st[STASH] = {};
  if (LOSS) {
    if (w != 0.f) {
      const ListEntry mine = list_entry(row, V, values, ids, threadIdx.x, a.K);
      const ExpSum o = distill_sum<T, NT>(row, V, sp, values, ids, a.K, a.rest != nullptr, c, member, &l.repeated);
      distill_row<T, NT>(row, V, values, ids, a, t, w, mine, o, l.repeated != 0, l, st, loss + t);
    } else if (threadIdx.x == 0) {
      loss[t] = 0.f;
    }
    if (!GRAD && threadIdx.x < STASH) {
      float v = 0.f;
#pragma unroll
      for (int i = 0; i < STASH; ++i) v = (int)threadIdx.x == i ? st[i] : v;
      stash[t * STASH + threadIdx.x] = v;
    }
  } else {
#pragma unroll
    for (int i = 0; i < STASH; ++i) st[i] = stash[t * STASH + i];
  }
  if (GRAD) distill_grad<T, NT>(row, V, sp, values, ids, a, st, w * a.tau * (upstream ? upstream[t] : 1.f), grad + t * ld_grad);
}

// Loss and gradient with the row in registers, read once: NT * 16 vectors of 16 bytes.  4096 x 32768 bf16, k 32: 130 us, against the
// 105 of reading and writing it once at the rate of a copy; two passes, the second from the memory-side cache, took 168.  2048 x 65536
// by 512 threads: 134 us; 4096 rows of 1000, where most of the 16 vectors a thread are empty: 50.
template <typename T, int NT>
__global__ __launch_bounds__(NT, 4) void distill_resident_kernel(const T* __restrict__ logits, int64_t ld, int V, DistillArgs a,
                                                                  float* __restrict__ loss, T* __restrict__ grad, int64_t ld_grad) {
  extern __shared__ uint32_t member[];
  __shared__ DistillLds l;
  constexpr int VPT = 16, E = Span<T>::E;
  const int64_t t = blockIdx.x;
  const float w = a.weights ? a.weights[t] : 1.f, c = (float)(LOG2E / (double)a.tau);
  const T* row = logits + t * ld;
  const T* values = (const T*)a.values + t * a.K;
  const int32_t* ids = a.ids + t * a.K;
  T* out = grad + t * ld_grad;
  const Span<T> sp(row, V, 0, 1);
  float st[STASH] = {};
  if (w == 0.f) {
    if (threadIdx.x == 0) loss[t] = 0.f;
    distill_grad<T, NT>(row, V, sp, values, ids, a, st, 0.f, out);
    return;
  }
  Segment<T, NT, VPT> sg;
  sg.load(row, V, 0, 1);
  const ListEntry mine = list_entry(row, V, values, ids, threadIdx.x, a.K);
  const bool tail = a.rest != nullptr;
  // bits as in distill_sum: element i at i - head + E
  const int off = E - sp.head;
  for (int i = threadIdx.x; i < (V + 2 * E + 31) / 32; i += NT) member[i] = 0;
  if (threadIdx.x == 0) l.repeated = 0;
  __syncthreads();
  auto mark = [&](int id) {
    const int b = id + off;
    if (atomicOr(&member[b >> 5], 1u << (b & 31)) >> (b & 31) & 1) l.repeated = 1;
  };
  if (mine.id >= 0) mark(mine.id);
  for (int e = threadIdx.x + NT; e < a.K; e += NT)
    if (valid_entry(values, ids, e, V)) mark(ids[e]);
  __syncthreads();
  const uint8_t* bytes = reinterpret_cast<const uint8_t*>(member);
  auto is_member = [&](int i) { return (member[(i + off) >> 5] >> ((i + off) & 31) & 1) != 0; };
  if (tail)  // the list's tokens leave the row here: their gradient is written at the end
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int at = j * NT + (int)threadIdx.x + 1;
      const uint32_t in = sg.has(j) ? (uint32_t)(E == 8 ? bytes[at] : bytes[at >> 1] >> (at & 1) * 4 & 15) : 0;
      if (in) {
        sg.remove(j, in);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  ExpSum o = {-FLT_MAX, 0.f};
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    float x[E];
    unpack(sg.d[j], x);
    exp_sum_vec<E, true>(o, x, vec_max<E>(x), c);
    __builtin_amdgcn_sched_barrier(0);  // (one vector unpacked at a time: the others' values would not fit the registers)
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (sg.end_at[i] >= 0 && !(tail && is_member(sg.end_at[i]))) exp_sum_add(o, sg.ends[i], c);
  const RowSums sums = distill_sums<T, NT>(row, V, values, ids, a, t, mine, o, l.repeated != 0, l, st);
  const float f = w * a.tau, mo = st[2], co = st[3] * f;
  const bool together = (((uintptr_t)out ^ (uintptr_t)row) & 15) == 0, live = st[6] != 0.f;
  auto g_of = [&](float x) { return live ? __builtin_amdgcn_exp2f((x - mo) * c) * co : 0.f; };
  sg.fresh();
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    if (!sg.has(j)) continue;
    float x[E];
    unpack(sg.d[j], x);
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = g_of(x[e]);
    T* p = out + sg.index(j);
    if (together) VecIO<T, E>::store(p, x);
    else
#pragma unroll
      for (int e = 0; e < E; ++e) p[e] = from_f32<T>(x[e]);
    __builtin_amdgcn_sched_barrier(0);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (sg.end_at[i] >= 0) out[sg.end_at[i]] = from_f32<T>(g_of(sg.ends[i]));
  // (only now: in 64 bits it would not fit the registers beside the row)
  distill_loss<T, NT>(row, V, values, ids, a, t, w, mine, sums, l, loss + t);
  if (!live) return;
  __threadfence_block();  // (the list's tokens are written again, by other threads)
  __syncthreads();
  const bool repeated = l.repeated != 0;
  for (int e = threadIdx.x; e < a.K; e += NT) {
    const ListEntry n = e < NT ? mine : list_entry(row, V, values, ids, e, a.K);
    if (n.id < 0) continue;
    bool first = true;
    float te = 0.f;
    for (int j = repeated ? 0 : e; j < (repeated ? a.K : e + 1) && first; ++j)
      if (ids[j] == n.id && valid_entry(values, ids, j, V)) {
        first = j >= e;
        te += __builtin_amdgcn_exp2f((to_f32<T>(values[j]) - st[4]) * c) * st[5];
      }
    if (first) out[n.id] = from_f32<T>((__builtin_amdgcn_exp2f((n.x - st[0]) * c) * st[1] - te) * f);
  }
}

// Few or long rows: the sums of a row's segments, then the row's loss and stash from them.  64 rows of 32003 fp32, k 20, in 7
// segments: 5 + 6 us, the gradient 10.
template <typename T, int NT>
__global__ __launch_bounds__(NT) void distill_part_kernel(const T* __restrict__ logits, int64_t ld, int V, DistillArgs a,
                                                          float4* __restrict__ parts) {
  extern __shared__ uint32_t member[];
  __shared__ float red[16];
  __shared__ int repeated;
  const int64_t t = blockIdx.x;
  const int seg = blockIdx.y, nseg = gridDim.y;
  if (a.weights && a.weights[t] == 0.f) return;
  const float c = (float)(LOG2E / (double)a.tau);
  const T* row = logits + t * ld;
  const Span<T> sp(row, V, seg, nseg);
  const ExpSum o = block_exp_sum<NT>(distill_sum<T, NT>(row, V, sp, (const T*)a.values + t * a.K, a.ids + t * a.K, a.K, a.rest != nullptr, c,
                                                        member, &repeated), c, red);
  if (threadIdx.x == 0) parts[t * nseg + seg] = make_float4(o.m, o.s, a.rest && repeated ? 1.f : 0.f, 0.f);
}

template <typename T, int NT>
__global__ __launch_bounds__(NT) void distill_join_kernel(const T* __restrict__ logits, int64_t ld, int V, DistillArgs a, int nseg,
                                                          const float4* __restrict__ parts, float* __restrict__ loss,
                                                          float* __restrict__ stash) {
  __shared__ DistillLds l;
  const int64_t t = blockIdx.x;
  const float w = a.weights ? a.weights[t] : 1.f, c = (float)(LOG2E / (double)a.tau);
  const T* row = logits + t * ld;
  const T* values = (const T*)a.values + t * a.K;
  const int32_t* ids = a.ids + t * a.K;
  float st[STASH] = {};
  if (w != 0.f) {
    const ListEntry mine = list_entry(row, V, values, ids, threadIdx.x, a.K);
    ExpSum o = {-FLT_MAX, 0.f};
    bool repeated = false;
    for (int s = threadIdx.x; s < nseg; s += NT) {
      const float4 p = parts[t * nseg + s];
      o = exp_sum_join(o, {p.x, p.y}, c);
      repeated = repeated || p.z != 0.f;
    }
    repeated = __syncthreads_or(repeated);
    distill_row<T, NT>(row, V, values, ids, a, t, w, mine, o, repeated, l, st, loss + t);
  } else if (threadIdx.x == 0) {
    loss[t] = 0.f;
  }
  if (threadIdx.x < STASH) {
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < STASH; ++i) v = (int)threadIdx.x == i ? st[i] : v;
    stash[t * STASH + threadIdx.x] = v;
  }
}

// ------------------------------------------------------------------ vocabularies of at most 64 entries: G lanes a row
// One lane per entry, G = 32 (two rows a wave) or 64.  The fill loop's 30-entry rows are 120 bytes: a workgroup per row costs
// 5.5 ms at 32768 rows where one lane per entry takes 9 us for the record (k 8) and 14 us for a nucleus, both bound by the vector
// instructions of rank and sums; 16384 rows' loss and gradient 11 us, half of it the 64-bit loss.  An entry's rank is the count of the entries
// before it, read from LDS four at a time; sums run over the G lanes by DPP, in one fixed order.
template <int G> struct Group {
  template <int CTRL> static __device__ __forceinline__ int dpp(int v) { return __builtin_amdgcn_update_dpp(v, v, CTRL, 0xf, 0xf, false); }
  template <int STEP> static __device__ __forceinline__ int other(int v) {
    if constexpr (STEP == 0) return dpp<0xB1>(v);   // lane ^ 1
    if constexpr (STEP == 1) return dpp<0x4E>(v);   // lane ^ 2
    if constexpr (STEP == 2) return dpp<0x141>(v);  // mirrored in 8: the other four
    if constexpr (STEP == 3) return dpp<0x140>(v);  // mirrored in 16: the other eight
    if constexpr (STEP == 4) return __builtin_amdgcn_ds_swizzle(v, 0x401F);  // lane ^ 16
    if constexpr (STEP == 5) return __shfl_xor(v, 32, 64);
  }
  template <int STEP> static __device__ __forceinline__ float other(float v) { return __int_as_float(other<STEP>(__float_as_int(v))); }
  template <int STEP> static __device__ __forceinline__ double other(double v) {
    return __hiloint2double(other<STEP>(__double2hiint(v)), other<STEP>(__double2loint(v)));
  }
  template <typename T, typename Op> static __device__ __forceinline__ T all(T v, Op op) {
    v = op(v, other<0>(v)); v = op(v, other<1>(v)); v = op(v, other<2>(v)); v = op(v, other<3>(v)); v = op(v, other<4>(v));
    if constexpr (G == 64) v = op(v, other<5>(v));
    return v;
  }
  static __device__ __forceinline__ float max(float v) { return all(v, [](float a, float b) { return fmaxf(a, b); }); }
  static __device__ __forceinline__ int min(int v) { return all(v, [](int a, int b) { return a < b ? a : b; }); }
  template <typename T> static __device__ __forceinline__ T sum(T v) { return all(v, [](T a, T b) { return a + b; }); }
};

// The number of entries before this lane's (key, v) in its row: those u < v with a key at least this one, those u > v with a larger
// one.  Keys in LDS, G per row, those past V zero.  The lanes behind u are a constant of the unrolled step, so a step is a select, a
// comparison and an addition of its carry.
template <int G> __device__ __forceinline__ int rank_of(const uint32_t* keys, int V, uint32_t key) {
  const int v = threadIdx.x & (G - 1);
  const uint32_t next = key + 1;  // (no key is ~0)
  int rank = 0;
#pragma unroll
  for (int u = 0; u < G; u += 4) {
    if (u >= V) break;
    const uint4 k = *reinterpret_cast<const uint4*>(keys + u);
    rank += k.x >= (v > u ? key : next);
    rank += k.y >= (v > u + 1 ? key : next);
    rank += k.z >= (v > u + 2 ? key : next);
    rank += k.w >= (v > u + 3 ? key : next);
  }
  return rank;
}

template <typename T, int G>
__global__ __launch_bounds__(256) void top_small_kernel(const T* __restrict__ logits, int64_t ld, int rows, int V, int K, float tau,
                                                        T* __restrict__ values, int32_t* __restrict__ ids, float* __restrict__ rest) {
  __shared__ __align__(16) uint32_t keys[256];
  const int v = threadIdx.x & (G - 1);
  const int64_t t0 = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G, t = t0 < rows ? t0 : rows - 1;
  const float c = (float)(LOG2E / (double)tau);
  const uint32_t key = v < V ? value_key(to_f32<T>(logits[t * ld + v])) : 0;
  keys[threadIdx.x] = key;
  __syncthreads();
  const int rank = rank_of<G>(keys + (threadIdx.x & ~(G - 1)), V, key);
  const float x = key_value(key);
  const bool left = v < V && rank >= K;
  const float m = Group<G>::max(left ? x : -INFINITY);
  const float sum = Group<G>::sum(left && x > -INFINITY ? __builtin_amdgcn_exp2f((x - m) * c) : 0.f);
  if (t0 >= rows) return;
  if (v < V && rank < K) {
    values[t * K + rank] = from_f32<T>(x);
    ids[t * K + rank] = v;
  }
  if (v == 0) rest[t] = m == -INFINITY || m == INFINITY ? m : (float)((double)m * (1.0 / (double)tau) + (double)logf(sum));
}

template <typename T, int G>
__global__ __launch_bounds__(256) void sample_small_kernel(const T* __restrict__ logits, int64_t ld, const float* __restrict__ noise,
                                                           int64_t ld_noise, int rows, int V, SampleArgs a,
                                                           int64_t* __restrict__ pred, float* __restrict__ conf) {
  __shared__ __align__(16) uint32_t keys[256];
  __shared__ __align__(16) double weights[256];
  const int v = threadIdx.x & (G - 1), first = threadIdx.x & ~(G - 1);
  const int64_t t0 = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G, t = t0 < rows ? t0 : rows - 1;
  const RowFilter f = a.row(t);
  const uint32_t key = v < V ? value_key(to_f32<T>(logits[t * ld + v])) : 0;
  const float q = v < V ? noise[t * ld_noise + v] : 1.f;
  const float x = v < V ? key_value(key) : -INFINITY;
  const float m = Group<G>::max(x);
  const bool greedy = !(f.temperature > 0.f);
  double w = 0.0;
  if (v < V) w = x == m ? 1.0 : greedy ? 0.0 : exp2_f64(((double)x - (double)m) * (LOG2E / (double)f.temperature));
  keys[threadIdx.x] = key;
  __syncthreads();
  bool keep = v < V && x > -INFINITY && f.above_min_p(x, m);
  double total;
  if (f.top_p < 1.f && !greedy) {
    // weights in the row's order, in multiples of 2^-40 as for wider vocabularies (by fixed()'s rounding; sums of 64 are exact), their
    // running sum, and from it how many entries stay: an entry does while the mass before it is below the share of the first k's
    const int rank = rank_of<G>(keys + first, V, key);
    weights[first + rank] = (w + 4096.0) - 4096.0;  // (lanes past V: key 0, w 0, ranks V.. by their lane)
    const int nk = f.top_k > 0 && f.top_k < V ? f.top_k : V;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const double mine = weights[threadIdx.x];
    double upto = mine;
#pragma unroll
    for (int o = 1; o < G; o <<= 1) {
      const double up = __shfl_up(upto, o, G);
      upto += v >= o ? up : 0.0;
    }
    const double mass = __shfl(upto, nk - 1, G);
    const uint64_t in = __ballot(v < nk && (v == 0 || upto - mine < (double)f.top_p * mass));
    const int n = __popcll(G == 64 ? in : (threadIdx.x & 32) ? in >> 32 : in & 0xffffffffu);
    keep = keep && rank < n;
    total = Group<G>::sum(keep ? w : 0.0);
  } else {
    if (f.top_k > 0 && f.top_k < V) keep = keep && rank_of<G>(keys + first, V, key) < f.top_k;
    if (greedy) keep = keep && x == m;
    total = Group<G>::sum(keep ? w : 0.0);
  }
  // the race: in fp32 (relative error below 2^-21) to find who can win, in 64 bits where more than one can
  const float r = keep ? ((float)w > 0.f ? (float)w / q : 0.f) : -1.f;
  const float top = Group<G>::max(greedy ? (keep ? 1.f : -1.f) : r);
  bool win = keep && (greedy || r >= top * (1.f - 0x1p-18f));
  const uint64_t ballot = __ballot(win), mine = G == 64 ? ballot : (threadIdx.x & 32) ? ballot >> 32 : ballot & 0xffffffffu;
  if (!greedy && __popcll(mine) > 1) {
    const double e = win ? (w > 0.0 ? w / (double)q : 0.0) : -1.0;
    const double best = Group<G>::all(e, [](double p, double s) { return p > s ? p : s; });
    win = win && e == best;
  }
  int at = Group<G>::min(win ? v : G);
  if (at == G) at = Group<G>::min(keep && x == m ? v : G);  // (noise without a usable draw)
  if (t0 >= rows) return;
  if (m == -INFINITY) {
    if (v == 0) pred[t] = a.empty, conf[t] = 0.f;
  } else if (v == at) {
    pred[t] = v;
    conf[t] = greedy ? 1.f : (float)(w / total);
  }
}

// exp((x - m) / temperature) in 64 bits, 0 for -inf; NaN stays NaN (an infinite x makes one).
__device__ __forceinline__ double weight_f64(float x, float m, double scale) {
  const float d = x - m;
  return d != d ? (double)NAN : x == -INFINITY ? 0.0 : exp2_f64(((double)x - (double)m) * scale);
}

// Distillation, V and K <= G: the row, its entries and every sum in one group's registers; an entry's teacher probability reaches
// its token's lane through LDS, added up over the list in order (an id that occurs twice adds twice).
// LOSS: forward (loss, stash); GRAD: the gradient, from this pass's own numbers (LOSS) or from the stash.
template <typename T, int G, bool LOSS, bool GRAD>
__global__ __launch_bounds__(256) void distill_small_kernel(const T* __restrict__ logits, int64_t ld, int rows, int V, DistillArgs a,
                                                            float* __restrict__ loss, float* __restrict__ stash,
                                                            const float* __restrict__ upstream, T* __restrict__ grad,
                                                            int64_t ld_grad) {
  __shared__ float xs[256];
  __shared__ __align__(16) int list_id[256];
  __shared__ __align__(16) float list_p[256];
  const int v = threadIdx.x & (G - 1), first = threadIdx.x & ~(G - 1);
  const int64_t t0 = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G, t = t0 < rows ? t0 : rows - 1;
  const double per = 1.0 / (double)a.tau, scale = per * LOG2E;
  const float c = (float)scale;
  const float w = a.weights ? a.weights[t] : 1.f;
  const bool on = w != 0.f;  // (a row of weight 0 is not read)
  const float x = on && v < V ? to_f32<T>(logits[t * ld + v]) : -INFINITY;
  int id = -1;
  float val = -INFINITY;
  if (on && v < a.K) {
    id = a.ids[t * a.K + v];
    val = to_f32<T>(((const T*)a.values)[t * a.K + v]);
  }
  const bool entry = (uint32_t)id < (uint32_t)V && val > -INFINITY;
  float all_m, all_s, o_m, coef, te_m, te_inv, live;
  xs[threadIdx.x] = x;
  list_id[threadIdx.x] = entry ? id : -1;
  if (LOSS) {
    __syncthreads();
    bool member = false;
    for (int e = 0; e < a.K; ++e) member = member || list_id[first + e] == v;
    const bool tail = a.rest != nullptr;
    all_m = Group<G>::max(v < V ? x : -INFINITY);  // (NaN and +inf reach the sums)
    all_m = all_m == -INFINITY ? 0.f : all_m;
    const bool out = v < V && !(tail && member);
    o_m = Group<G>::max(out ? x : -INFINITY);
    o_m = o_m == -INFINITY ? 0.f : o_m;
    // In 64 bits, as where the rows are long (distill_row): weights, sums and the terms of the loss.
    const double mass = v < V ? weight_f64(x, out ? o_m : all_m, scale) : 0.0;
    const double o_s = Group<G>::sum(out ? mass : 0.0), in_s = Group<G>::sum(out ? 0.0 : mass);
    const double o_all = o_s == 0.0 ? 0.0 : o_s * exp2_f64(((double)o_m - (double)all_m) * scale), sum = o_all + in_s;
    const float rest = tail ? a.rest[t] : -INFINITY;
    const bool has_rest = on && !(rest == -INFINITY);
    te_m = Group<G>::max(entry ? val : -INFINITY);
    const bool entries = te_m > -INFINITY;
    if (te_m == -INFINITY) te_m = 0.f;
    const double rest_x = (double)rest * (double)a.tau, tm = has_rest ? fmax((double)te_m, rest_x) : (double)te_m;
    const double rest_e = has_rest ? exp2_or_nan((rest_x - tm) * scale) : 0.0;
    const double mine = entry ? exp2_or_nan(((double)val - tm) * scale) : 0.0;
    const double te_s = Group<G>::sum(mine) + rest_e;
    const bool counts = entries && sum != 0.0;  // (NaN counts)
    double part = 0.0;
    if (mine > 1e-300) part = mine * (((double)val - tm) - ((double)xs[first + id] - (double)all_m)) * per;
    part = Group<G>::sum(part);
    if (rest_e > 1e-300) part += rest_e * ((rest_x - tm - ((double)o_m - (double)all_m)) * per - log_f64(o_s));
    part = part / te_s + (log_f64(sum) - log_f64(te_s));
    const float t_s = 1.f / (float)te_s;
    te_inv = (float)exp2_f64(((double)te_m - tm) * scale) * t_s;
    all_s = 1.f / (float)sum;
    coef = o_s != 0.0 ? ((tail ? (float)o_all * all_s : 1.f) - (float)rest_e * t_s) / (float)o_s : 0.f;
    live = counts ? 1.f : 0.f;
    if (v == 0 && t0 < rows) {
      loss[t] = counts ? (float)((double)w * a.tau * a.tau * part) : 0.f;
      if (!GRAD) {
        float* st = stash + t * STASH;
        *reinterpret_cast<float4*>(st) = make_float4(all_m, counts ? all_s : 0.f, o_m, counts ? coef : 0.f);
        *reinterpret_cast<float4*>(st + 4) = make_float4(te_m, counts ? te_inv : 0.f, live, 0.f);
      }
    }
  } else {
    const float4 s0 = *reinterpret_cast<const float4*>(stash + t * STASH), s1 = *reinterpret_cast<const float4*>(stash + t * STASH + 4);
    all_m = s0.x; all_s = s0.y; o_m = s0.z; coef = s0.w; te_m = s1.x; te_inv = s1.y; live = s1.z;
  }
  if (!GRAD) return;
  list_p[threadIdx.x] = entry ? __builtin_amdgcn_exp2f((val - te_m) * c) * te_inv : 0.f;  // (one expression, so one result, for both ways)
  __syncthreads();
  bool member = false;
  float tv = 0.f;
  for (int e = 0; e < a.K; ++e) {
    const bool hit = list_id[first + e] == v;
    member = member || hit;
    tv += hit ? list_p[first + e] : 0.f;
  }
  const float f = w * a.tau * (upstream ? upstream[t] : 1.f);
  float g = member ? __builtin_amdgcn_exp2f((x - all_m) * c) * all_s - tv : __builtin_amdgcn_exp2f((x - o_m) * c) * coef;
  if (live == 0.f) g = 0.f;
  else g *= f;
  if (t0 < rows && v < V) grad[t * ld_grad + v] = from_f32<T>(g);
}

int check_launch() { return hipGetLastError() == hipSuccess ? PG_OK : PG_ERR_LAUNCH; }

// A launch counts its threads in 32 bits: no call with more rows than that leaves for so many threads a row (their number rounded up to
// a workgroup's eight).
bool fits(int rows, int threads) { return ((int64_t)rows + 8) * threads < 1ll << 32; }

int check_rows(int dtype, const void* logits, int64_t ld, int T, int V) {
  if (!logits || T <= 0 || V <= 0 || ld < 0 || (dtype != PG_F32 && dtype != PG_BF16)) return PG_ERR_ARG;
  return V > MAX_VOCAB || !fits(T, 32) ? PG_ERR_UNSUPPORTED : PG_OK;
}
bool small_rows(int V, int k) { return V <= 64 && k <= 64; }
int check_distill(int dtype, const void* logits, int64_t ld, int T, int V, const void* values, const int32_t* ids, int k,
                  float tau) {
  const int rc = check_rows(dtype, logits, ld, T, V);
  if (rc != PG_OK) return rc;
  if (!values || !ids || k <= 0 || !(tau >= MIN_TAU && tau <= MAX_TAU)) return PG_ERR_ARG;
  return k > MAX_K || !fits(T, !small_rows(V, k) ? 256 : V <= 32 && k <= 32 ? 32 : 64) ? PG_ERR_UNSUPPORTED : PG_OK;
}

template <typename T>
int top_rows(const T* x, int64_t ld, int n, int V, int k, float tau, T* values, int32_t* ids, float* rest, void* ws, hipStream_t s) {
  const Cut cut = cut_rows(sizeof(T) == 4 ? PG_F32 : PG_BF16, n, V, k);
  if (cut.nt) {
    SegHead* heads = (SegHead*)ws;
    uint64_t* lists = (uint64_t*)(heads + (int64_t)n * cut.nseg);
    const dim3 grid(n, cut.nseg);
    by_cut(cut, [&](auto nt, auto vpt, auto many) {
      constexpr int NT = decltype(nt)::value;
      hipLaunchKernelGGL((top_segment_kernel<T, NT, decltype(vpt)::value, decltype(many)::value>), grid, dim3(NT), 0, s, x, ld, V, k, cut.cap,
                         cut.count, tau, values, ids, rest, heads, lists);
    });
    if (cut.nseg > 1)
      hipLaunchKernelGGL((top_merge_kernel<T, 256>), dim3(n), dim3(256), 0, s, cut.nseg, k, cut.cap, tau, values, ids, rest, heads, lists);
    return check_launch();
  }
  if (V <= 32)
    hipLaunchKernelGGL((top_small_kernel<T, 32>), dim3((n + 7) / 8), dim3(256), 0, s, x, ld, n, V, k, tau, values, ids, rest);
  else if (V <= 64)
    hipLaunchKernelGGL((top_small_kernel<T, 64>), dim3((n + 3) / 4), dim3(256), 0, s, x, ld, n, V, k, tau, values, ids, rest);
  else
    hipLaunchKernelGGL((top_kernel<T, 256>), dim3(n), dim3(256), 0, s, x, ld, V, k, tau, values, ids, rest);
  return check_launch();
}

// The entries the segments look for: k itself where it is one number up to 512, else 128, the end of most nucleus and min-p
// sets.  No segments where they could not end the kept set: no filter at all, or a larger k that only top_p or nothing can undercut.
bool few_long_rows(int T, int V) { return T <= 256 && V >= 16384; }  // (more rows: each that the lists leave by one workgroup)
int sample_k(int top_k) { return top_k > 0 && top_k <= MAX_SEG_K ? (top_k < 16 ? 16 : top_k) : 128; }
Cut sample_cut(int dtype, int T, int V, const SampleArgs& a) {
  const bool rows = a.temps || a.ks || a.ps || a.mins;
  const bool by_k = a.top_k > 0 && a.top_k <= MAX_SEG_K && a.top_k < V, large_k = a.top_k > MAX_SEG_K && a.top_k < V;
  const bool ends = by_k || (!large_k && a.top_p < 1.f) || a.min_p > 0.f || a.temperature == 0.f;
  // (few rows are cut into parts behind the lists, whatever the filters)
  if (!rows && !ends && !few_long_rows(T, V)) return {0, 0, 0, 0, false, 1};
  return cut_rows(dtype, T, V, sample_k(a.ks ? 0 : a.top_k));
}
// The segments' lists hold the first k of every row.
bool settled(const Cut& cut, const SampleArgs& a) { return cut.nt && !a.ks && a.top_k > 0 && a.top_k <= MAX_SEG_K; }
// Parts of a row that the lists do not settle, 0: whole rows only.
int split_parts(int dtype, int T, int V, const SampleArgs& a) {
  const bool both = !a.ks && a.top_k > MAX_SEG_K && a.top_k < V && !a.ps && a.top_p < 1.f;
  const Cut cut = sample_cut(dtype, T, V, a);
  if (settled(cut, a) || both || !few_long_rows(T, V) || cut.nt == 0) return 0;
  int parts = 1024 / T;
  if (parts > V / 8192) parts = V / 8192;
  return parts > 16 ? 16 : parts < 2 ? 2 : parts;
}

template <typename T>
int sample_rows(const T* x, int64_t ld, const float* q, int64_t ldq, int n, int V, const SampleArgs& a, int64_t* pred, float* conf,
                void* ws, hipStream_t s) {
  if (V <= 32)
    hipLaunchKernelGGL((sample_small_kernel<T, 32>), dim3((n + 7) / 8), dim3(256), 0, s, x, ld, q, ldq, n, V, a, pred, conf);
  else if (V <= 64)
    hipLaunchKernelGGL((sample_small_kernel<T, 64>), dim3((n + 3) / 4), dim3(256), 0, s, x, ld, q, ldq, n, V, a, pred, conf);
  else {
    const Cut cut = sample_cut(sizeof(T) == 4 ? PG_F32 : PG_BF16, n, V, a);
    SegHead* heads = (SegHead*)ws;
    uint64_t* lists = (uint64_t*)(heads + (int64_t)n * cut.nseg);
    const dim3 grid(n, cut.nseg);
    const int K = sample_k(a.ks ? 0 : a.top_k);
    if (cut.nt)
      by_cut(cut, [&](auto nt, auto vpt, auto many) {
        constexpr int NT = decltype(nt)::value;
        hipLaunchKernelGGL((sample_segment_kernel<T, NT, decltype(vpt)::value, decltype(many)::value>), grid, dim3(NT), 0, s, x, ld, V, a, K,
                           cut.cap, cut.count, heads, lists);
      });
    const int parts = split_parts(sizeof(T) == 4 ? PG_F32 : PG_BF16, n, V, a);
    SplitRow* split = parts ? (SplitRow*)(lists + (int64_t)n * cut.nseg * cut.cap) : nullptr;
    if (cut.nt)
      hipLaunchKernelGGL((sample_list_kernel<T, 256>), dim3(n), dim3(256), 0, s, q, ldq, V, a, cut.nseg, cut.cap, heads, lists, pred, conf,
                         (uint64_t*)split, (int64_t)(sizeof(SplitRow) / 8));
    if (parts) {
      hipLaunchKernelGGL((sample_bins_kernel<T, 512>), dim3(n, parts), dim3(512), 0, s, x, ld, V, a, pred, conf, split);
      hipLaunchKernelGGL((sample_part_kernel<T, 512>), dim3(n, parts), dim3(512), 0, s, x, ld, q, ldq, V, a, pred, conf, split);
      hipLaunchKernelGGL((sample_join_kernel<256>), dim3(n), dim3(256), 0, s, q, ldq, V, a, parts, pred, conf, split);
    }
    if (!settled(cut, a))
      hipLaunchKernelGGL((sample_row_kernel<T, 512>), dim3(n), dim3(512), 0, s, x, ld, q, ldq, V, a, cut.nt == 0, pred, conf);
  }
  return check_launch();
}

template <typename T, bool LOSS, bool GRAD>
int distill_small(const T* x, int64_t ld, int n, int V, const DistillArgs& a, float* loss, float* stash, const float* up, T* grad,
                  int64_t ldg, hipStream_t s) {
  if (V <= 32 && a.K <= 32)
    hipLaunchKernelGGL((distill_small_kernel<T, 32, LOSS, GRAD>), dim3((n + 7) / 8), dim3(256), 0, s, x, ld, n, V, a, loss, stash,
                       up, grad, ldg);
  else
    hipLaunchKernelGGL((distill_small_kernel<T, 64, LOSS, GRAD>), dim3((n + 3) / 4), dim3(256), 0, s, x, ld, n, V, a, loss, stash,
                       up, grad, ldg);
  return check_launch();
}

// Segments of a row: one where the rows fill the chip (four workgroups a CU), else as many as do, none below 1024 vectors; a
// segment's membership bits fit MAX_MEMBER.
int distill_segs(int dtype, int T, int V) {
  const int e = dtype == PG_F32 ? 4 : 8;
  int nseg = T < 1024 ? (1024 + T - 1) / T : 1;
  const int most = V / (1024 * e), least = (V + MAX_MEMBER - 1) / MAX_MEMBER;
  if (nseg > most) nseg = most;
  return nseg < least ? least : nseg < 1 ? 1 : nseg;
}
size_t member_bytes(int V, int nseg, bool tail) { return tail ? ((size_t)(V / nseg) + 64) / 32 * 4 + 16 : 0; }

template <typename T>
int distill_forward(const T* x, int64_t ld, int n, int V, const DistillArgs& a, float* loss, float* stash, void* ws, hipStream_t s) {
  if (small_rows(V, a.K))
    return distill_small<T, true, false>(x, ld, n, V, a, loss, stash, nullptr, nullptr, 0, s);
  const int nseg = distill_segs(sizeof(T) == 4 ? PG_F32 : PG_BF16, n, V);
  const size_t lds = member_bytes(V, nseg, a.rest != nullptr);
  if (nseg == 1) {
    hipLaunchKernelGGL((distill_kernel<T, 256, true, false>), dim3(n), dim3(256), lds, s, x, ld, V, a, loss, stash,
                       (const float*)nullptr, (T*)nullptr, (int64_t)0);
  } else {
    hipLaunchKernelGGL((distill_part_kernel<T, 256>), dim3(n, nseg), dim3(256), lds, s, x, ld, V, a, (float4*)ws);
    hipLaunchKernelGGL((distill_join_kernel<T, 256>), dim3(n), dim3(256), 0, s, x, ld, V, a, nseg, (const float4*)ws, loss, stash);
  }
  return check_launch();
}

template <typename T>
int distill_backward(const T* x, int64_t ld, int n, int V, const DistillArgs& a, const float* up, const float* stash, T* grad,
                     int64_t ldg, hipStream_t s) {
  if (small_rows(V, a.K))
    return distill_small<T, false, true>(x, ld, n, V, a, nullptr, const_cast<float*>(stash), up, grad, ldg, s);
  hipLaunchKernelGGL((distill_kernel<T, 256, false, true>), dim3(n, distill_segs(sizeof(T) == 4 ? PG_F32 : PG_BF16, n, V)), dim3(256),
                     0, s, x, ld, V, a, (float*)nullptr, const_cast<float*>(stash), up, grad, ldg);
  return check_launch();
}

template <typename T>
int distill_both(const T* x, int64_t ld, int n, int V, const DistillArgs& a, float* loss, T* grad, int64_t ldg, void* ws, hipStream_t s) {
  if (small_rows(V, a.K)) return distill_small<T, true, true>(x, ld, n, V, a, loss, nullptr, nullptr, grad, ldg, s);
  if (distill_segs(sizeof(T) == 4 ? PG_F32 : PG_BF16, n, V) == 1) {
    const int vecs = V / (16 / (int)sizeof(T));
    const size_t lds = member_bytes(V, 1, true);
    if (vecs <= 256 * 16)
      hipLaunchKernelGGL((distill_resident_kernel<T, 256>), dim3(n), dim3(256), lds, s, x, ld, V, a, loss, grad, ldg);
    else if (vecs <= 512 * 16)
      hipLaunchKernelGGL((distill_resident_kernel<T, 512>), dim3(n), dim3(512), lds, s, x, ld, V, a, loss, grad, ldg);
    else  // (a workgroup of 1024 holds 131072 bf16 entries, alone on its CU: 354 us for 2048 rows, two passes 312)
      hipLaunchKernelGGL((distill_kernel<T, 256, true, true>), dim3(n), dim3(256), member_bytes(V, 1, a.rest != nullptr), s, x, ld, V, a,
                         loss, (float*)nullptr, (const float*)nullptr, grad, ldg);
    return check_launch();
  }
  float* stash = (float*)ws;
  const int rc = distill_forward(x, ld, n, V, a, loss, stash, stash + (int64_t)n * STASH, s);
  return rc != PG_OK ? rc : distill_backward(x, ld, n, V, a, nullptr, stash, grad, ldg, s);
}

}  // namespace

extern "C" int64_t pg_top_logits_workspace_bytes(int dtype, int T, int V, int k) {
  if (T <= 0 || V <= 0 || k <= 0) return 0;  // (sizes that the call refuses)
  const Cut cut = cut_rows(dtype, T, V, k);
  return cut.nseg > 1 ? (int64_t)T * cut.nseg * (sizeof(SegHead) + (int64_t)cut.cap * 8) : 0;
}

extern "C" int pg_top_logits(int dtype, const void* logits, int64_t ld, int T, int V, int k, float temperature, void* values,
                             int32_t* ids, float* rest, void* workspace, int64_t workspace_bytes, void* stream) {
  const int rc = check_rows(dtype, logits, ld, T, V);
  if (rc != PG_OK) return rc;
  if (!values || !ids || !rest || k <= 0 || k > V || !(temperature >= MIN_TAU && temperature <= MAX_TAU)) return PG_ERR_ARG;
  if (k > MAX_K || !fits(T, V <= 32 ? 32 : V <= 64 ? 64 : 256)) return PG_ERR_UNSUPPORTED;
  const int64_t need = pg_top_logits_workspace_bytes(dtype, T, V, k);
  if (need && (!workspace || workspace_bytes < need)) return PG_ERR_WORKSPACE;
  if ((uintptr_t)workspace & 15) return PG_ERR_ALIGN;
  return dtype == PG_F32 ? top_rows((const float*)logits, ld, T, V, k, temperature, (float*)values, ids, rest, workspace, (hipStream_t)stream)
                         : top_rows((const bf16_t*)logits, ld, T, V, k, temperature, (bf16_t*)values, ids, rest, workspace, (hipStream_t)stream);
}

extern "C" int64_t pg_sample_filtered_workspace_bytes(int dtype, int T, int V, int top_k) {
  if (T <= 0 || V <= 0 || top_k < 0) return 0;
  const Cut cut = cut_rows(dtype, T, V, sample_k(top_k));
  return (int64_t)T * cut.nseg * (sizeof(SegHead) + (int64_t)cut.cap * 8) + (few_long_rows(T, V) ? (int64_t)T * sizeof(SplitRow) : 0);
}

extern "C" int pg_sample_filtered(int dtype, const void* logits, int64_t ld, const float* noise, int64_t ld_noise, int T, int V,
                                  float temperature, int top_k, float top_p, float min_p, const float* temps, const int32_t* ks,
                                  const float* ps, const float* mins, int empty, int64_t* pred, float* conf, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
  const int rc = check_rows(dtype, logits, ld, T, V);
  if (rc != PG_OK) return rc;
  if (V == MAX_VOCAB) return PG_ERR_UNSUPPORTED;
  if (!noise || ld_noise < 0 || !pred || !conf || empty < -1) return PG_ERR_ARG;  // (below -1: rows still open between two launches)
  if ((!temps && !(temperature >= 0.f && temperature <= FLT_MAX)) || (!ks && top_k < 0) || (!ps && !(top_p > 0.f && top_p <= 1.f)) ||
      (!mins && !(min_p >= 0.f && min_p <= 1.f)))
    return PG_ERR_ARG;
  const SampleArgs a = {temperature, top_p, min_p, top_k, empty, temps, ks, ps, mins};
  if (!fits(T, V <= 32 ? 32 : V <= 64 ? 64 : settled(sample_cut(dtype, T, V, a), a) ? 256 : 512)) return PG_ERR_UNSUPPORTED;
  const int64_t need = pg_sample_filtered_workspace_bytes(dtype, T, V, ks ? 0 : top_k);
  if (need && (!workspace || workspace_bytes < need)) return PG_ERR_WORKSPACE;
  if ((uintptr_t)workspace & 15) return PG_ERR_ALIGN;
  return dtype == PG_F32 ? sample_rows((const float*)logits, ld, noise, ld_noise, T, V, a, pred, conf, workspace, (hipStream_t)stream)
                         : sample_rows((const bf16_t*)logits, ld, noise, ld_noise, T, V, a, pred, conf, workspace, (hipStream_t)stream);
}

extern "C" int64_t pg_distill_stash_floats(void) { return STASH; }
extern "C" int64_t pg_distill_workspace_bytes(int dtype, int T, int V, int k, int with_grad) {
  if (T <= 0 || V <= 0 || k <= 0 || small_rows(V, k)) return 0;
  const int64_t nseg = distill_segs(dtype, T, V);
  return nseg == 1 ? 0 : T * (nseg * 16 + (with_grad ? STASH * 4 : 0));
}

extern "C" int pg_distill_fwd(int dtype, const void* logits, int64_t ld, int T, int V, const void* values, const int32_t* ids,
                              int k, const float* rest, const float* weights, float temperature, float* loss, float* stash,
                              void* workspace, int64_t workspace_bytes, void* stream) {
  const int rc = check_distill(dtype, logits, ld, T, V, values, ids, k, temperature);
  if (rc != PG_OK) return rc;
  if (!loss || !stash) return PG_ERR_ARG;
  if ((uintptr_t)stash & 15) return PG_ERR_ALIGN;
  const int64_t need = pg_distill_workspace_bytes(dtype, T, V, k, 0);
  if (need && (!workspace || workspace_bytes < need)) return PG_ERR_WORKSPACE;
  if ((uintptr_t)workspace & 15) return PG_ERR_ALIGN;
  const DistillArgs a = {values, ids, rest, weights, k, temperature};
  hipStream_t s = (hipStream_t)stream;
  return dtype == PG_F32 ? distill_forward((const float*)logits, ld, T, V, a, loss, stash, workspace, s)
                         : distill_forward((const bf16_t*)logits, ld, T, V, a, loss, stash, workspace, s);
}

extern "C" int pg_distill_bwd(int dtype, const void* logits, int64_t ld, int T, int V, const void* values, const int32_t* ids,
                              int k, const float* weights, float temperature, const float* dloss, const float* stash,
                              void* dlogits, int64_t ld_dlogits, void* stream) {
  const int rc = check_distill(dtype, logits, ld, T, V, values, ids, k, temperature);
  if (rc != PG_OK) return rc;
  if (!stash || !dlogits || ld_dlogits < V) return PG_ERR_ARG;
  if ((uintptr_t)stash & 15) return PG_ERR_ALIGN;
  const DistillArgs a = {values, ids, nullptr, weights, k, temperature};
  hipStream_t s = (hipStream_t)stream;
  return dtype == PG_F32
             ? distill_backward((const float*)logits, ld, T, V, a, dloss, stash, (float*)dlogits, ld_dlogits, s)
             : distill_backward((const bf16_t*)logits, ld, T, V, a, dloss, stash, (bf16_t*)dlogits, ld_dlogits, s);
}

extern "C" int pg_distill_loss_grad(int dtype, const void* logits, int64_t ld, int T, int V, const void* values,
                                    const int32_t* ids, int k, const float* rest, const float* weights, float temperature,
                                    float* loss, void* dlogits, int64_t ld_dlogits, void* workspace, int64_t workspace_bytes,
                                    void* stream) {
  const int bad = check_distill(dtype, logits, ld, T, V, values, ids, k, temperature);
  if (bad != PG_OK) return bad;
  if (!loss || !dlogits || ld_dlogits < V) return PG_ERR_ARG;
  if (V / (dtype == PG_F32 ? 4 : 8) > 256 * 16 && !fits(T, 512)) return PG_ERR_UNSUPPORTED;  // (rows in the registers of 512 threads)
  const int64_t need = pg_distill_workspace_bytes(dtype, T, V, k, 1);
  if (need && (!workspace || workspace_bytes < need)) return PG_ERR_WORKSPACE;
  if ((uintptr_t)workspace & 15) return PG_ERR_ALIGN;
  const DistillArgs a = {values, ids, rest, weights, k, temperature};
  hipStream_t s = (hipStream_t)stream;
  return dtype == PG_F32
             ? distill_both((const float*)logits, ld, T, V, a, loss, (float*)dlogits, ld_dlogits, workspace, s)
             : distill_both((const bf16_t*)logits, ld, T, V, a, loss, (bf16_t*)dlogits, ld_dlogits, workspace, s);
}
