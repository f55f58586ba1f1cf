// Distillation from a teacher's K stored top logits: the loss, its gradient, and both in one call.
//
//   p_k = exp(t_k / T) / sum_j exp(t_j / T)       over a row's K stored entries (index < 0 or t = -inf: no entry)
//   q_v = exp(x_v / T) / sum_u exp(x_u / T)       over the whole vocabulary
//   loss = w T^2 sum_k p_k (log p_k - log q_{i_k})
//   d loss / d x_v = w T (q_v - sum_{k: i_k = v} p_k)
//
// A row takes two passes: a running maximum and sum give the softmax statistics, then q is written everywhere and the
// K entries are written over it.  All sums are fp32, the gradient is rounded once.  Exponentials are 2^(x c - M) with
// c = log2(e) / T and M = RN(m c), one fma and one hardware exponential each.
// Three kernels, by the size of the problem (distill_launch):
//   rows    rows of up to 16 KB: every warp takes rows of its own, copied into shared memory some rows ahead
//   stream  larger rows: persistent CTAs (or clusters that share a row's columns), a ring of bulk copies
//   split   few rows: one CTA or one cluster per row
#include <cooperative_groups.h>

#include <atomic>

#include "loss_common.cuh"

namespace cg = cooperative_groups;

namespace lpmm_b200 {

enum { DISTILL_LOSS = 0, DISTILL_BOTH = 1, DISTILL_GRAD = 2 };

constexpr int MAX_K = LPMM_B200_DISTILL_MAX_K;

// saved per row for the gradient: maximum and sum of the student's exponentials, the same of the teacher's (its sum is
// NaN where an entry is invalid)
struct __align__(16) RowStats {
  float m, s, tm, ts;
};

struct DistillArgs {
  const void* logits;
  void* grad;
  const void* teacher;
  const void* index;
  const float* weights;
  const float* upstream;
  float* row_loss;
  RowStats* stats;
  const float* norm;  // 1 / sum of the weights, for the mean; with few rows the kernels sum the weights themselves
  int own_norm;
  long long rows, inner, outer_stride, inner_stride, grad_outer_stride, grad_inner_stride;
  int vocab, k, teacher_dtype, index_bits, upstream_per_row;
  float temperature, c;  // c = log2(e) / T
  float scale;
  int slice;             // stream, split: columns per CTA of the cluster
  int k_pad, mark_bits;  // entries per row rounded up; bits that find an index given twice
  int stages, resident;  // stream: chunks in the ring; a row stays in it for both passes.  rows: rows ahead per warp
  int slot;              // rows: bytes of a row in shared memory
  int tellers;           // stream: warps that prepare entries
};

constexpr float LOWEST = -3.402823466e38f;
constexpr float FAR = 16777216.0f;  // 2^24
constexpr float LN2 = 0.6931471805599453f;

// The exponent at x = m is what the rounding of M left of m c: at most 1 up to |m c| = FAR, beyond it soon more than an
// exponential can hold.  A running maximum below -FAR (columns at a mask's value, whatever that is) therefore counts as -FAR:
// its terms are 2^(x c + FAR), next to nothing.  A row whose own maximum lies beyond FAR to either side is done with
// (x - m) c instead.
__device__ __forceinline__ float ref_of(float m, float c) { return fmaxf(m * c, -FAR); }
__device__ __forceinline__ bool far_off(float m, float c) { return !(fabsf(m * c) <= FAR); }

// s stands for s * 2^ref_of(m).  m starts at the lowest finite value: a -inf logit then adds 2^-inf = 0, and a NaN or
// +inf reaches s.
struct Running {
  float m, s;
};

__device__ __forceinline__ Running join(const Running& a, const Running& b, float c) {
  Running r;
  r.m = fmaxf(a.m, b.m);
  const float ref = ref_of(r.m, c);
  r.s = a.s * ex2(ref_of(a.m, c) - ref) + b.s * ex2(ref_of(b.m, c) - ref);
  return r;
}

__device__ __forceinline__ Running warp_join(Running r, float c) {
  float m = r.m;
#pragma unroll
  for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, d));
  float s = r.s * ex2(ref_of(r.m, c) - ref_of(m, c));
#pragma unroll
  for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(~0u, s, d);
  return Running{m, s};
}

// N vectors of 16 bytes
template <typename T, int N>
__device__ __forceinline__ void take(Running& r, const uint4* u, float c) {
  using E = Elem<T>;
  const float m = fmaxf(r.m, E::template maximum<N>(u));
  const float ref = ref_of(m, c);
  r.s *= ex2(ref_of(r.m, c) - ref);
  r.m = m;
  const f2 c2 = f2_splat(c), ref2 = f2_splat(-ref);
  f2 sum[2] = {f2_splat(0.0f), f2_splat(0.0f)};
#pragma unroll
  for (int j = 0; j < N; ++j) {
    float x[E::VE];
    E::unpack(u[j], x);
#pragma unroll
    for (int i = 0; i < E::VE; i += 2) {
      float a, b;
      f2_unpack(f2_fma(f2_pack(x[i], x[i + 1]), c2, ref2), a, b);
      sum[i / 2 % 2] = f2_add(sum[i / 2 % 2], f2_pack(ex2(a), ex2(b)));
    }
  }
  float a, b;
  f2_unpack(f2_add(sum[0], sum[1]), a, b);
  r.s += a + b;
}

__device__ __forceinline__ void take_one(Running& r, float x, float c) {
  const float m = fmaxf(r.m, x), ref = ref_of(m, c);
  r.s = r.s * ex2(ref_of(r.m, c) - ref) + ex2(fmaf(x, c, -ref));
  r.m = m;
}

// The exponentials of one row: 2^(x c - M), or 2^((x - m) c) where M is out of range.
struct Expo {
  float m, c, ref;
  bool far;
  __device__ __forceinline__ Expo(float m_, float c_) : m(m_), c(c_), ref(ref_of(m_, c_)), far(far_off(m_, c_)) {}
  __device__ __forceinline__ float log2_of(float x) const { return far ? (x - m) * c : fmaf(x, c, -ref); }
  __device__ __forceinline__ float operator()(float x) const { return ex2(log2_of(x)); }
  template <typename T>
  __device__ __forceinline__ uint4 scaled(const uint4& u, float g) const {
    using E = Elem<T>;
    float x[E::VE];
    E::unpack(u, x);
    if (!far) {
      const f2 c2 = f2_splat(c), ref2 = f2_splat(-ref), g2 = f2_splat(g);
#pragma unroll
      for (int i = 0; i < E::VE; i += 2) {
        float a, b;
        f2_unpack(f2_fma(f2_pack(x[i], x[i + 1]), c2, ref2), a, b);
        f2_unpack(f2_mul(f2_pack(ex2(a), ex2(b)), g2), x[i], x[i + 1]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < E::VE; ++i) x[i] = g * ex2((x[i] - m) * c);
    }
    return E::pack(x);
  }
};

template <typename T>
__device__ __forceinline__ const T* logits_row(const DistillArgs& a, long long row) {
  return reinterpret_cast<const T*>(a.logits) + row_at(row, a.inner, a.outer_stride, a.inner_stride);
}
template <typename T>
__device__ __forceinline__ T* grad_row(const DistillArgs& a, long long row) {
  return reinterpret_cast<T*>(a.grad) + row_at(row, a.inner, a.grad_outer_stride, a.grad_inner_stride);
}

// Columns [lo, hi) of a row in steps of 16 bytes: up to VE - 1 single columns before the first boundary, vectors, the
// rest singly.
struct Span {
  int lo, head, vecs, tail, tail_at;
};
template <typename T>
__device__ __forceinline__ Span span_of(const T* row, int lo, int hi) {
  constexpr int VE = Elem<T>::VE;
  Span s;
  s.lo = lo;
  const int n = hi - lo;
  const int off = (int)(((uintptr_t)(row + lo) & 15) / sizeof(T));
  s.head = off ? min(VE - off, n) : 0;
  s.vecs = (n - s.head) / VE;
  s.tail_at = lo + s.head + s.vecs * VE;
  s.tail = hi - s.tail_at;
  return s;
}
// the single column of thread t, or -1 (threads 0 ... 2 VE - 3 have one)
template <typename T>
__device__ __forceinline__ int edge_of(const Span& s, int t) {
  constexpr int VE = Elem<T>::VE;
  if (t < VE - 1) return t < s.head ? s.lo + t : -1;
  t -= VE - 1;
  return t < s.tail ? s.tail_at + t : -1;
}

// ---------------------------------------------------------------------------------------------
// A row's stored entries in shared memory, prepared by a team of threads (a warp, or a CTA)
// ---------------------------------------------------------------------------------------------
struct Warp {  // a team of 32 threads
  static constexpr int SIZE = 32;
  __device__ __forceinline__ int rank() const { return threadIdx.x & 31; }
  __device__ __forceinline__ int size() const { return 32; }
  __device__ __forceinline__ void sync() const { __syncwarp(); }
  __device__ __forceinline__ bool any(bool v) const { return __any_sync(~0u, v); }
  __device__ __forceinline__ float max(float v) const {
#pragma unroll
    for (int d = 16; d; d >>= 1) v = fmaxf(v, __shfl_xor_sync(~0u, v, d));
    return v;
  }
  __device__ __forceinline__ float sum(float v) const {
#pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(~0u, v, d);
    return v;
  }
  __device__ __forceinline__ Running joined(Running r, float c) const { return warp_join(r, c); }
};

struct Block {  // all threads of the CTA (at most 16 warps)
  float2* red;  // [2, 16] in shared memory
  int turn = 0;
  __device__ __forceinline__ explicit Block(float2* r) : red(r) {}
  __device__ __forceinline__ int rank() const { return threadIdx.x; }
  __device__ __forceinline__ int size() const { return blockDim.x; }
  __device__ __forceinline__ void sync() const { __syncthreads(); }
  __device__ __forceinline__ bool any(bool v) const { return __syncthreads_or(v); }
  // two halves in turn: a barrier lies between a read and the next write of the same half
  __device__ __forceinline__ float2* exchange(float2 v) {
    float2* r = red + 16 * (turn ^= 1);
    if ((threadIdx.x & 31) == 0) r[threadIdx.x >> 5] = v;
    __syncthreads();
    return r;
  }
  __device__ __forceinline__ float max(float v) {
    const float2* r = exchange(make_float2(Warp().max(v), 0.0f));
    v = r[0].x;
    for (int i = 1; i < (int)(blockDim.x >> 5); ++i) v = fmaxf(v, r[i].x);
    return v;
  }
  __device__ __forceinline__ float sum(float v) {
    const float2* r = exchange(make_float2(Warp().sum(v), 0.0f));
    v = r[0].x;
    for (int i = 1; i < (int)(blockDim.x >> 5); ++i) v += r[i].x;
    return v;
  }
  __device__ __forceinline__ Running joined(Running v, float c) {
    v = warp_join(v, c);
    const float2* r = exchange(make_float2(v.m, v.s));
    const int n = blockDim.x >> 5, lane = threadIdx.x & 31;
    v = lane < n ? Running{r[lane].x, r[lane].y} : Running{LOWEST, 0.0f};
    return warp_join(v, c);
  }
};

template <typename T>
struct Entries {
  int* idx;  // [k_pad], -1: no entry
  float* z;  // [k_pad] (t - tm) c: the probability is 2^z / ts
  T* x;      // [k_pad] the student's logit
  static constexpr size_t BYTES = 8 + sizeof(T);
  __device__ __forceinline__ Entries(char* p, const DistillArgs& a)
      : idx(reinterpret_cast<int*>(p)), z(reinterpret_cast<float*>(p + 4 * a.k_pad)), x(reinterpret_cast<T*>(p + 8 * a.k_pad)) {}
};

struct Teacher {
  float w, tm, ts;
  bool live;  // weight and entries: the row has a part in the loss
};

// N entries k, k + step, ... of a row as they lie in memory: all loads of a kind one after another, whatever the types are,
// and no conversion here, which would wait for its load.  What is behind the last entry has index -1.
template <int N>
struct RawEntries {
  unsigned long long i_raw[N];
  uint32_t t_raw[N];
  __device__ __forceinline__ void load(const DistillArgs& a, long long row, int k, int step) {
    const long long first = row * a.k;
#pragma unroll
    for (int j = 0; j < N; ++j) i_raw[j] = ~0ull, t_raw[j] = 0;
    if (a.index_bits == 64) {
      const unsigned long long* p = reinterpret_cast<const unsigned long long*>(a.index) + first;
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (k + j * step < a.k) i_raw[j] = p[k + j * step];
    } else {
      const uint32_t* p = reinterpret_cast<const uint32_t*>(a.index) + first;
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (k + j * step < a.k) i_raw[j] = p[k + j * step];
    }
    if (a.teacher_dtype == LPMM_B200_DTYPE_FP32) {
      const uint32_t* p = reinterpret_cast<const uint32_t*>(a.teacher) + first;
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (k + j * step < a.k) t_raw[j] = p[k + j * step];
    } else {
      const unsigned short* p = reinterpret_cast<const unsigned short*>(a.teacher) + first;
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (k + j * step < a.k) t_raw[j] = p[k + j * step];
    }
  }
  __device__ __forceinline__ long long index(const DistillArgs& a, int j) const {
    return a.index_bits == 64 ? (long long)i_raw[j] : (long long)(int)(uint32_t)i_raw[j];
  }
  __device__ __forceinline__ float teacher(const DistillArgs& a, int j) const {
    if (a.teacher_dtype == LPMM_B200_DTYPE_FP32) return __uint_as_float(t_raw[j]);
    if (a.teacher_dtype == LPMM_B200_DTYPE_BF16) return __uint_as_float(t_raw[j] << 16);
    return __half2float(__ushort_as_half((unsigned short)t_raw[j]));
  }
};

// Columns of a CTA's part of a row that entries have named, a bit each (some columns share a bit where there are more than
// `bits`, a power of two: a pair of them is then taken for one column that occurs twice, which costs a look and no more).
// Marked and cleared entry by entry.
struct Marks {
  uint32_t* word;
  int bits;
  __device__ __forceinline__ bool mark(int column) const {
    const unsigned c = (unsigned)column & (bits - 1);
    return atomicOr(&word[c >> 5], 1u << (c & 31)) >> (c & 31) & 1;
  }
  __device__ __forceinline__ void clear(int column) const { word[((unsigned)column & (bits - 1)) >> 5] = 0; }
};

// Reads the row's entries.  GRAD: the statistics are in `st`.  The team's threads may read `e` afterwards.
template <typename T, int MODE, typename Team>
__device__ __forceinline__ Teacher prepare(const DistillArgs& a, long long row, const T* x, const Entries<T>& e, Team& team,
                                           const RowStats& st) {
  Teacher t;
  t.w = a.weights ? a.weights[row] : 1.0f;
  t.tm = LOWEST;
  bool any = false, bad = false;
  // four entries per thread at a time, first all of their loads, then all of the logits that they point to
  for (int k0 = team.rank(); k0 < a.k; k0 += 4 * team.size()) {
    RawEntries<4> raw;
    raw.load(a, row, k0, team.size());
    float v[4];
    uint32_t xr[4];
    int in[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const long long i = raw.index(a, j);
      v[j] = raw.teacher(a, j);
      const bool entry = i >= 0 && v[j] != -__int_as_float(0x7f800000);
      const bool inside = entry && i < a.vocab;  // an index outside of the vocabulary is not followed
      bad |= entry && !inside;
      any |= entry;
      in[j] = inside ? (int)i : -1;
      if (entry) t.tm = fmaxf(t.tm, v[j]);
      xr[j] = 0;
      if (inside) xr[j] = Elem<T>::raw(x + in[j]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int k = k0 + j * team.size();
      if (k < a.k) {
        e.idx[k] = in[j];
        e.z[k] = v[j];
        e.x[k] = Elem<T>::type_of(xr[j]);
      }
    }
  }
  t.live = team.any(any) && t.w != 0.0f;
  t.ts = 0.0f;
  if (!t.live) return t;
  if (MODE == DISTILL_GRAD)
    t.tm = st.tm;
  else
    t.tm = team.max(t.tm);
  float sum = 0.0f;
  for (int k = team.rank(); k < a.k; k += team.size()) {
    const float z = (e.z[k] - t.tm) * a.c;
    e.z[k] = z;
    if (e.idx[k] >= 0) sum += ex2(z);
  }
  if (MODE == DISTILL_GRAD) {
    t.ts = st.ts;
  } else {
    t.ts = team.sum(sum);
    if (team.any(bad)) t.ts = nan_f();
  }
  team.sync();
  return t;
}

// sum = sum_k 2^z_k (z_k - log2 e_k).  One logarithm, of the quotient: two that nearly cancel would each be rounded at their size.
__device__ __forceinline__ float divergence_of(float sum, float s, float ts) {
  const float r = rcp_nr(ts);
  return LN2 * (sum * r) + logf(s * r);
}

// sum_k p_k (log p_k - log q_k) of a prepared row, for all threads of the team: log2 p_k = z - log2 ts
template <typename T, typename Team>
__device__ __forceinline__ float divergence(const DistillArgs& a, const Teacher& t, const Entries<T>& e, Team& team,
                                            const Expo& ex, float s) {
  float sum = 0.0f;
  for (int k = team.rank(); k < a.k; k += team.size()) {
    const float z = e.z[k], p = ex2(z);
    if (e.idx[k] < 0 || p == 0.0f) continue;
    sum += p * (z - ex.log2_of(Elem<T>::widen(e.x[k])));
  }
  return divergence_of(team.sum(sum), s, t.ts);
}

// Marks the entries' columns within [lo, hi); true for a thread that found one marked.
template <typename T, typename Team>
__device__ __forceinline__ bool mark_entries(const DistillArgs& a, const Entries<T>& e, const Team& team, const Marks& marks,
                                             int lo, int hi) {
  bool twice = false;
  for (int k = team.rank(); k < a.k; k += team.size()) {
    const int i = e.idx[k];
    if (i >= lo && i < hi) twice |= marks.mark(i - lo);
  }
  return twice;
}

// The entries' columns within [lo, hi): q - p, written over q.  After a barrier behind the stores of q and the marks, which
// are cleared here.
template <typename T, typename Team>
__device__ __forceinline__ void write_entries(const DistillArgs& a, T* g, const Entries<T>& e, const Team& team,
                                              const Marks& marks, bool twice, const Expo& ex, float gs, float G, float ts,
                                              int lo, int hi) {
  const float Gp = G * rcp_nr(ts);
  for (int k = team.rank(); k < a.k; k += team.size()) {
    const int i = e.idx[k];
    if (i < lo || i >= hi) continue;
    marks.clear(i - lo);
    float p = ex2(e.z[k]);
    if (twice) {  // an index that occurs several times: its first entry writes for all, in their order
      bool first = true;
      for (int j = 0; j < k; ++j) first &= e.idx[j] != i;
      if (!first) continue;
      for (int j = k + 1; j < a.k; ++j)
        if (e.idx[j] == i) p += ex2(e.z[j]);
    }
    g[i] = Elem<T>::narrow(gs * ex(Elem<T>::widen(e.x[k])) - Gp * p);
  }
}

// brings a row's entries into L2
__device__ __forceinline__ void prefetch_entries(const DistillArgs& a, long long row) {
  const char* i = reinterpret_cast<const char*>(a.index) + row * a.k * (a.index_bits / 8);
  const int ni = a.k * (a.index_bits / 8), size = a.teacher_dtype == LPMM_B200_DTYPE_FP32 ? 4 : 2;
  const char* t = reinterpret_cast<const char*>(a.teacher) + row * a.k * size;
  const int lane = threadIdx.x & 31;
  for (int at = lane * 128; at < ni; at += 32 * 128) prefetch_l2(i + at);
  for (int at = lane * 128; at < a.k * size; at += 32 * 128) prefetch_l2(t + at);
}

// The gradient's factor that all rows share, for whole warps.  With few rows its norm is 1 / sum of the weights (0 if that is
// 0), added up here: in double and in the order of distill_reduce_kernel (32 rows by a tree, these sums one after another), so
// that gradient and loss are means over the same number, also where weights of both signs cancel.  `load` and `get` lie apart
// where there is work to do in between.
constexpr int OWN_NORM_ROWS = 256;
__device__ __noinline__ float far_reciprocal(double w) { return w == 0.0 ? 0.0f : (float)(1.0 / w); }
struct SharedFactor {
  float v[OWN_NORM_ROWS / 32], norm;
  __device__ __forceinline__ void load(const DistillArgs& a) {
    norm = a.norm ? *a.norm : 1.0f;
#pragma unroll
    for (int i = 0; i < OWN_NORM_ROWS / 32; ++i) {
      const int r = i * 32 + (threadIdx.x & 31);
      v[i] = a.own_norm && r < a.rows ? a.weights[r] : 0.0f;
    }
  }
  __device__ __forceinline__ float get(const DistillArgs& a) const {
    float n = norm;
    if (a.own_norm) {
      double w = 0.0;
#pragma unroll
      for (int i = 0; i < OWN_NORM_ROWS / 32; ++i) {
        if (i * 32 >= a.rows) break;
        double t = v[i];
#pragma unroll
        for (int d = 16; d; d >>= 1) t += __shfl_xor_sync(~0u, t, d);
        w += t;
      }
      const float f = (float)w;  // an fp32 division is off by one rounding more than one in double and much shorter
      n = fabsf(f) > 1e-30f && fabsf(f) < 1e30f ? 1.0f / f : far_reciprocal(w);
    }
    return a.scale * a.temperature * n;
  }
};
__device__ __forceinline__ float shared_factor(const DistillArgs& a) {
  SharedFactor f;
  f.load(a);
  return f.get(a);
}
__device__ __forceinline__ float upstream_of(const DistillArgs& a, long long row) {
  return a.upstream ? a.upstream[a.upstream_per_row ? row : 0] : 1.0f;
}

// Statistics of a row whose maximum lies beyond FAR, from its logits in memory.
template <typename T, typename Team>
__device__ __noinline__ float far_sum(const DistillArgs& a, const T* x, int lo, int hi, float m, Team& team) {
  float s = 0.0f;
  for (int v = lo + team.rank(); v < hi; v += team.size()) s += ex2((Elem<T>::widen(x[v]) - m) * a.c);
  return team.sum(s);
}

// ---------------------------------------------------------------------------------------------
// rows: every warp takes rows of its own; their logits are copied into its slots of shared memory some rows ahead, the
// entries of the next row are loaded into registers (KV per lane).  A warp needs no barrier with others, and a gathered logit
// comes from shared memory.  Bound by instructions: about 900 per row and warp beside its columns (loss and gradient of
// 512 MB of bf16 logits, 64 entries: 4096 columns 316 us = 0.53 of the copy rate, 1000 columns 426 us = 0.42).
// ---------------------------------------------------------------------------------------------
constexpr int ROWS_MAX_WARPS = 8, ROWS_MAX_STAGES = 4, ROWS_MAX_BYTES = 16384;
constexpr size_t rows_room(int ctas) { return 227 * 1024 / ctas - 2048; }  // shared memory of a CTA

// What a warp loads of its next row
template <typename T, int MODE, int KV>
struct RowFetch : RawEntries<KV> {
  uint32_t edge_raw;
  float w, up;
  RowStats st;
  __device__ __forceinline__ void load(const DistillArgs& a, long long row) {
    const int lane = threadIdx.x & 31;
    if (row >= a.rows) return;
    w = a.weights ? a.weights[row] : 1.0f;
    RawEntries<KV>::load(a, row, lane, 32);
    const T* x = logits_row<T>(a, row);
    const int at = edge_of<T>(span_of(x, 0, a.vocab), lane);
    edge_raw = Elem<T>::none().x;
    if (at >= 0) edge_raw = Elem<T>::raw(x + at);
    if (MODE == DISTILL_GRAD) {
      st = a.stats[row];
      up = a.upstream[a.upstream_per_row ? row : 0];
    }
  }
  __device__ __forceinline__ float edge() const { return Elem<T>::of_raw(edge_raw); }
};

template <typename T, int MODE, int KV>
__global__ void __launch_bounds__(ROWS_MAX_WARPS * 32, KV <= 2 ? 3 : 2) distill_rows_kernel(const DistillArgs a) {
  using E = Elem<T>;
  extern __shared__ __align__(16) char smem[];
  __shared__ unsigned long long full[ROWS_MAX_WARPS][ROWS_MAX_STAGES];
  __shared__ int failed;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  char* slots = smem + warp * a.stages * a.slot;
  if (lane == 0) {
    for (int i = 0; i < a.stages; ++i) mbar_init(&full[warp][i], 1);
    mbar_fence();
  }
  if (threadIdx.x == 0) failed = 0;
  __syncthreads();
  const int rows = (int)a.rows, stride = gridDim.x * warps, row0 = blockIdx.x * warps + warp;
  // bit i of `dead`: row number 32 n + i of this warp has weight 0 and is not copied; `dead_next`: of the next 32
  auto weights_of = [&](int it) {
    const long long r = row0 + (long long)(it + lane) * stride;
    return __ballot_sync(~0u, a.weights && r < rows && a.weights[r] == 0.0f);
  };
  uint32_t dead = weights_of(0), dead_next = weights_of(32);
  auto copy = [&](long long row, int st, bool none) {
    if (lane != 0 || row >= rows) return;
    const T* x = logits_row<T>(a, row);
    const Span o = span_of(x, 0, a.vocab);
    const uint32_t n = none ? 0 : o.vecs * 16;
    mbar_expect(&full[warp][st], n);
    if (n) bulk_load(slots + st * a.slot, x + o.head, n, &full[warp][st]);
  };
  for (int i = 0; i < a.stages; ++i) copy(row0 + (long long)i * stride, i, dead >> i & 1);
  RowFetch<T, MODE, KV> next;
  next.load(a, row0);
  pdl_wait();
  const float up0 = MODE == DISTILL_LOSS ? 0.0f : shared_factor(a);
  int st = 0, it = 0;
  uint32_t phase = 0;
  long long row = row0;
  for (; row < rows; ++it, row += stride) {
    const RowFetch<T, MODE, KV> f = next;
    next.load(a, row + stride);
    const T* x = logits_row<T>(a, row);
    const Span o = span_of(x, 0, a.vocab);
    const bool edges = o.head + o.tail != 0;
    char* slot = slots + st * a.slot;
    const T* xs = reinterpret_cast<const T*>(slot);  // column `head` is its first
    const uint4* buf = reinterpret_cast<const uint4*>(slot);
    if (!__all_sync(~0u, mbar_wait(&full[warp][st], phase, &failed))) break;

    // entries
    int idx[KV];
    float z[KV], xk[KV], tm = LOWEST;
    bool any = false, bad = false;
#pragma unroll
    for (int j = 0; j < KV; ++j) {
      const long long i = f.index(a, j);
      z[j] = f.teacher(a, j);
      const bool entry = i >= 0 && z[j] != -__int_as_float(0x7f800000);
      const bool in = entry && i < a.vocab;  // an index outside of the vocabulary is not followed
      bad |= entry && !in;
      any |= entry;
      idx[j] = in ? (int)i : -1;
      if (entry) tm = fmaxf(tm, z[j]);
    }
    const bool live = __any_sync(~0u, any) && f.w != 0.0f;
    if (live) {
#pragma unroll
      for (int j = 0; j < KV; ++j) {
        const int i = idx[j];
        xk[j] = 0.0f;
        if (i >= 0) xk[j] = E::widen(i >= o.head && i < o.tail_at ? xs[i - o.head] : x[i]);
      }
      // statistics
      Running r{LOWEST, 0.0f};
      float ts = 0.0f, p[KV];
      if (MODE == DISTILL_GRAD) {
        tm = f.st.tm, ts = f.st.ts, r.m = f.st.m, r.s = f.st.s;
      } else {
        for (int v = lane; v < o.vecs; v += 128) {
          uint4 u[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) u[j] = v + 32 * j < o.vecs ? buf[v + 32 * j] : E::none();
          take<T, 4>(r, u, a.c);
        }
        if (edges) take_one(r, f.edge(), a.c);
        float m = r.m;
#pragma unroll
        for (int d = 16; d; d >>= 1) {
          m = fmaxf(m, __shfl_xor_sync(~0u, m, d));
          tm = fmaxf(tm, __shfl_xor_sync(~0u, tm, d));
        }
        r.s *= ex2(ref_of(r.m, a.c) - ref_of(m, a.c));
        r.m = m;
      }
#pragma unroll
      for (int j = 0; j < KV; ++j) {
        z[j] = (z[j] - tm) * a.c;
        p[j] = idx[j] >= 0 ? ex2(z[j]) : 0.0f;
        if (MODE != DISTILL_GRAD) ts += p[j];
      }
      const Expo ex(r.m, a.c);
      if (MODE != DISTILL_GRAD) {
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < KV; ++j)
          if (p[j] != 0.0f) sum += p[j] * (z[j] - ex.log2_of(xk[j]));
#pragma unroll
        for (int d = 16; d; d >>= 1) {
          r.s += __shfl_xor_sync(~0u, r.s, d);
          ts += __shfl_xor_sync(~0u, ts, d);
          sum += __shfl_xor_sync(~0u, sum, d);
        }
        if (__any_sync(~0u, bad)) ts = nan_f();
        if (ex.far) {
          Warp team;
          r.s = far_sum(a, x, 0, a.vocab, r.m, team);
          if (r.s == 0.0f) r.s = nan_f();  // every logit -inf: no distribution
        }
        if (lane == 0) {
          a.row_loss[row] = f.w * a.temperature * a.temperature * divergence_of(sum, r.s, ts);
          a.stats[row] = RowStats{r.m, r.s, tm, ts};
        }
      }
      if (MODE != DISTILL_LOSS) {
        T* g = grad_row<T>(a, row);
        uint4* gv = reinterpret_cast<uint4*>(g + o.head);
        const float G = up0 * (MODE == DISTILL_GRAD ? f.up : 1.0f) * f.w + (ts - ts);
        const float gs = G * rcp_nr(r.s), Gp = G * rcp_nr(ts);
        for (int v = lane; v < o.vecs; v += 128) {
          uint4 u[4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (v + 32 * j < o.vecs) u[j] = buf[v + 32 * j];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (v + 32 * j < o.vecs) gv[v + 32 * j] = ex.scaled<T>(u[j], gs);
        }
        if (edges) {
          const int at = edge_of<T>(o, lane);
          if (at >= 0) g[at] = E::narrow(gs * ex(f.edge()));
        }
        // the row is not needed any more: its slot shows an index that occurs twice, by the second one's number
        unsigned short* claim = reinterpret_cast<unsigned short*>(slot);
        __syncwarp();
#pragma unroll
        for (int j = 0; j < KV; ++j)
          if (idx[j] >= 0) claim[idx[j]] = (unsigned short)(lane + 32 * j);
        __syncwarp();
        bool mine[KV], twice = false;
#pragma unroll
        for (int j = 0; j < KV; ++j) {
          mine[j] = idx[j] >= 0;
          twice |= mine[j] && claim[idx[j]] != lane + 32 * j;
        }
        bulk_load_fence();
        if (__any_sync(~0u, twice)) {  // its first entry writes for all, in their order
          float all[KV];
#pragma unroll
          for (int j = 0; j < KV; ++j) all[j] = 0.0f;
#pragma unroll
          for (int q = 0; q < KV; ++q)
            for (int l = 0; l < 32; ++l) {
              const int other = __shfl_sync(~0u, idx[q], l);
              const float po = __shfl_sync(~0u, p[q], l);
#pragma unroll
              for (int j = 0; j < KV; ++j)
                if (other == idx[j]) {
                  all[j] += po;
                  if (q * 32 + l < j * 32 + lane) mine[j] = false;
                }
            }
#pragma unroll
          for (int j = 0; j < KV; ++j) p[j] = all[j];
        }
#pragma unroll
        for (int j = 0; j < KV; ++j)
          if (mine[j]) g[idx[j]] = E::narrow(gs * ex(xk[j]) - Gp * p[j]);
      }
    } else {
      if (MODE != DISTILL_GRAD && lane == 0) {
        a.row_loss[row] = 0.0f;
        a.stats[row] = RowStats{0.0f, 1.0f, 0.0f, 0.0f};
      }
      if (MODE != DISTILL_LOSS) {
        T* g = grad_row<T>(a, row);
        uint4* gv = reinterpret_cast<uint4*>(g + o.head);
        for (int v = lane; v < o.vecs; v += 32) gv[v] = make_uint4(0, 0, 0, 0);
        const int at = edge_of<T>(o, lane);
        if (at >= 0) g[at] = E::narrow(0.0f);
      }
    }
    __syncwarp();
    if ((it & 31) == 31) {
      dead = dead_next;
      dead_next = weights_of(it + 33);
    }
    // row number it + stages takes the slot; its bit is in the word of row number it + 1 or in the next one
    const int ahead = ((it + 1) & 31) + a.stages - 1;
    copy(row + (long long)a.stages * stride, st, (ahead < 32 ? dead >> ahead : dead_next >> (ahead - 32)) & 1);
    if (++st == a.stages) st = 0, phase ^= 1;
  }
  if (lane == 0)  // only where a wait ran out: the copies under way, of this row and the next ones, still have to land
    for (int i = 0; i < a.stages && row + (long long)i * stride < rows; ++i) {
      mbar_wait_landed(&full[warp][st], phase);
      if (++st == a.stages) st = 0, phase ^= 1;
    }
  __syncthreads();
  if (failed)  // a wait ran out (it never has): what this CTA wrote is not to be taken for a result
    for (row = row0; row < rows; row += stride)
      if (lane == 0) {
        if (MODE != DISTILL_GRAD) a.row_loss[row] = nan_f();
        if (MODE != DISTILL_LOSS) grad_row<T>(a, row)[0] = E::narrow(nan_f());
      }
}

// ---------------------------------------------------------------------------------------------
// stream: persistent CTAs, or clusters of them that share the columns of a row; one warp copies the rows into a ring of
// chunks, one to four prepare the entries of rows to come, four or eight take the passes.  Gathered logits, the teacher's
// softmax and the losses, a chain of latencies per row, are thus off the path that the row's columns take.
// Bound by memory and, for 16-bit types, by how many chunks' latencies four warps per scheduler hide (the pipe of the
// exponentials is 54-65 % busy).  512 MB of logits, 64 entries: loss, bf16, 32000 columns 106 us = 0.78 of the copy rate
// (fp32 97 us, 0.84); gradient 213 us, 0.77; both 225 us, 0.73 (fp32 206 us, 0.79).
// ---------------------------------------------------------------------------------------------
constexpr int PER = 4;  // vectors per consuming thread and chunk
constexpr int MAX_STAGES = 14, MAX_TELLERS = 4, MAX_PARTS = 8;

// CW: consuming warps.  Eight with chunks of 16 KB in two CTAs per SM, or four with chunks of 8 KB in four or five: more
// rows under way at a time hide what a row costs beside its columns (a reduction, a barrier or two), but leave each less
// room to stay in the ring.
template <int MODE, int CW>
struct Shape {
  static constexpr int CHUNK = 2048 * CW, THREADS = 32 * CW;
  static constexpr int CTAS = CW == 8 ? 2 : MODE == DISTILL_BOTH ? 4 : 5;
  static constexpr int TELLERS = CW == 8 ? 4 : 1;
  static constexpr size_t ROOM = 227 * 1024 / CTAS - 1024;
};

struct StreamRow {  // what the consumers are told about a row, and what they tell
  Teacher t;
  int skip;
  float m, s, G;
};

struct StreamSmem {
  unsigned long long full[MAX_STAGES], empty[MAX_STAGES];
  // per slot: entries ready / no longer read / statistics of the row known
  unsigned long long told[2 * MAX_TELLERS], freed[2 * MAX_TELLERS], stat[2 * MAX_TELLERS];
  unsigned long long joined[2];  // the statistics of all parts of a row are in `part`
  float2 part[2][MAX_PARTS];
  StreamRow row[2 * MAX_TELLERS];
  float2 red[2][8];
  int twice[4];  // of row number n in twice[n & 3]
  int failed;
};

// the consumers as a team: named barrier 1
template <int CW>
struct Consumers {
  float2 (*red)[8];
  int turn = 0;
  __device__ __forceinline__ explicit Consumers(float2 (*r)[8]) : red(r) {}
  __device__ __forceinline__ int rank() const { return threadIdx.x; }
  __device__ __forceinline__ int size() const { return CW * 32; }
  __device__ __forceinline__ void sync() const { asm volatile("bar.sync 1, %0;" ::"n"(CW * 32) : "memory"); }
  __device__ __forceinline__ float2* exchange(float2 v) {
    float2* r = red[turn ^= 1];
    if ((threadIdx.x & 31) == 0) r[threadIdx.x >> 5] = v;
    sync();
    return r;
  }
  __device__ __forceinline__ float sum(float v) {
    const float2* r = exchange(make_float2(Warp().sum(v), 0.0f));
    v = r[0].x;
    for (int i = 1; i < CW; ++i) v += r[i].x;
    return v;
  }
  // of n <= 8 values that lanes 0 ... n - 1, repeated over the warp, hold
  static __device__ __forceinline__ Running join_of(float2 o, int n, float c) {
    float m = o.x;
#pragma unroll
    for (int d = 4; d; d >>= 1)
      if (d < n) m = fmaxf(m, __shfl_xor_sync(~0u, m, d));
    float s = o.y * ex2(ref_of(o.x, c) - ref_of(m, c));
#pragma unroll
    for (int d = 4; d; d >>= 1)
      if (d < n) s += __shfl_xor_sync(~0u, s, d);
    return Running{m, s};
  }
  __device__ __forceinline__ Running joined(Running v, float c) {
    v = warp_join(v, c);
    return join_of(exchange(make_float2(v.m, v.s))[threadIdx.x % CW], CW, c);
  }
};

template <typename T, int MODE, int CW>
__global__ void __launch_bounds__(32 * (CW + 1 + Shape<MODE, CW>::TELLERS), Shape<MODE, CW>::CTAS)
    distill_stream_kernel(const DistillArgs a) {
  using E = Elem<T>;
  constexpr int CHUNK = Shape<MODE, CW>::CHUNK, CTHREADS = Shape<MODE, CW>::THREADS;
  extern __shared__ __align__(16) char smem[];
  char* ring = smem;
  StreamSmem& sm = *reinterpret_cast<StreamSmem*>(smem + (size_t)a.stages * CHUNK);
  char* entry_mem = smem + (size_t)a.stages * CHUNK + (sizeof(StreamSmem) + 15) / 16 * 16;
  const size_t per_slot = Entries<T>::BYTES * a.k_pad;
  // two sets of marks in turn where no barrier lies between the end of a row and the next one's marks
  uint32_t* mark_words = reinterpret_cast<uint32_t*>(entry_mem + 2 * a.tellers * per_slot);
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
  const int lo = min(part * a.slice, a.vocab), hi = min(lo + a.slice, a.vocab);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < a.stages; ++i) {
      mbar_init(&sm.full[i], 1);
      mbar_init(&sm.empty[i], CW);
    }
    for (int i = 0; i < 2 * a.tellers; ++i) {
      mbar_init(&sm.told[i], 1);
      mbar_init(&sm.freed[i], CW);
      mbar_init(&sm.stat[i], 1);
    }
    for (int i = 0; i < 2; ++i) mbar_init(&sm.joined[i], 1);
    sm.failed = 0;
    for (int i = 0; i < 4; ++i) sm.twice[i] = 0;
    mbar_fence();
  }
  if (MODE != DISTILL_LOSS)
    for (int i = threadIdx.x; i < a.mark_bits / 32 * (MODE == DISTILL_GRAD ? 2 : 1); i += blockDim.x) mark_words[i] = 0;
  if (parts > 1)
    cluster.sync();
  else
    __syncthreads();
  const long long grid = gridDim.x / parts, row0 = blockIdx.x / parts;
  // passes over the chunks: once where the row stays in the ring, or only one pass is made
  const int loads = MODE == DISTILL_BOTH && !a.resident ? 2 : 1;

  if (warp == CW) {  // the copies
    int st = 0, fills = 0;
    uint32_t phase = 0, skips = 0;
    long long it = 0;
    for (long long row = row0; row < a.rows; row += grid, ++it) {
      if ((it & 31) == 0) {
        const long long r = row + lane * grid;
        skips = __ballot_sync(~0u, a.weights && r < a.rows && a.weights[r] == 0.0f);
      }
      if (skips >> (it & 31) & 1) continue;
      if (lane == 0) {
        const T* x = logits_row<T>(a, row);
        const Span o = span_of(x, lo, hi);
        const char* from = reinterpret_cast<const char*>(x + lo + o.head);
        const long long bytes = (long long)o.vecs * 16;
        for (int pass = 0; pass < loads; ++pass)
          for (long long at = 0; at < bytes; at += CHUNK) {
            if (fills >= a.stages) mbar_wait(&sm.empty[st], phase ^ 1, &sm.failed);
            if (*(volatile int*)&sm.failed) break;  // nothing is copied any more
            const uint32_t n = (uint32_t)min((long long)CHUNK, bytes - at);
            mbar_expect(&sm.full[st], n);
            bulk_load(ring + (size_t)st * CHUNK, from + at, n, &sm.full[st]);
            if (fills < a.stages) ++fills;
            if (++st == a.stages) st = 0, phase ^= 1;
          }
      }
      __syncwarp();
    }
    if (lane == 0 && *(volatile int*)&sm.failed) {  // a wait ran out: the copies under way still have to land
      for (int i = 0; i < fills; ++i) {
        if (--st < 0) st = a.stages - 1, phase ^= 1;
        mbar_wait_landed(&sm.full[st], phase);
      }
    }
    __syncwarp();
  } else if (warp > CW) {  // the entries
    pdl_wait();  // *norm
    const float up0 = MODE == DISTILL_LOSS ? 0.0f : shared_factor(a);
    Warp team;
    const int teller = warp - CW - 1;
    const long long step = a.tellers * grid;
    long long before = -1;  // the row whose loss is still to be written
    int n = 0;              // rows begun; row number n has slot teller + (n & 1) * tellers
    for (long long row = row0 + teller * grid;; row += step, ++n) {
      if (row < a.rows) {
        const int slot = teller + (n & 1) * a.tellers;
        StreamRow& h = sm.row[slot];
        const Entries<T> e(entry_mem + slot * per_slot, a);
        if (n >= 2) mbar_wait(&sm.freed[slot], (n >> 1 & 1) ^ 1, &sm.failed);
        RowStats st = {0.0f, 1.0f, 0.0f, 0.0f};
        if (MODE == DISTILL_GRAD) st = a.stats[row];
        const Teacher t = prepare<T, MODE>(a, row, logits_row<T>(a, row), e, team, st);
        if (lane == 0) {
          h.t = t;
          h.skip = t.w == 0.0f;
          if (MODE == DISTILL_GRAD) h.m = st.m, h.s = st.s;
          if (MODE != DISTILL_LOSS) h.G = up0 * upstream_of(a, row) * t.w + (t.ts - t.ts);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.told[slot]);
        if (row + step < a.rows) prefetch_entries(a, row + step);
      }
      if (MODE != DISTILL_GRAD && before >= 0) {
        const int slot = teller + ((n - 1) & 1) * a.tellers;
        const StreamRow& h = sm.row[slot];
        mbar_wait(&sm.stat[slot], (n - 1) >> 1 & 1, &sm.failed);
        if (part == 0) {
          const Teacher t = h.t;
          float loss = 0.0f;
          if (t.live)
            loss = t.w * a.temperature * a.temperature *
                   divergence(a, t, Entries<T>(entry_mem + slot * per_slot, a), team, Expo(h.m, a.c), h.s);
          if (lane == 0) {
            a.row_loss[before] = loss;
            a.stats[before] = RowStats{h.m, h.s, t.tm, t.ts};
          }
        }
        __syncwarp();
      }
      if (row >= a.rows) break;
      before = row;
    }
  } else {
    const int tid = threadIdx.x;
    Consumers<CW> team(sm.red);
    int st = 0, slot = 0;
    uint32_t phase = 0, told = 0, joins = 0, number = 0;  // of live rows
    for (long long row = row0; row < a.rows; row += grid) {
      const T* x = logits_row<T>(a, row);
      T* g = MODE == DISTILL_LOSS ? nullptr : grad_row<T>(a, row);
      const Span o = span_of(x, lo, hi);
      const int chunks = (int)(((long long)o.vecs * 16 + CHUNK - 1) / CHUNK);
      const int at = edge_of<T>(o, tid);
      float edge = at >= 0 ? E::widen(x[at]) : -__int_as_float(0x7f800000);
      uint4* gv = MODE == DISTILL_LOSS ? nullptr : reinterpret_cast<uint4*>(g + lo + o.head);
      mbar_wait(&sm.told[slot], told, &sm.failed);
      StreamRow& h = sm.row[slot];
      const bool live = h.t.live;
      if (!live) {
        if (!h.skip)  // weight, but no entry: the copies are under way
          for (int i = 0; i < chunks * loads; ++i) {
            mbar_wait(&sm.full[st], phase, &sm.failed);
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.empty[st]);
            if (++st == a.stages) st = 0, phase ^= 1;
          }
        if (MODE != DISTILL_LOSS) {
          for (int i = tid; i < o.vecs; i += CTHREADS) gv[i] = make_uint4(0, 0, 0, 0);
          if (at >= 0) g[at] = E::narrow(0.0f);
        }
        if (MODE != DISTILL_GRAD && tid == 0) {
          h.m = 0.0f, h.s = 1.0f;
          mbar_arrive(&sm.stat[slot]);
        }
      } else {
        float m, s;
        const int st0 = st;
        if (MODE == DISTILL_GRAD) {
          m = h.m, s = h.s;
        } else {
          Running r{LOWEST, 0.0f};
          for (int i = 0; i < chunks; ++i) {
            mbar_wait(&sm.full[st], phase, &sm.failed);
            const uint4* buf = reinterpret_cast<const uint4*>(ring + (size_t)st * CHUNK);
            const int n = o.vecs - i * (CHUNK / 16);
            uint4 u[PER];
            if (n >= CHUNK / 16) {
#pragma unroll
              for (int j = 0; j < PER; ++j) u[j] = buf[tid + j * CTHREADS];
            } else {
#pragma unroll
              for (int j = 0; j < PER; ++j) u[j] = tid + j * CTHREADS < n ? buf[tid + j * CTHREADS] : E::none();
            }
            if (MODE == DISTILL_LOSS || !a.resident) {
              __syncwarp();
              if (lane == 0) mbar_arrive(&sm.empty[st]);
            }
            take<T, PER>(r, u, a.c);
            if (++st == a.stages) st = 0, phase ^= 1;
          }
          take_one(r, edge, a.c);
          r = team.joined(r, a.c);
          if (parts > 1) {
            // every part sends its statistics to all.  Two sets in turn: a part sends for row n + 2 after it has all of
            // row n + 1, that is after every part has read row n's.
            const int set = joins & 1;
            if (!*(volatile int*)&sm.failed) {  // a barrier whose phase did not come is not armed again
              if (tid == 0) mbar_expect(&sm.joined[set], parts * (uint32_t)sizeof(float2));
              if (tid < parts) send_async(&sm.part[set][part], make_float2(r.m, r.s), &sm.joined[set], tid);
            }
            mbar_wait_cluster(&sm.joined[set], joins >> 1 & 1, &sm.failed);
            ++joins;
            r = Consumers<CW>::join_of(sm.part[set][lane % parts], parts, a.c);
          }
          m = r.m, s = r.s;
          if (far_off(m, a.c)) {  // every part over the whole row: rare, and needs no exchange
            s = far_sum(a, x, 0, a.vocab, m, team);
            if (s == 0.0f) s = nan_f();  // every logit -inf: no distribution
          }
          if (tid == 0) {
            h.m = m, h.s = s;
            mbar_arrive(&sm.stat[slot]);
          }
        }
        if (MODE != DISTILL_LOSS) {
          const Expo ex(m, a.c);
          const float G = h.G, gs = G * rcp_nr(s);
          const Entries<T> e(entry_mem + slot * per_slot, a);
          const Marks marks{mark_words + (MODE == DISTILL_GRAD ? (number & 1) * (a.mark_bits / 32) : 0), a.mark_bits};
          // the flag of row n is read behind its barrier and cleared in row n + 2: behind the barrier of row n + 1, before that
          // of row n + 2, behind which row n + 4 sets it again
          if (mark_entries(a, e, team, marks, lo, hi)) sm.twice[number & 3] = 1;
          if (tid == 0) sm.twice[(number + 2) & 3] = 0;
          int s2 = MODE == DISTILL_BOTH && a.resident ? st0 : st;
          for (int i = 0; i < chunks; ++i) {
            if (MODE == DISTILL_GRAD || !a.resident) mbar_wait(&sm.full[s2], phase, &sm.failed);
            const uint4* buf = reinterpret_cast<const uint4*>(ring + (size_t)s2 * CHUNK);
            const int first = i * (CHUNK / 16), n = o.vecs - first;
            uint4 u[PER];
#pragma unroll
            for (int j = 0; j < PER; ++j) u[j] = buf[tid + j * CTHREADS];  // behind the row's end: not used
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.empty[s2]);
            uint4* to = gv + first + tid;
            if (n >= CHUNK / 16) {
#pragma unroll
              for (int j = 0; j < PER; ++j) to[j * CTHREADS] = ex.scaled<T>(u[j], gs);
            } else {
#pragma unroll
              for (int j = 0; j < PER; ++j)
                if (tid + j * CTHREADS < n) to[j * CTHREADS] = ex.scaled<T>(u[j], gs);
            }
            if (++s2 == a.stages) {
              s2 = 0;
              if (MODE == DISTILL_GRAD || !a.resident) phase ^= 1;
            }
          }
          if (MODE == DISTILL_GRAD || !a.resident) st = s2;
          if (at >= 0) g[at] = E::narrow(gs * ex(edge));
          team.sync();
          write_entries(a, g, e, team, marks, sm.twice[number & 3] != 0, ex, gs, G, h.t.ts, lo, hi);
          ++number;
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.freed[slot]);
      if (++slot == 2 * a.tellers) slot = 0, told ^= 1;
    }
  }
  if (parts > 1)
    cluster.sync();  // nobody leaves while another part may still send to it
  else
    __syncthreads();
  if (sm.failed)  // a wait ran out (it never has): what this CTA wrote is not to be taken for a result
    for (long long row = row0 + threadIdx.x * grid; row < a.rows; row += blockDim.x * grid) {
      if (MODE != DISTILL_GRAD) a.row_loss[row] = nan_f();
      if (MODE != DISTILL_LOSS && lo < hi) grad_row<T>(a, row)[lo] = E::narrow(nan_f());
    }
}

// ---------------------------------------------------------------------------------------------
// split: one CTA, or one cluster of CTAs that share the columns, per row: fewer rows than SMs, or more entries than the
// kernel for short rows takes.  Bound by latencies: entries, the gathered logits, the row, two barriers of the cluster (7 rows
// of 50257 bf16 columns, both: 13 us).
// ---------------------------------------------------------------------------------------------
template <typename T, int MODE>
__global__ void __launch_bounds__(512) distill_split_kernel(const DistillArgs a) {
  using E = Elem<T>;
  extern __shared__ __align__(16) char smem[];
  __shared__ float2 red[32];
  __shared__ int twice;
  __shared__ Running mine;  // this CTA's part of the row, read by the cluster
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
  const long long row = blockIdx.x / parts;
  const int tid = threadIdx.x, nthr = blockDim.x;
  const int lo = min(part * a.slice, a.vocab), hi = min(lo + a.slice, a.vocab);
  const T* x = logits_row<T>(a, row);
  T* g = MODE == DISTILL_LOSS ? nullptr : grad_row<T>(a, row);
  const Entries<T> e(smem, a);
  const Marks marks{reinterpret_cast<uint32_t*>(smem + Entries<T>::BYTES * a.k_pad), a.mark_bits};
  Block team(red);
  if (tid == 0) twice = 0;
  if (MODE != DISTILL_LOSS)
    for (int i = tid; i < a.mark_bits / 32; i += nthr) marks.word[i] = 0;
  __syncthreads();
  pdl_wait();
  RowStats st = {0.0f, 1.0f, 0.0f, 0.0f};
  if (MODE == DISTILL_GRAD) st = a.stats[row];
  const Teacher t = prepare<T, MODE>(a, row, x, e, team, st);
  if (!t.live) {  // uniform over the cluster: every CTA of it has read the same entries
    if (MODE != DISTILL_LOSS) {
      const Span o = span_of(g, lo, hi);
      const int at = edge_of<T>(o, tid);
      uint4* gv = reinterpret_cast<uint4*>(g + o.lo + o.head);
      for (int i = tid; i < o.vecs; i += nthr) gv[i] = make_uint4(0, 0, 0, 0);
      if (at >= 0) g[at] = E::narrow(0.0f);
    }
    if (MODE != DISTILL_GRAD && tid == 0 && part == 0) {
      a.row_loss[row] = 0.0f;
      a.stats[row] = st;
    }
    return;
  }
  SharedFactor factor;
  if (MODE != DISTILL_LOSS) factor.load(a);
  if (MODE != DISTILL_GRAD) {
    // one pass over the row: running maximum and sum
    const Span o = span_of(x, lo, hi);
    const int at = edge_of<T>(o, tid);
    const float edge = at >= 0 ? E::widen(x[at]) : -__int_as_float(0x7f800000);
    Running r{LOWEST, 0.0f};
    const uint4* xv = reinterpret_cast<const uint4*>(x + o.lo + o.head);
    for (int i = tid; i < o.vecs; i += 4 * nthr) {
      uint4 u[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) u[j] = i + j * nthr < o.vecs ? xv[i + j * nthr] : E::none();
      take<T, 4>(r, u, a.c);
    }
    take_one(r, edge, a.c);
    r = team.joined(r, a.c);
    if (parts > 1) {
      if (tid == 0) mine = r;
      cluster.sync();
      r = *cluster.map_shared_rank(&mine, 0);
      for (int j = 1; j < parts; ++j) r = join(r, *cluster.map_shared_rank(&mine, j), a.c);
      cluster.sync();  // nobody leaves while its part is still read
    }
    st.m = r.m;
    st.s = r.s;
    if (far_off(r.m, a.c)) {  // every CTA over the whole row: rare, and needs no exchange
      st.s = far_sum(a, x, 0, a.vocab, r.m, team);
      if (st.s == 0.0f) st.s = nan_f();  // every logit -inf: no distribution
    }
  }
  const Expo ex(st.m, a.c);
  if (MODE != DISTILL_GRAD && part == 0) {
    const float d = divergence(a, t, e, team, ex, st.s);
    if (tid == 0) {
      a.row_loss[row] = t.w * a.temperature * a.temperature * d;
      a.stats[row] = RowStats{st.m, st.s, t.tm, t.ts};
    }
  }
  if (MODE == DISTILL_LOSS) return;
  const float G = factor.get(a) * upstream_of(a, row) * t.w + (t.ts - t.ts);  // NaN for a row with invalid entries
  const float gs = G * rcp_nr(st.s);
  if (mark_entries(a, e, team, marks, lo, hi)) twice = 1;
  {
    const Span o = span_of(g, lo, hi);
    const int at = edge_of<T>(o, tid);
    if (at >= 0) g[at] = E::narrow(gs * ex(E::widen(x[at])));
    uint4* gv = reinterpret_cast<uint4*>(g + o.lo + o.head);
    const uint4* xv = reinterpret_cast<const uint4*>(x + o.lo + o.head);
    for (int i = tid; i < o.vecs; i += nthr) gv[i] = ex.scaled<T>(xv[i], gs);
  }
  __syncthreads();
  write_entries(a, g, e, team, marks, twice != 0, ex, gs, G, t.ts, lo, hi);
}

// One CTA: the sum of the weights and of the weighted row losses in a fixed order, in double (3 us up to some
// thousand rows, 5 us at 16384, 12 at 67108, 40 at 268435).
__global__ void __launch_bounds__(1024) distill_reduce_kernel(const float* __restrict__ row_loss,
                                                              const float* __restrict__ weights, long long rows, int mean,
                                                              float* __restrict__ loss, float* __restrict__ norm) {
  __shared__ double red[2][32];
  pdl_start_next();
  pdl_wait();
  double l = 0.0, w = 0.0;
  for (long long i = threadIdx.x; i < rows; i += blockDim.x) {
    if (row_loss) l += row_loss[i];
    if (mean && weights) w += weights[i];
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    l += __shfl_xor_sync(~0u, l, o);
    w += __shfl_xor_sync(~0u, w, o);
  }
  if ((threadIdx.x & 31) == 0) red[0][threadIdx.x >> 5] = l, red[1][threadIdx.x >> 5] = w;
  __syncthreads();
  if (threadIdx.x == 0) {
    l = w = 0.0;
    for (int i = 0; i < (int)(blockDim.x >> 5); ++i) l += red[0][i], w += red[1][i];
    if (mean && !weights) w = (double)rows;
    const double n = !mean ? 1.0 : w == 0.0 ? 0.0 : 1.0 / w;
    if (norm) *norm = (float)n;
    if (loss) *loss = n == 0.0 ? 0.0f : (float)(l * n);
  }
}

static int distill_check(const lpmm_b200_distill* d, int mode) {
  if (!d) return LPMM_B200_ERR_NULL_POINTER;
  if (d->rows < 0 || d->inner < 1 || d->vocab < 1 || d->k < 1) return LPMM_B200_ERR_BAD_SIZE;
  if (d->dtype < 0 || d->dtype > 2 || d->teacher_dtype < 0 || d->teacher_dtype > 2) return LPMM_B200_ERR_BAD_KIND;
  if (d->index_bits != 32 && d->index_bits != 64) return LPMM_B200_ERR_BAD_KIND;
  if (d->reduction < 0 || d->reduction > 2) return LPMM_B200_ERR_BAD_KIND;
  if (!(d->temperature >= LPMM_B200_DISTILL_MIN_T && d->temperature <= LPMM_B200_DISTILL_MAX_T)) return LPMM_B200_ERR_BAD_SIZE;
  if (d->k > MAX_K || d->vocab > (1 << 30) || d->rows >= (1ll << 28) ||
      d->inner >= (1ll << 28)) return LPMM_B200_ERR_TOO_LARGE;
  if (d->rows && (!d->logits || !d->teacher || !d->index || !d->work)) return LPMM_B200_ERR_NULL_POINTER;
  if (d->rows && mode != DISTILL_LOSS && !d->grad) return LPMM_B200_ERR_NULL_POINTER;
  if (mode != DISTILL_GRAD && !d->loss && (d->rows || d->reduction != LPMM_B200_REDUCE_NONE)) return LPMM_B200_ERR_NULL_POINTER;
  // without rows there are no values of REDUCE_NONE either, neither losses nor their derivatives
  if (mode == DISTILL_GRAD && !d->upstream && (d->rows || d->reduction != LPMM_B200_REDUCE_NONE)) return LPMM_B200_ERR_NULL_POINTER;
  if ((uintptr_t)d->work & 15) return LPMM_B200_ERR_BAD_SIZE;
  if (d->rows && mode != DISTILL_LOSS) {  // 16-byte accesses follow both
    const int64_t size = d->dtype == LPMM_B200_DTYPE_FP32 ? 4 : 2;
    if ((((uintptr_t)d->logits - (uintptr_t)d->grad) & 15) || (d->outer_stride - d->grad_outer_stride) * size % 16 ||
        (d->inner_stride - d->grad_inner_stride) * size % 16)
      return LPMM_B200_ERR_BAD_SIZE;
  }
  return LPMM_B200_OK;
}

// `most`: the most shared memory that any call gives this kernel.  The limit belongs to the kernel on the device, and other
// threads launch it too: set to one call's size it would refuse another's.
template <typename K>
static cudaError_t launch(K kernel, const DistillArgs& a, long long grid, int threads, size_t smem, size_t most, int cluster,
                          bool after, cudaStream_t stream) {
  if (smem > most) return cudaErrorInvalidValue;
  if (smem > 40 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  if (cluster > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = cluster;
    attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  if (after) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    ++cfg.numAttrs;
  }
  return cudaLaunchKernelEx(&cfg, kernel, a);
}

// How many clusters of `parts` CTAs the GPU holds at a time with all the shared memory that a call may give them, which does for
// every call: asked once per kernel, cluster, number of tellers and device.  0: none, or no answer; then it is asked again.
template <typename T, int MODE, int CW>
static int most_clusters(int parts, int threads) {
  const auto kernel = distill_stream_kernel<T, MODE, CW>;
  static std::atomic<int> known[64][4][MAX_TELLERS + 1];  // 0: not asked yet
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  std::atomic<int>& n = known[dev][parts == 2 ? 1 : parts == 4 ? 2 : 3][threads / 32 - CW - 1];
  int got = n.load();
  if (got == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(Shape<MODE, CW>::CTAS * num_sms() / parts * parts), cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = Shape<MODE, CW>::ROOM;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = parts, attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr, cfg.numAttrs = 1;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Shape<MODE, CW>::ROOM) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&got, kernel, &cfg) != cudaSuccess || got < 0)
      got = 0;
    if (got > 0) n.store(got);
  }
  return got;
}

// bits for `columns` columns: up to 8 KB
static int mark_bits(long long columns) {
  int bits = 1024;
  while (bits < columns && bits < 65536) bits *= 2;
  return bits;
}

template <typename T, int MODE, int CW>
static cudaError_t stream_launch(DistillArgs& a, long long row_bytes, bool after, cudaStream_t stream) {
  using S = Shape<MODE, CW>;
  const size_t fixed = (sizeof(StreamSmem) + 15) / 16 * 16, told = 2 * Entries<T>::BYTES * a.k_pad;
  // With both passes in one call a row stays in the ring where it fits.  Up to 128 KB it is else copied a second time: the
  // rows under way are then less than 38 MB and still in L2 (bf16, 65536 columns: 214 us, and 235 shared by a cluster).
  // Larger rows would come from memory again; clusters of CTAs share their columns (131072: 246, and 268 copied twice).
  const bool share = MODE == DISTILL_BOTH && row_bytes > 128 * 1024;
  int parts = 1;
  for (;; parts *= 2) {
    a.slice = ((a.vocab + parts - 1) / parts + 63) / 64 * 64;
    a.mark_bits = MODE == DISTILL_LOSS ? 0 : mark_bits(a.slice);
    const size_t marks = a.mark_bits / 8 * (MODE == DISTILL_GRAD ? 2 : 1);
    a.tellers = S::TELLERS;
    while (a.tellers > 1 && a.tellers * told > S::ROOM / 5) --a.tellers;
    const auto stages = [&] { return (int)((S::ROOM - fixed - marks - a.tellers * told) / S::CHUNK); };
    // long rows: as few tellers as leave the ring the most chunks
    if (share) {
      const int most = (int)((S::ROOM - fixed - marks - told) / S::CHUNK);
      while (stages() < most) --a.tellers;
    }
    a.stages = stages() < MAX_STAGES ? stages() : MAX_STAGES;
    a.resident = MODE == DISTILL_BOTH && row_bytes <= (long long)parts * (a.stages - 1) * S::CHUNK;
    if (!share || a.resident || parts == MAX_PARTS) {
      const size_t smem = a.stages * S::CHUNK + fixed + marks + a.tellers * told;
      const int threads = S::THREADS + 32 + 32 * a.tellers;
      const int clusters = parts > 1 ? most_clusters<T, MODE, CW>(parts, threads) : S::CTAS * num_sms();
      if (clusters <= 0) return cudaErrorInvalidConfiguration;
      return launch(distill_stream_kernel<T, MODE, CW>, a, (a.rows < clusters ? a.rows : clusters) * parts, threads, smem,
                    S::ROOM, parts, after, stream);
    }
  }
}

// `after`: the kernel before it in the stream is this call's sum of the weights
template <typename T, int MODE>
static cudaError_t distill_launch(DistillArgs& a, bool after, cudaStream_t stream) {
  constexpr int VE = Elem<T>::VE;
  const long long row_bytes = (long long)a.vocab * sizeof(T);
  const int sms = num_sms();
  // A warp per row up to 16 KB for the loss, 12 KB for the gradient, 8 KB for both (us, here / streaming: loss, bf16 8192 columns
  // 171 / 179, fp32 4096 130 / 155; gradient, bf16 6000 221 / 262, 8192 250 / 238; both, bf16 4096 311 / 420, 6000 362 / 373,
  // fp32 4096 341 / 234).
  constexpr long long ROW = MODE == DISTILL_LOSS ? ROWS_MAX_BYTES : MODE == DISTILL_GRAD ? ROWS_MAX_BYTES / 4 * 3 : ROWS_MAX_BYTES / 2;
  if (row_bytes <= ROW && a.k <= 256) {
    a.slot = (int)((row_bytes + 15) / 16 * 16);
    int warps = ROWS_MAX_WARPS, ctas = a.k <= 64 ? 3 : 2;
    a.stages = ROWS_MAX_STAGES;
    const auto bytes = [&] { return (size_t)warps * a.stages * a.slot; };
    const auto room = [&] { return rows_room(ctas); };
    while (a.stages > 2 && bytes() > room()) --a.stages;
    if (bytes() > room()) ctas = 2;
    while (bytes() > room()) --warps;
    long long grid = (a.rows + warps - 1) / warps;
    if (grid > ctas * sms) grid = ctas * sms;
    if (a.k <= 64) return launch(distill_rows_kernel<T, MODE, 2>, a, grid, warps * 32, bytes(), rows_room(2), 1, after, stream);
    return launch(distill_rows_kernel<T, MODE, 8>, a, grid, warps * 32, bytes(), rows_room(2), 1, after, stream);
  }
  if (a.rows >= sms && row_bytes > ROWS_MAX_BYTES / 2) {
    // Four consuming warps per CTA or eight, measured with 64 entries and 512 MB of logits (us, four / eight): the loss of
    // bf16 rows of 12000 columns 138 / 210, 32000 107 / 126, 65536 102 / 105, 131072 102 / 96; both, bf16 12000 274 / 353,
    // 20000 246 / 289, 32000 226 / 232, 50257 258 / 234, fp32 12000 197 / 212, 16000 222 / 198 (fp32 has half the
    // exponentials per byte to hide); the gradient alone is about the same (12000 194 / 200, 131072 196 / 190) and has eight.
    const long long most = MODE == DISTILL_LOSS ? 128 : MODE == DISTILL_GRAD ? 0 : sizeof(T) == 2 ? 64 : 48;
    const bool few = a.k <= 256 && row_bytes <= most * 1024;  // more entries take the room of the smaller ring
    const cudaError_t e = few ? stream_launch<T, MODE, 4>(a, row_bytes, after, stream)
                              : stream_launch<T, MODE, 8>(a, row_bytes, after, stream);
    if (e != cudaErrorInvalidConfiguration) return e;
    cudaGetLastError();  // the kernel below takes the call; the next one to ask for the last error shall not find this
  }
  // few rows: their columns are shared by clusters of up to 8 CTAs, so that all SMs have work
  int parts = 1;
  const int vecs = (a.vocab + VE - 1) / VE;
  while (parts < 8 && a.rows * parts < 2ll * sms && vecs / (parts * 2) >= 512) parts *= 2;
  a.slice = ((vecs + parts - 1) / parts + 7) / 8 * 8 * VE;
  const int per = a.slice / VE;
  const int threads = per >= 2048 ? 512 : per >= 512 ? 256 : 128;
  a.mark_bits = MODE == DISTILL_LOSS ? 0 : mark_bits(a.slice);
  return launch(distill_split_kernel<T, MODE>, a, a.rows * parts, threads, Entries<T>::BYTES * a.k_pad + a.mark_bits / 8,
                Entries<T>::BYTES * MAX_K + 65536 / 8, parts, after, stream);
}

template <int MODE>
static int distill_run(const lpmm_b200_distill* d, void* stream_) {
  const int bad = distill_check(d, MODE);
  if (bad) return bad;
  cudaStream_t stream = (cudaStream_t)stream_;
  const bool mean = d->reduction == LPMM_B200_REDUCE_MEAN, none = d->reduction == LPMM_B200_REDUCE_NONE;
  float* norm = d->work;
  DistillArgs a = {};
  a.logits = d->logits, a.grad = d->grad, a.teacher = d->teacher, a.index = d->index, a.weights = d->weights;
  a.upstream = MODE == DISTILL_GRAD ? d->upstream : nullptr;
  a.stats = reinterpret_cast<RowStats*>(d->work + 4);
  a.row_loss = none ? d->loss : d->work + 4 + 4 * d->rows;
  a.norm = mean ? norm : nullptr;
  a.rows = d->rows, a.inner = d->inner, a.outer_stride = d->outer_stride, a.inner_stride = d->inner_stride;
  a.vocab = (int)d->vocab, a.k = (int)d->k, a.teacher_dtype = d->teacher_dtype, a.index_bits = d->index_bits;
  a.upstream_per_row = none;
  a.temperature = d->temperature;
  a.c = (float)(1.4426950408889634 / (double)d->temperature);
  a.scale = d->grad_scale;
  a.grad_outer_stride = d->grad_outer_stride, a.grad_inner_stride = d->grad_inner_stride;
  a.k_pad = (a.k + 3) / 4 * 4;
  if (d->rows == 0) {
    if (MODE != DISTILL_GRAD && !none) LPMM_CUDA_TRY(cudaMemsetAsync(d->loss, 0, sizeof(float), stream));
    return LPMM_B200_OK;
  }
  bool first = MODE == DISTILL_BOTH && mean;
  if (first && (!d->weights || d->rows <= OWN_NORM_ROWS)) {
    first = false;
    a.norm = nullptr;
    if (d->weights)
      a.own_norm = 1;
    else
      a.scale = (float)((double)d->grad_scale / (double)d->rows);
  }
  if (first) {
    distill_reduce_kernel<<<1, 1024, 0, stream>>>(nullptr, d->weights, d->rows, 1, nullptr, norm);
    LPMM_CUDA_TRY(cudaGetLastError());
  }
  cudaError_t e;
  if (d->dtype == LPMM_B200_DTYPE_FP32)
    e = distill_launch<float, MODE>(a, first, stream);
  else if (d->dtype == LPMM_B200_DTYPE_BF16)
    e = distill_launch<__nv_bfloat16, MODE>(a, first, stream);
  else
    e = distill_launch<__half, MODE>(a, first, stream);
  LPMM_CUDA_TRY(e);
  if (MODE != DISTILL_GRAD && !none) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(1), cfg.blockDim = dim3(1024), cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr, cfg.numAttrs = 1;
    const float *row_loss = a.row_loss, *weights = d->weights;
    LPMM_CUDA_TRY(cudaLaunchKernelEx(&cfg, distill_reduce_kernel, row_loss, weights, (long long)d->rows, (int)mean, d->loss, norm));
  }
  return LPMM_B200_OK;
}

}  // namespace lpmm_b200

using namespace lpmm_b200;

extern "C" int64_t lpmm_b200_distill_work_floats(int64_t rows) { return rows < 0 ? LPMM_B200_ERR_BAD_SIZE : 4 + 5 * rows; }

extern "C" int lpmm_b200_distill_forward(const lpmm_b200_distill* d, void* stream) {
  return distill_run<DISTILL_LOSS>(d, stream);
}
extern "C" int lpmm_b200_distill_backward(const lpmm_b200_distill* d, void* stream) {
  return distill_run<DISTILL_GRAD>(d, stream);
}
extern "C" int lpmm_b200_distill_forward_backward(const lpmm_b200_distill* d, void* stream) {
  return distill_run<DISTILL_BOTH>(d, stream);
}
