// The load-balance loss of a router, the assignments per expert, and the loss's gradient.
//
//   p = softmax(x), or sigmoid(x) / sum sigmoid(x), over a token's experts;  c_e = assignments of the sequence to e
//   loss = F sum_e c_e sum_n p_ne,   d loss / d x_ne = F p_ne (c_e - sum_j c_j p_nj) [(1 - sigmoid(x_ne))],
//   F = experts / (k n^2), n = valid tokens of the sequence
//
// The gradient needs the counts, not the summed scores, so loss and gradient share one pass over the logits once the
// indices are counted.  A token's logits lie in the registers of up to 32 lanes, some tokens per warp at a time; a warp
// walks a contiguous run of tokens and sums the scores of its columns in registers, in fp32.  Those sums (of MAX_RUN tokens at
// most, so that their rounding does not grow with the batch) meet as 64-bit whole numbers, in units of 2^-shift with
// tokens * 2^shift < 2^62: atomics on them give the same result in any order, and what is rounded off is far below fp32 of the
// scores' sum (of the loss, whose usual size is 1, at most experts * tokens * 2^-62).
// Bound by memory for large batches (a logit is read once, a gradient written once), by launches for small ones: these
// are done in one launch of a CTA or a cluster, larger ones in three (clear, count, scores; the last CTA adds up).
#include <cooperative_groups.h>

#include "loss_common.cuh"

namespace cg = cooperative_groups;

namespace lpmm_b200 {

constexpr int MAX_WARPS = 16;
constexpr int MAX_RUN = 512;  // tokens whose scores are summed in fp32: reached from 1.2 million tokens on

struct BalanceArgs {
  const void* logits;
  void* grad;
  const void* index;
  const uint8_t* valid;
  const void* offsets;
  const float* upstream;
  float* loss;
  unsigned long long* counts;  // [sequences, experts]
  unsigned long long* counts_out;  // the same for the caller to hand on, or nullptr
  float* factor;
  unsigned long long* psum;    // [sequences, experts] summed scores in units of 2^-shift
  unsigned long long* sizes;   // valid tokens per sequence
  int* bad;                    // per sequence: 1 an index out of range, 2 a score that is NaN; [sequences]: offsets not in order
  unsigned* ticket;            // CTAs that are done
  long long inner, outer_stride, inner_stride;
  int tokens, sequences, tile, experts, k, index_bits, offset_bits, sigmoid, group, shift;
  int finish;                  // the last CTA of the scores adds up
  float scale;
};

__device__ __forceinline__ long long raw_offset(const BalanceArgs& a, int i) {
  if (!a.offsets) return i == 0 ? 0 : a.tokens;
  return load_index(a.offsets, i, a.offset_bits);
}
// Offsets kept within [0, tokens], in shared memory where there are few: a search is then a matter of nanoseconds.
constexpr int SHARED_OFFSETS = 1024;
struct Offsets {
  int at[SHARED_OFFSETS + 1];
};
__device__ __forceinline__ int clamped_offset(const BalanceArgs& a, int i) {
  return (int)min(max(raw_offset(a, i), 0ll), (long long)a.tokens);
}
__device__ __forceinline__ void load_offsets(const BalanceArgs& a, Offsets& o) {
  if (a.offsets && a.sequences <= SHARED_OFFSETS)
    for (int i = threadIdx.x; i <= a.sequences; i += blockDim.x) o.at[i] = clamped_offset(a, i);
  __syncthreads();
}
__device__ __forceinline__ int offset_at(const BalanceArgs& a, const Offsets& o, int i) {
  return a.sequences <= SHARED_OFFSETS ? o.at[i] : clamped_offset(a, i);
}

// The stretch of tokens from r on that belongs to one sequence: s in [0, sequences), or s < 0 for tokens of none.
// Whatever the offsets hold, r < end <= hi and s is in range.
struct Stretch {
  int s, end;
};
__device__ __forceinline__ Stretch stretch_at(const BalanceArgs& a, const Offsets& o, int r, int hi) {
  if (!a.offsets) return Stretch{0, hi};
  int lo = -1, up = a.sequences + 1;  // offset(lo) <= r < offset(up)
  while (up - lo > 1) {
    const int mid = (lo + up) >> 1;
    if (offset_at(a, o, mid) <= r)
      lo = mid;
    else
      up = mid;
  }
  if (lo == a.sequences) return Stretch{-1, hi};
  return Stretch{lo, max(min(offset_at(a, o, lo + 1), hi), r + 1)};
}

__device__ __forceinline__ long long cell(const BalanceArgs& a, int s, int e) { return (long long)s * a.experts + e; }

// (what earlier phases of the same launch have written is read past L1)
__device__ __forceinline__ double factor_of(const BalanceArgs& a, int s) {
  const int bad = __ldcg(&a.bad[s]), off = __ldcg(&a.bad[a.sequences]);
  const double n = (double)__ldcg(&a.sizes[s]);
  if ((bad & 1) | off) return (double)nan_f();
  return n == 0.0 ? 0.0 : (double)a.experts / ((double)a.k * n * n);
}

// An expert's count for the gradient, less that of the first expert: c_e - sum_j c_j p_j does not change with a constant, for the
// scores add up to 1, and in a well balanced sequence the differences are small next to the counts: even counts give exactly 0.
__device__ __forceinline__ float count_of(const BalanceArgs& a, int s, int e) {
  return (float)(long long)(__ldcg(&a.counts[cell(a, s, e)]) - __ldcg(&a.counts[cell(a, s, 0)]));
}

// A CTA's part of the tokens.  What its first and its last sequence gather is put together in shared memory (they may
// have many tokens here); sequences between them lie within the CTA and go straight to memory.
struct Tile {
  int lo, hi, first, last;
  __device__ __forceinline__ Tile(const BalanceArgs& a, const Offsets& o, int cta) {
    lo = (int)min((long long)cta * a.tile, (long long)a.tokens);
    hi = min(lo + a.tile, a.tokens);
    first = last = -1;
    if (lo < hi) {
      first = stretch_at(a, o, lo, hi).s;
      last = stretch_at(a, o, hi - 1, hi).s;
    }
  }
  // this warp's run
  __device__ __forceinline__ void run(int& from, int& to) const {
    const int warps = blockDim.x >> 5, n = (hi - lo + warps - 1) / warps;
    from = min(lo + (int)(threadIdx.x >> 5) * n, hi);
    to = min(from + n, hi);
  }
  __device__ __forceinline__ int set(int s) const { return s == first ? 0 : s == last ? 1 : -1; }
};

// Assignments per expert and valid tokens per sequence.  hist: int[2, experts] in shared memory
__device__ __forceinline__ void count_phase(const BalanceArgs& a, const Offsets& o, int cta, int* hist) {
  const int lane = threadIdx.x & 31;
  if (cta == 0 && a.offsets) {
    bool off = false;
    for (int i = threadIdx.x; i <= a.sequences; i += blockDim.x) {
      const long long at = raw_offset(a, i);
      off |= at < 0 || at > a.tokens || (i && raw_offset(a, i - 1) > at);
    }
    if (off) a.bad[a.sequences] = 1;
  }
  for (int e = threadIdx.x; e < 2 * a.experts; e += blockDim.x) hist[e] = 0;
  const Tile tile(a, o, cta);
  __syncthreads();
  int lo, hi;
  tile.run(lo, hi);
  const unsigned kth = 0xffffffffu / (unsigned)a.k + 1;  // x / k = the upper half of x * kth, for x < 2^15 and 1 < k <= 2^10
  for (int r = lo; r < hi;) {
    const Stretch t = stretch_at(a, o, r, hi);
    if (t.s >= 0) {
      const int set = tile.set(t.s);
      int size = 0;
      for (int q = r; q < t.end; q += 32) {  // 32 tokens at a time
        const int n = min(32, t.end - q);
        const unsigned ok = __ballot_sync(~0u, lane < n && (!a.valid || a.valid[q + lane]));
        size += __popc(ok);
        const long long first = (long long)q * a.k;
        const int entries = n * a.k;
        for (int i = lane; i < entries; i += 32 * 4) {
          long long e[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) e[u] = i + 32 * u < entries ? load_index(a.index, first + i + 32 * u, a.index_bits) : -1;
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            if (e[u] < 0) continue;
            if (a.valid && !(ok >> (a.k == 1 ? (unsigned)(i + 32 * u) : __umulhi(i + 32 * u, kth)) & 1)) continue;
            if (e[u] >= a.experts)
              atomicOr(&a.bad[t.s], 1);
            else if (set >= 0)
              atomicAdd(&hist[set * a.experts + (int)e[u]], 1);
            else
              atomicAdd(&a.counts[cell(a, t.s, (int)e[u])], 1ull);
          }
        }
      }
      if (lane == 0 && size) atomicAdd(&a.sizes[t.s], (unsigned long long)size);
    }
    r = t.end;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < a.experts; e += blockDim.x) {
    if (tile.first >= 0 && hist[e]) atomicAdd(&a.counts[cell(a, tile.first, e)], (unsigned long long)hist[e]);
    if (tile.last >= 0 && hist[a.experts + e])
      atomicAdd(&a.counts[cell(a, tile.last, e)], (unsigned long long)hist[a.experts + e]);
  }
}

// Logits as they lie in memory, for U tokens per group of lanes
template <typename T, int V, int J, int U>
struct Raw {
  static constexpr int WORDS = V == 1 ? 1 : 4;
  uint32_t w[U][J][WORDS];
  bool ok[U];
  // tokens base + u * per + gi below `end`; what is not there, or not valid, is 0, a column that is not there -inf
  __device__ __forceinline__ void load(const BalanceArgs& a, int base, int end, bool any, int per, int gi, int gl) {
    using E = Elem<T>;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = base + u * per + gi;
      ok[u] = any && r < end && (!a.valid || a.valid[r]);
      const T* row = reinterpret_cast<const T*>(a.logits) + row_at(r, a.inner, a.outer_stride, a.inner_stride);
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int col = (j * a.group + gl) * V;
        const uint32_t fill = ok[u] ? E::none().x : 0u;
#pragma unroll
        for (int i = 0; i < WORDS; ++i) w[u][j][i] = fill;
        if (ok[u] && col < a.experts) {
          if constexpr (V == 1) {
            w[u][j][0] = E::raw(row + col);
          } else {
            const uint4 q = *reinterpret_cast<const uint4*>(row + col);
            w[u][j][0] = q.x, w[u][j][1] = q.y, w[u][j][2] = q.z, w[u][j][3] = q.w;
          }
        }
      }
    }
  }
  __device__ __forceinline__ void unpack(int u, float* x) const {
    using E = Elem<T>;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      if constexpr (V == 1)
        x[j] = E::of_raw(w[u][j][0]);
      else
        E::unpack(make_uint4(w[u][j][0], w[u][j][1], w[u][j][2], w[u][j][3]), x + j * V);
    }
  }
};

// Scores of all tokens: their sums (SUM), the gradient (GRAD).  V: elements per load (16 bytes, or 1 where rows are
// not 16-byte aligned), J: loads per lane; a.group lanes (a power of two) hold a token's logits, U tokens each are under
// way at a time and the next U on their way from memory.  sums: unsigned long long[2, experts] in shared memory, behind them
// float[2, experts]: the counts of the CTA's first and last sequence (read once per CTA: thousands of warps that read the
// same few lines of L2 wait for one another, 10 us at 256 experts)
template <typename T, int V, int J, int U, bool SIG, bool SUM, bool GRAD>
__device__ __forceinline__ void score_phase(const BalanceArgs& a, const Offsets& o, int cta, unsigned long long* sums) {
  using E = Elem<T>;
  constexpr int JV = J * V, N2 = (JV + 1) / 2;  // pairs; an odd last one is filled up with -inf
  const int lane = threadIdx.x & 31;
  const int G = a.group, per = 32 / G, gl = lane & (G - 1), gi = lane / G;
  if (SUM)
    for (int e = threadIdx.x; e < 2 * a.experts; e += blockDim.x) sums[e] = 0;
  const Tile tile(a, o, cta);
  float* counts = reinterpret_cast<float*>(SUM ? sums + 2 * a.experts : sums);
  if (GRAD) {
    if (SUM) pdl_wait();  // the counts
    for (int e = threadIdx.x; e < a.experts; e += blockDim.x) {
      if (tile.first >= 0) counts[e] = count_of(a, tile.first, e);
      if (tile.last >= 0) counts[a.experts + e] = count_of(a, tile.last, e);
    }
  }
  __syncthreads();
  int lo, hi;
  tile.run(lo, hi);
  constexpr float LOG2E = 1.4426950408889634f;
  const float minus_inf = -__int_as_float(0x7f800000), units = __int_as_float((a.shift + 127) << 23);
  const f2 log2e = f2_splat(LOG2E), zero = f2_splat(0.0f);

  for (int r0 = lo; r0 < hi;) {
    Stretch t = stretch_at(a, o, r0, hi);
    if (SUM) t.end = min(t.end, r0 + MAX_RUN);
    const bool any = t.s >= 0;
    Raw<T, V, J, U> next;
    next.load(a, r0, t.end, any, per, gi, gl);
    f2 c[N2], acc[N2];
    float fac = 0.0f;
    const int set = tile.set(t.s);
    if (GRAD && any) fac = a.scale * (SUM ? (float)factor_of(a, t.s) : a.factor[t.s] * a.upstream[t.s]);
#pragma unroll
    for (int n = 0; n < N2; ++n) {
      float v[2] = {0.0f, 0.0f};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int i = 2 * n + h, col = (i / V * G + gl) * V + i % V;
        if (GRAD && any && i < JV && col < a.experts)
          v[h] = set >= 0 ? counts[set * a.experts + col] : count_of(a, t.s, col);
      }
      c[n] = f2_pack(v[0], v[1]);
      acc[n] = zero;
    }
    for (int base = r0; base < t.end; base += per * U) {
      const Raw<T, V, J, U> now = next;
      if (base + per * U < t.end) next.load(a, base + per * U, t.end, any, per, gi, gl);
      f2 p[U][N2];                 // the scores
      f2 slope[SIG ? U : 1][N2];   // 1 - sigmoid
      float m[U], sum[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float x[2 * N2];
        x[2 * N2 - 1] = minus_inf;
        now.unpack(u, x);
        m[u] = x[0];
#pragma unroll
        for (int i = 1; i < JV; ++i) m[u] = fmaxf(m[u], x[i]);
#pragma unroll
        for (int n = 0; n < N2; ++n) p[u][n] = f2_pack(x[2 * n], x[2 * n + 1]);
      }
      for (int d = G >> 1; d; d >>= 1) {
#pragma unroll
        for (int u = 0; u < U; ++u) m[u] = fmaxf(m[u], __shfl_xor_sync(~0u, m[u], d));
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        f2 total = zero;
        if constexpr (SIG) {
          // sigmoid(x) = e^min(x,0) / (1 + e^-|x|), scaled by e^-min(m,0) so that the largest one stays near 1
          const float top = fminf(m[u], 0.0f);
#pragma unroll
          for (int n = 0; n < N2; ++n) {
            float x[2], y[2], z[2];
            f2_unpack(p[u][n], x[0], x[1]);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float v = x[h], fall = ex2(-fabsf(v) * LOG2E), d = rcp_nr(1.0f + fall);
              y[h] = v == v ? ex2((fminf(v, 0.0f) - top) * LOG2E) * d : v;
              z[h] = v >= 0.0f ? fall * d : d;
            }
            p[u][n] = f2_pack(y[0], y[1]);
            slope[u][n] = f2_pack(z[0], z[1]);
            total = f2_add(total, p[u][n]);
          }
        } else {
          const f2 top = f2_splat(-m[u]);
#pragma unroll
          for (int n = 0; n < N2; ++n) {
            float x, y;
            f2_unpack(f2_mul(f2_add(p[u][n], top), log2e), x, y);
            p[u][n] = f2_pack(ex2(x), ex2(y));
            total = f2_add(total, p[u][n]);
          }
        }
        float x, y;
        f2_unpack(total, x, y);
        sum[u] = x + y;
      }
      for (int d = G >> 1; d; d >>= 1) {
#pragma unroll
        for (int u = 0; u < U; ++u) sum[u] += __shfl_xor_sync(~0u, sum[u], d);
      }
      float dot[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const f2 inv = f2_splat(now.ok[u] ? rcp_nr(sum[u]) : 0.0f);  // 0: the logits stand as 0, the scores are 0 from here on
        f2 total = zero;
#pragma unroll
        for (int n = 0; n < N2; ++n) {
          p[u][n] = f2_mul(p[u][n], inv);
          if (SUM) acc[n] = f2_add(acc[n], p[u][n]);
          if (GRAD) total = f2_fma(c[n], p[u][n], total);
        }
        float x, y;
        f2_unpack(total, x, y);
        dot[u] = x + y;
      }
      if (GRAD) {
        for (int d = G >> 1; d; d >>= 1) {
#pragma unroll
          for (int u = 0; u < U; ++u) dot[u] += __shfl_xor_sync(~0u, dot[u], d);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int r = base + u * per + gi;
          const f2 f = f2_splat(now.ok[u] ? fac : 0.0f), less = f2_splat(-dot[u]);
          float y[2 * N2];
#pragma unroll
          for (int n = 0; n < N2; ++n) {
            f2 v = f2_mul(f2_mul(f, p[u][n]), f2_add(c[n], less));
            if (SIG) v = f2_mul(v, slope[SIG ? u : 0][n]);
            f2_unpack(v, y[2 * n], y[2 * n + 1]);
          }
          T* g = reinterpret_cast<T*>(a.grad) + (long long)r * a.experts;
#pragma unroll
          for (int j = 0; j < J; ++j) {
            const int col = (j * G + gl) * V;
            if (r < t.end && col < a.experts) {
              if constexpr (V == 1)
                g[col] = E::narrow(y[j]);
              else
                *reinterpret_cast<uint4*>(g + col) = E::pack(y + j * V);
            }
          }
        }
      }
    }
    if (SUM && any) {
      bool nan = false;
#pragma unroll
      for (int n = 0; n < N2; ++n) {
        float v[2];
        f2_unpack(acc[n], v[0], v[1]);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int i = 2 * n + h, col = (i / V * G + gl) * V + i % V;
          for (int d = G; d < 32; d <<= 1) v[h] += __shfl_xor_sync(~0u, v[h], d);
          if (gi == 0 && i < JV && col < a.experts) {
            nan |= !(v[h] == v[h]);
            const unsigned long long q = (unsigned long long)__float2ll_rn(v[h] * units);
            if (set >= 0)
              atomicAdd(&sums[set * a.experts + col], q);
            else
              atomicAdd(&a.psum[cell(a, t.s, col)], q);
          }
        }
      }
      if (nan) atomicOr(&a.bad[t.s], 2);
    }
    r0 = t.end;
  }
  if (!SUM) return;
  __syncthreads();
  for (int e = threadIdx.x; e < a.experts; e += blockDim.x) {
    if (tile.first >= 0 && sums[e]) atomicAdd(&a.psum[cell(a, tile.first, e)], sums[e]);
    if (tile.last >= 0 && sums[a.experts + e]) atomicAdd(&a.psum[cell(a, tile.last, e)], sums[a.experts + e]);
  }
}

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(~0u, v, d);
  return v;
}

// Loss and factor of the sequences, and the second copy of their counts.  Reads what other CTAs have written; the loads of a
// thread are independent of one another.  A sequence has a warp, or, where there is one sequence only, the CTA (`red`: double[32]).
__device__ __forceinline__ void loss_phase(const BalanceArgs& a, int first, int step, double* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool one = a.sequences == 1;
  for (int s = one ? 0 : first + warp; s < a.sequences; s += step) {
    double sum = 0.0;
    const int from = one ? threadIdx.x : lane, by = one ? blockDim.x : 32;
    for (int e0 = from; e0 < a.experts; e0 += 4 * by) {  // four at a time: their loads first, which a store would hold up
      unsigned long long c[4], p[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int e = e0 + j * by;
        c[j] = e < a.experts ? __ldcg(&a.counts[cell(a, s, e)]) : 0;
        p[j] = e < a.experts ? __ldcg(&a.psum[cell(a, s, e)]) : 0;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        sum += (double)c[j] * (double)p[j];
        if (a.counts_out && e0 + j * by < a.experts) a.counts_out[cell(a, s, e0 + j * by)] = c[j];
      }
    }
    const double f = factor_of(a, s);
    const int nan = __ldcg(&a.bad[s]) & 2;
    sum = warp_sum(sum);
    if (one) {
      if (lane == 0) red[warp] = sum;
      __syncthreads();
      sum = warp_sum(lane < (int)(blockDim.x >> 5) ? red[lane] : 0.0);
      if (warp != 0) return;
    }
    if (lane == 0) {
      a.factor[s] = (float)f;
      a.loss[s] = nan ? nan_f() : (float)(sum * f * __longlong_as_double((1023ll - a.shift) << 52));
    }
  }
}

// 74 CTAs: their histograms meet in atomics on the same few lines of memory, 2 ns each (131072 x 8 int64 indices: 6-8 us)
__global__ void __launch_bounds__(1024) balance_count_kernel(const BalanceArgs a) {
  extern __shared__ unsigned long long shared[];
  __shared__ Offsets offsets;
  pdl_start_next();
  load_offsets(a, offsets);
  count_phase(a, offsets, blockIdx.x, reinterpret_cast<int*>(shared));
}

// Two CTAs per SM, so that four tokens per group of lanes and the next four fit in registers (131072 x 256 bf16, both: 46-50 us;
// three CTAs 55, two tokens 51).  Bound by issue: 190 instructions per warp and token, 64 % of the slots.  With the gradient,
// more than 512 experts spill (80-700 bytes, single loads up to 944; the traffic stays on the chip): 32768 x 1024 bf16 62 us
// a call, 0.33 of the copy rate, fp32 76 us, 0.54; 32768 x 1023 bf16 139 us, 0.15.
template <typename T, int V, int J, bool SIG, bool SUM, bool GRAD>
__global__ void __launch_bounds__(256, 2) balance_score_kernel(const BalanceArgs a) {
  extern __shared__ unsigned long long shared[];
  __shared__ Offsets offsets;
  __shared__ bool last;
  __shared__ double red[32];
  constexpr int U = J * V <= 8 ? (SIG ? 2 : 4) : J * V <= 16 && !SIG ? 2 : 1;
  load_offsets(a, offsets);
  score_phase<T, V, J, U, SIG, SUM, GRAD>(a, offsets, blockIdx.x, shared);
  if (SUM) pdl_wait();  // without the gradient nothing needs the counts but the CTA that adds up
  if (SUM && a.finish) {
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) last = atomicAdd(a.ticket, 1u) == gridDim.x - 1;
    __syncthreads();
    if (last) {
      __threadfence();
      loss_phase(a, 0, blockDim.x >> 5, red);
    }
  }
}

__global__ void __launch_bounds__(256) balance_loss_kernel(const BalanceArgs a) {
  __shared__ double red[32];
  loss_phase(a, blockIdx.x * (blockDim.x >> 5), gridDim.x * (blockDim.x >> 5), red);
}

// Everything in one launch of one cluster (of one CTA, where that is enough).  Bound by latencies: four phases with a barrier
// of the cluster between them, 11-17 us (1024 x 64 bf16: 14 us, 4096 x 64: 16.5 us, as much
// as the three launches take at 16384 x 64).
template <typename T, int V, int J, int U, bool SIG, bool GRAD>
__global__ void __launch_bounds__(MAX_WARPS * 32, 1) balance_small_kernel(const BalanceArgs a) {
  extern __shared__ unsigned long long shared[];
  __shared__ Offsets offsets;
  __shared__ double red[32];
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = gridDim.x, cta = blockIdx.x;
  const auto all = [&] {
    __threadfence();
    if (ctas > 1)
      cluster.sync();
    else
      __syncthreads();
  };
  const long long cells = (long long)a.sequences * a.experts, id = (long long)cta * blockDim.x + threadIdx.x;
  for (long long i = id; i < cells; i += ctas * blockDim.x) a.counts[i] = a.psum[i] = 0;
  for (long long i = id; i <= a.sequences; i += ctas * blockDim.x) {
    if (i < a.sequences) a.sizes[i] = 0;
    a.bad[i] = 0;
  }
  load_offsets(a, offsets);
  all();
  count_phase(a, offsets, cta, reinterpret_cast<int*>(shared));
  all();
  score_phase<T, V, J, U, SIG, true, GRAD>(a, offsets, cta, shared);
  all();
  if (a.sequences > 1 || cta == 0) loss_phase(a, cta * (blockDim.x >> 5), ctas * (blockDim.x >> 5), red);
}

constexpr int BALANCE_CTAS = 2;  // per SM, all at once
constexpr int COUNT_CTAS = 74;   // of 1024 threads: few, for their atomics on the counts follow one another
constexpr int SMALL_CLUSTER = 8;
constexpr int64_t SMALL_WORK = 8192, MEDIUM_WORK = 262144;  // logits for one CTA, for one cluster

// workspace: psum, sizes, bad, ticket
struct BalanceLayout {
  int64_t sizes_at, bad_at, ticket_at, bytes;
};

static BalanceLayout balance_layout(int64_t experts, int64_t sequences) {
  BalanceLayout l;
  l.sizes_at = 8 * sequences * experts;
  l.bad_at = l.sizes_at + 8 * sequences;
  l.ticket_at = l.bad_at + 4 * (sequences + 1);
  l.bytes = (l.ticket_at + 4 + 15) / 16 * 16;
  return l;
}

static int balance_check(const lpmm_b200_balance* b, bool sum, bool grad) {
  if (!b) return LPMM_B200_ERR_NULL_POINTER;
  if (b->tokens < 0 || b->inner < 1 || b->experts < 1 || b->k < 1 || b->sequences < 1) return LPMM_B200_ERR_BAD_SIZE;
  if (b->dtype < 0 || b->dtype > 2) return LPMM_B200_ERR_BAD_KIND;
  if (b->index_bits != 32 && b->index_bits != 64) return LPMM_B200_ERR_BAD_KIND;
  if (b->score != LPMM_B200_SCORE_SOFTMAX && b->score != LPMM_B200_SCORE_SIGMOID) return LPMM_B200_ERR_BAD_KIND;
  if (b->offsets ? b->offset_bits != 32 && b->offset_bits != 64 : b->sequences != 1) return LPMM_B200_ERR_BAD_KIND;
  if (b->experts > LPMM_B200_BALANCE_MAX_EXPERTS || b->k > LPMM_B200_BALANCE_MAX_EXPERTS ||
      b->tokens > LPMM_B200_BALANCE_MAX_TOKENS || b->inner > (1ll << 30) || b->sequences > (1 << 24))
    return LPMM_B200_ERR_TOO_LARGE;
  if (!b->counts || !b->factor) return LPMM_B200_ERR_NULL_POINTER;
  if (b->tokens && (!b->logits || (sum && !b->index) || (grad && !b->grad))) return LPMM_B200_ERR_NULL_POINTER;
  if (sum && (!b->loss || !b->work)) return LPMM_B200_ERR_NULL_POINTER;
  if (!sum && !b->upstream) return LPMM_B200_ERR_NULL_POINTER;
  if (sum && ((uintptr_t)b->work & 7)) return LPMM_B200_ERR_BAD_SIZE;
  return LPMM_B200_OK;
}

template <typename K>
static cudaError_t balance_launch(K kernel, const BalanceArgs& a, int ctas, int threads, size_t smem, int cluster, bool after,
                                  cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas), cfg.blockDim = dim3(threads), cfg.dynamicSmemBytes = smem, cfg.stream = stream;
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

// ctas < 0: everything in one launch of a cluster of -ctas
template <typename T, int V, int J, bool SUM, bool GRAD>
static cudaError_t balance_scores(const BalanceArgs& a, int ctas, cudaStream_t stream) {
  const size_t smem = (SUM ? 16 : 0) * (size_t)a.experts + (GRAD ? 8 : 0) * (size_t)a.experts;
  if constexpr (SUM && J * V <= 8) {
    if (ctas == -1)  // one token at a time: less code to fetch
      return a.sigmoid ? balance_launch(balance_small_kernel<T, V, J, 1, true, GRAD>, a, 1, MAX_WARPS * 32, smem, 1, false, stream)
                       : balance_launch(balance_small_kernel<T, V, J, 1, false, GRAD>, a, 1, MAX_WARPS * 32, smem, 1, false, stream);
    if (ctas < 0)
      return a.sigmoid
                 ? balance_launch(balance_small_kernel<T, V, J, 2, true, GRAD>, a, -ctas, MAX_WARPS * 32, smem, -ctas, false, stream)
                 : balance_launch(balance_small_kernel<T, V, J, 4, false, GRAD>, a, -ctas, MAX_WARPS * 32, smem, -ctas, false, stream);
  }
  return a.sigmoid ? balance_launch(balance_score_kernel<T, V, J, true, SUM, GRAD>, a, ctas, 256, smem, 1, SUM, stream)
                   : balance_launch(balance_score_kernel<T, V, J, false, SUM, GRAD>, a, ctas, 256, smem, 1, SUM, stream);
}

// 16-byte loads where every row (and row of the gradient) begins on a 16-byte boundary
static bool balance_wide(const lpmm_b200_balance* b, bool grad) {
  const int64_t ve = b->dtype == LPMM_B200_DTYPE_FP32 ? 4 : 8;
  return b->experts % ve == 0 && ((uintptr_t)b->logits & 15) == 0 && (!grad || ((uintptr_t)b->grad & 15) == 0) &&
         b->outer_stride % ve == 0 && b->inner_stride % ve == 0;
}
// values per lane
static int balance_per_lane(const lpmm_b200_balance* b, bool wide) {
  const int ve = !wide ? 1 : b->dtype == LPMM_B200_DTYPE_FP32 ? 4 : 8;
  return (int)((b->experts + 32 * ve - 1) / (32 * ve)) * ve;
}

template <typename T, bool SUM, bool GRAD>
static cudaError_t balance_shape(BalanceArgs& a, bool wide, int ctas, cudaStream_t stream) {
  constexpr int VE = Elem<T>::VE;
  const int loads = wide ? a.experts / VE : a.experts;
  a.group = 1;
  while (a.group < loads && a.group < 32) a.group *= 2;
  const int j = (loads + 31) / 32;
  if (wide) {
    if (j <= 1) return balance_scores<T, VE, 1, SUM, GRAD>(a, ctas, stream);
    if (j <= 2) return balance_scores<T, VE, 2, SUM, GRAD>(a, ctas, stream);
    if (j <= 4) return balance_scores<T, VE, 4, SUM, GRAD>(a, ctas, stream);
    if constexpr (VE == 4) return balance_scores<T, VE, 8, SUM, GRAD>(a, ctas, stream);
  }
  if (j <= 1) return balance_scores<T, 1, 1, SUM, GRAD>(a, ctas, stream);
  if (j <= 8) return balance_scores<T, 1, 8, SUM, GRAD>(a, ctas, stream);
  if (j <= 16) return balance_scores<T, 1, 16, SUM, GRAD>(a, ctas, stream);
  return balance_scores<T, 1, 32, SUM, GRAD>(a, ctas, stream);
}

template <bool SUM, bool GRAD>
static int balance_run(const lpmm_b200_balance* b, void* stream_) {
  const int bad = balance_check(b, SUM, GRAD);
  if (bad) return bad;
  cudaStream_t stream = (cudaStream_t)stream_;
  BalanceArgs a = {};
  a.logits = b->logits, a.grad = b->grad, a.index = b->index, a.valid = b->valid, a.offsets = b->offsets;
  a.upstream = b->upstream, a.loss = b->loss, a.factor = b->factor;
  a.counts = reinterpret_cast<unsigned long long*>(b->counts);
  a.counts_out = reinterpret_cast<unsigned long long*>(b->counts_out);
  const BalanceLayout l = balance_layout(b->experts, b->sequences);
  if (SUM) {
    char* work = reinterpret_cast<char*>(b->work);
    a.psum = reinterpret_cast<unsigned long long*>(work);
    a.sizes = reinterpret_cast<unsigned long long*>(work + l.sizes_at);
    a.bad = reinterpret_cast<int*>(work + l.bad_at);
    a.ticket = reinterpret_cast<unsigned*>(work + l.ticket_at);
  }
  a.tokens = (int)b->tokens, a.inner = b->inner, a.outer_stride = b->outer_stride, a.inner_stride = b->inner_stride;
  a.sequences = (int)b->sequences, a.experts = (int)b->experts, a.k = (int)b->k;
  a.index_bits = b->index_bits, a.offset_bits = b->offset_bits;
  a.sigmoid = b->score == LPMM_B200_SCORE_SIGMOID;
  a.scale = b->grad_scale;
  for (a.shift = 61; a.shift > 1 && (b->tokens >> (62 - a.shift)) != 0;) --a.shift;
  const int64_t work_size = b->tokens * b->experts;
  int ctas;
  const bool wide = balance_wide(b, GRAD);
  if (SUM && work_size <= MEDIUM_WORK && b->sequences * b->experts <= 16384 && balance_per_lane(b, wide) <= 8) {
    ctas = work_size <= SMALL_WORK ? -1 : -SMALL_CLUSTER;
    a.tile = (int)((b->tokens - ctas - 1) / -ctas);
  } else {
    // runs of 8 tokens per warp at least
    int64_t n = (b->tokens + 63) / 64;
    if (n > BALANCE_CTAS * num_sms()) n = BALANCE_CTAS * num_sms();
    if (n < 1) n = 1;
    a.tile = (int)((b->tokens + n - 1) / n);
    ctas = a.tile ? (int)((b->tokens + a.tile - 1) / a.tile) : 1;
    a.finish = b->sequences <= 64;
  }
  if (a.tile < 1) a.tile = 1;
  if (SUM && ctas > 0) {
    // counts, psum, sizes, bad, ticket: cleared, in one go where the workspace follows the counts
    const size_t cells = 8 * (size_t)(b->sequences * b->experts);
    if (reinterpret_cast<char*>(b->counts) + cells == reinterpret_cast<char*>(b->work)) {
      LPMM_CUDA_TRY(cudaMemsetAsync(b->counts, 0, cells + l.bytes, stream));
    } else {
      LPMM_CUDA_TRY(cudaMemsetAsync(b->counts, 0, cells, stream));
      LPMM_CUDA_TRY(cudaMemsetAsync(b->work, 0, l.bytes, stream));
    }
    BalanceArgs c = a;
    int n = (int)((b->tokens + 255) / 256);
    if (n > COUNT_CTAS) n = COUNT_CTAS;
    if (n < 1) n = 1;
    c.tile = (int)((b->tokens + n - 1) / n);
    LPMM_CUDA_TRY(balance_launch(balance_count_kernel, c, n, 1024, 8 * (size_t)a.experts, 1, false, stream));
  }
  if (SUM || b->tokens) {
    if (b->dtype == LPMM_B200_DTYPE_FP32)
      LPMM_CUDA_TRY((balance_shape<float, SUM, GRAD>(a, wide, ctas, stream)));
    else if (b->dtype == LPMM_B200_DTYPE_BF16)
      LPMM_CUDA_TRY((balance_shape<__nv_bfloat16, SUM, GRAD>(a, wide, ctas, stream)));
    else
      LPMM_CUDA_TRY((balance_shape<__half, SUM, GRAD>(a, wide, ctas, stream)));
  }
  if (SUM && ctas > 0 && !a.finish) {
    const int64_t n = (b->sequences + 7) / 8;
    balance_loss_kernel<<<(unsigned)(n < 4096 ? n : 4096), 256, 0, stream>>>(a);
    LPMM_CUDA_TRY(cudaGetLastError());
  }
  return LPMM_B200_OK;
}

}  // namespace lpmm_b200

using namespace lpmm_b200;

extern "C" int64_t lpmm_b200_balance_work_bytes(int64_t experts, int64_t sequences) {
  if (experts < 1 || sequences < 1 || experts > LPMM_B200_BALANCE_MAX_EXPERTS || sequences > (1 << 24))
    return LPMM_B200_ERR_BAD_SIZE;
  return balance_layout(experts, sequences).bytes;
}

extern "C" int lpmm_b200_balance_forward(const lpmm_b200_balance* b, void* stream) {
  return balance_run<true, false>(b, stream);
}
extern "C" int lpmm_b200_balance_backward(const lpmm_b200_balance* b, void* stream) {
  return balance_run<false, true>(b, stream);
}
extern "C" int lpmm_b200_balance_forward_backward(const lpmm_b200_balance* b, void* stream) {
  return balance_run<true, true>(b, stream);
}
