// The load-balance loss of a router, the assignments per expert, and the loss's gradient.
//
//   p = softmax(x), or sigmoid(x) / sum sigmoid(x), over a token's experts;  c_e = assignments of the sequence to e
//   loss = F sum_e c_e sum_n p_ne,   d loss / d x_ne = F p_ne (c_e - sum_j c_j p_nj) [(1 - sigmoid(x_ne))],
//   F = experts / (k n^2), n = valid tokens of the sequence
//
// The gradient needs the counts, not the summed scores, so loss and gradient share one pass over the logits once the
// indices are counted.  A token's logits lie in the registers of 2 ... 32 lanes; a warp walks a contiguous run of
// tokens and sums the scores of its columns in registers.  Sums meet in a fixed order: groups of a warp by shuffles,
// warps of a CTA in shared memory, CTAs in the last kernel; a sequence that ends inside a run is written out there.
// Bound by memory for large batches (a logit is read once, a gradient written once), by launches for small ones.
#include "loss_common.cuh"

namespace lpmm_b200 {

constexpr int WARPS = 8;

struct BalanceArgs {
  const void* logits;
  void* grad;
  const void* index;
  const uint8_t* valid;
  const void* offsets;
  const float* upstream;
  float* loss;
  unsigned long long* counts;
  float* factor;
  unsigned long long* sizes;  // valid tokens per sequence
  int* bad;                   // per sequence: an index out of range; [sequences]: the offsets are not in order
  float* psum;                // [sequences, experts]: sequences that lie within one CTA's tokens
  float* partial;             // [CTAs, 2, experts]: the sequence that a CTA's first / last tokens share with others
  long long tokens, inner, outer_stride, inner_stride, sequences, tile;
  int experts, k, index_bits, offset_bits, sigmoid, group;
  float scale;
};

__device__ __forceinline__ long long raw_offset(const BalanceArgs& a, long long i) {
  if (!a.offsets) return i == 0 ? 0 : a.tokens;
  return load_index(a.offsets, i, a.offset_bits);
}
__device__ __forceinline__ long long offset_at(const BalanceArgs& a, long long i) {
  return min(max(raw_offset(a, i), 0ll), a.tokens);
}

// The stretch of tokens from r on that belongs to one sequence: s in [0, sequences), or s < 0 for tokens of none.
// Whatever the offsets hold, r < end <= hi and s is in range.
struct Stretch {
  long long s, end;
};
__device__ __forceinline__ Stretch stretch_at(const BalanceArgs& a, long long r, long long hi) {
  if (!a.offsets) return Stretch{0, hi};
  long long lo = -1, up = a.sequences + 1;  // offset(lo) <= r < offset(up)
  while (up - lo > 1) {
    const long long mid = (lo + up) >> 1;
    if (offset_at(a, mid) <= r)
      lo = mid;
    else
      up = mid;
  }
  Stretch t;
  t.s = lo == a.sequences ? -1 : lo;
  t.end = lo == a.sequences ? hi : max(min(offset_at(a, lo + 1), hi), r + 1);
  return t;
}

__device__ __forceinline__ double factor_of(const BalanceArgs& a, long long s) {
  if (a.bad[s] || a.bad[a.sequences]) return (double)nan_f();
  const double n = (double)a.sizes[s];
  return n == 0.0 ? 0.0 : (double)a.experts / ((double)a.k * n * n);
}

// Assignments per expert and valid tokens per sequence.  One sequence: a histogram per CTA in shared memory; several:
// a warp counts its run of tokens straight into the sequence's row.
__global__ void __launch_bounds__(WARPS * 32) balance_count_kernel(const BalanceArgs a) {
  extern __shared__ int hist[];
  const bool one = a.sequences == 1;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (blockIdx.x == 0 && a.offsets) {
    bool off = false;
    for (long long i = threadIdx.x; i <= a.sequences; i += blockDim.x) {
      const long long o = raw_offset(a, i);
      off |= o < 0 || o > a.tokens || (i && raw_offset(a, i - 1) > o);
    }
    if (off) a.bad[a.sequences] = 1;
  }
  if (one) {
    for (int e = threadIdx.x; e < a.experts; e += blockDim.x) hist[e] = 0;
    __syncthreads();
  }
  const long long tile_lo = blockIdx.x * a.tile, tile_hi = min(tile_lo + a.tile, a.tokens);
  const long long run = (a.tile + WARPS - 1) / WARPS;
  const long long lo = tile_lo + warp * run, hi = min(lo + run, tile_hi);
  for (long long r = lo; r < hi;) {
    const Stretch t = stretch_at(a, r, hi);
    if (t.s >= 0) {
      int size = 0;
      for (long long q = r + lane; q < t.end; q += 32) size += !a.valid || a.valid[q];
      size = __reduce_add_sync(~0u, size);
      if (lane == 0 && size) atomicAdd(&a.sizes[t.s], (unsigned long long)size);
      for (long long q = r * a.k + lane; q < t.end * a.k; q += 32) {
        if (a.valid && !a.valid[q / a.k]) continue;
        const long long e = load_index(a.index, q, a.index_bits);
        if (e < 0) continue;
        if (e >= a.experts)
          a.bad[t.s] = 1;
        else if (one)
          atomicAdd(&hist[e], 1);
        else
          atomicAdd(&a.counts[t.s * a.experts + e], 1ull);
      }
    }
    r = t.end;
  }
  if (one) {
    __syncthreads();
    for (int e = threadIdx.x; e < a.experts; e += blockDim.x)
      if (hist[e]) atomicAdd(&a.counts[e], (unsigned long long)hist[e]);
  }
}

// Scores of all tokens: their sums (SUM), the gradient (GRAD).  V: elements per load (16 bytes, or 1 where rows are
// not 16-byte aligned), J: loads per lane; a.group lanes (a power of two) hold a token's logits.
template <typename T, int V, int J, bool SUM, bool GRAD>
__global__ void __launch_bounds__(WARPS * 32) balance_kernel(const BalanceArgs a) {
  using E = Elem<T>;
  extern __shared__ float slots[];  // [WARPS, 2, experts]
  __shared__ long long owner[WARPS][2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int G = a.group, per = 32 / G, gl = lane & (G - 1), gi = lane / G;
  const long long tile_lo = blockIdx.x * a.tile, tile_hi = min(tile_lo + a.tile, a.tokens);
  const long long run = (a.tile + WARPS - 1) / WARPS;
  const long long lo = tile_lo + warp * run, hi = min(lo + run, tile_hi);
  if (SUM && threadIdx.x < WARPS * 2) owner[threadIdx.x >> 1][threadIdx.x & 1] = -1;
  if (SUM) __syncthreads();
  constexpr float LOG2E = 1.4426950408889634f;
  const float minus_inf = -__int_as_float(0x7f800000);

  for (long long r0 = lo; r0 < hi;) {
    const Stretch t = stretch_at(a, r0, hi);
    float c[J * V], acc[J * V], fac = 0.0f;
    if (GRAD) {
      if (t.s >= 0) {
        fac = a.scale * (SUM ? (float)factor_of(a, t.s) : a.factor[t.s] * a.upstream[t.s]);
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const int col = (j * G + gl) * V + i;
            c[j * V + i] = col < a.experts ? (float)a.counts[t.s * a.experts + col] : 0.0f;
          }
      }
    }
#pragma unroll
    for (int i = 0; i < J * V; ++i) acc[i] = 0.0f;
    for (long long base = r0; base < t.end; base += per) {
      const long long r = base + gi;
      const bool here = r < t.end, ok = here && t.s >= 0 && (!a.valid || a.valid[r]);
      float x[J * V];
      const T* row = reinterpret_cast<const T*>(a.logits) + (r / a.inner) * a.outer_stride + (r % a.inner) * a.inner_stride;
      float m = minus_inf;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int col = (j * G + gl) * V;
        if (ok && col < a.experts) {
          if (V == 1)
            x[j] = E::widen(row[col]);
          else
            E::unpack(*reinterpret_cast<const uint4*>(row + col), x + j * V);
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) x[j * V + i] = ok ? minus_inf : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < V; ++i) m = fmaxf(m, x[j * V + i]);
      }
      for (int d = G >> 1; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, d));
      // p holds the score, x (sigmoid only) 1 - sigmoid
      float p[J * V], sum = 0.0f;
#pragma unroll
      for (int i = 0; i < J * V; ++i) {
        if (a.sigmoid) {
          // sigmoid(x) = e^min(x,0) / (1 + e^-|x|), scaled by e^-min(m,0) so that the largest one stays near 1
          const float fall = ex2(-fabsf(x[i]) * LOG2E), d = __frcp_rn(1.0f + fall);
          p[i] = ex2((fminf(x[i], 0.0f) - fminf(m, 0.0f)) * LOG2E) * d;
          if (!(x[i] == x[i])) p[i] = x[i];
          x[i] = x[i] >= 0.0f ? fall * d : d;
        } else {
          p[i] = ex2((x[i] - m) * LOG2E);
        }
        sum += p[i];
      }
      for (int d = G >> 1; d; d >>= 1) sum += __shfl_xor_sync(~0u, sum, d);
      const float inv = __frcp_rn(sum);
      float dot = 0.0f;
#pragma unroll
      for (int i = 0; i < J * V; ++i) {
        p[i] *= inv;
        if (SUM) acc[i] += ok ? p[i] : 0.0f;
        if (GRAD) dot = fmaf(c[i], p[i], dot);
      }
      if (GRAD) {
        for (int d = G >> 1; d; d >>= 1) dot += __shfl_xor_sync(~0u, dot, d);
        T* g = reinterpret_cast<T*>(a.grad) + r * a.experts;
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const int col = (j * G + gl) * V;
          if (here && col < a.experts) {
            float y[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
              float v = fac * p[j * V + i] * (c[j * V + i] - dot);
              if (a.sigmoid) v *= x[j * V + i];
              y[i] = ok ? v : 0.0f;
            }
            if (V == 1)
              g[col] = E::narrow(y[0]);
            else
              *reinterpret_cast<uint4*>(g + col) = E::pack(y);
          }
        }
      }
    }
    if (SUM && t.s >= 0) {
      const long long first = offset_at(a, t.s), last = offset_at(a, t.s + 1);
      const bool whole = first >= lo && last <= hi;  // the sequence lies within this warp's run
      const int slot = first <= lo ? 0 : 1;
      float* to = whole ? a.psum + t.s * a.experts : slots + (warp * 2 + slot) * a.experts;
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float v = acc[j * V + i];
          for (int d = G; d < 32; d <<= 1) v += __shfl_xor_sync(~0u, v, d);
          const int col = (j * G + gl) * V + i;
          if (gi == 0 && col < a.experts) to[col] = v;
        }
      if (!whole && lane == 0) owner[warp][slot] = t.s;
    }
    r0 = t.end;
  }
  if (!SUM) return;
  __syncthreads();
  // the warps' first and last stretches, in order
  for (int e = threadIdx.x; e < a.experts; e += blockDim.x) {
    long long s = -1;
    float v = 0.0f;
    for (int i = 0; i <= WARPS * 2; ++i) {
      const long long o = i < WARPS * 2 ? owner[i >> 1][i & 1] : -1;
      if (i < WARPS * 2 && o < 0) continue;
      if (o != s || i == WARPS * 2) {
        if (s >= 0) {
          const long long first = offset_at(a, s), last = offset_at(a, s + 1);
          if (first >= tile_lo && last <= tile_hi)
            a.psum[s * a.experts + e] = v;
          else
            a.partial[((long long)blockIdx.x * 2 + (first <= tile_lo ? 0 : 1)) * a.experts + e] = v;
        }
        s = o;
        v = 0.0f;
      }
      if (i < WARPS * 2) v += slots[i * a.experts + e];
    }
  }
}

// One CTA per sequence: the score sums of the CTAs that shared it, the loss and the gradient's factor.
__global__ void __launch_bounds__(256) balance_loss_kernel(const BalanceArgs a) {
  __shared__ float part[256];
  __shared__ double red[8];
  const long long s = blockIdx.x;
  const double f = factor_of(a, s);
  const long long first = offset_at(a, s), last = offset_at(a, s + 1);
  double sum = 0.0;
  if (f != 0.0 && f == f) {  // uniform
    const long long t0 = first / a.tile, t1 = (last - 1) / a.tile;
    int cols = 32;
    while (cols < a.experts && cols < 256) cols *= 2;
    const int ny = 256 / cols, y = threadIdx.x / cols, cx = threadIdx.x % cols;
    for (int e0 = 0; e0 < a.experts; e0 += cols) {
      const int e = e0 + cx;
      float v = 0.0f;
      if (e < a.experts) {
        if (t0 == t1) {
          if (y == 0) v = a.psum[s * a.experts + e];
        } else {
          for (long long t = t0 + y; t <= t1; t += ny)
            v += a.partial[(t * 2 + (first <= t * a.tile ? 0 : 1)) * a.experts + e];
        }
      }
      part[threadIdx.x] = v;
      __syncthreads();
      if (y == 0 && e < a.experts) {
        for (int i = 1; i < ny; ++i) v += part[i * cols + cx];
        sum += (double)a.counts[s * a.experts + e] * (double)v;
      }
      __syncthreads();
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    sum = 0.0;
    for (int i = 0; i < 8; ++i) sum += red[i];
    a.loss[s] = (float)(sum * f);
    a.factor[s] = (float)f;
  }
}

// workspace: sizes, bad (cleared before each call), psum, partial; 16-byte aligned parts
struct BalanceLayout {
  int64_t ctas, tile, bad_at, psum_at, partial_at, bytes;
};

static BalanceLayout balance_layout(int64_t tokens, int64_t experts, int64_t sequences) {
  BalanceLayout l;
  int64_t ctas = (tokens + 4 * WARPS - 1) / (4 * WARPS);
  const int64_t most = 2 * 148;
  if (ctas > most) ctas = most;
  if (ctas < 1) ctas = 1;
  l.tile = (tokens + ctas - 1) / ctas;
  if (l.tile < 1) l.tile = 1;
  l.ctas = (tokens + l.tile - 1) / l.tile;
  if (l.ctas < 1) l.ctas = 1;
  auto up = [](int64_t v) { return (v + 15) / 16 * 16; };
  l.bad_at = up(8 * sequences);
  l.psum_at = l.bad_at + up(4 * (sequences + 1));
  l.partial_at = l.psum_at + up(4 * sequences * experts);
  l.bytes = l.partial_at + 4 * l.ctas * 2 * experts;
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
      b->tokens > (1ll << 40) || b->sequences >= (1ll << 31) - 1)
    return LPMM_B200_ERR_TOO_LARGE;
  if (!b->counts || !b->factor) return LPMM_B200_ERR_NULL_POINTER;
  if (b->tokens && (!b->logits || (sum && !b->index) || (grad && !b->grad))) return LPMM_B200_ERR_NULL_POINTER;
  if (sum && (!b->loss || !b->work)) return LPMM_B200_ERR_NULL_POINTER;
  if (!sum && !b->upstream) return LPMM_B200_ERR_NULL_POINTER;
  if (sum && ((uintptr_t)b->work & 15)) return LPMM_B200_ERR_BAD_SIZE;
  return LPMM_B200_OK;
}

template <typename T, int V, int J, bool SUM, bool GRAD>
static cudaError_t balance_launch(const BalanceArgs& a, int64_t ctas, cudaStream_t stream) {
  const size_t smem = SUM ? sizeof(float) * WARPS * 2 * a.experts : 0;
  if (smem > 40 * 1024) {
    cudaError_t e = cudaFuncSetAttribute(balance_kernel<T, V, J, SUM, GRAD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)smem);
    if (e != cudaSuccess) return e;
  }
  balance_kernel<T, V, J, SUM, GRAD><<<(unsigned)ctas, WARPS * 32, smem, stream>>>(a);
  return cudaGetLastError();
}

template <typename T, bool SUM, bool GRAD>
static cudaError_t balance_shape(BalanceArgs& a, int64_t ctas, cudaStream_t stream) {
  constexpr int VE = Elem<T>::VE;
  // 16-byte loads where every row (and row of the gradient) begins on a 16-byte boundary
  const bool wide = a.experts % VE == 0 && ((uintptr_t)a.logits & 15) == 0 && (!GRAD || ((uintptr_t)a.grad & 15) == 0) &&
                    a.outer_stride % VE == 0 && a.inner_stride % VE == 0;
  const int loads = wide ? a.experts / VE : a.experts;
  a.group = 1;
  while (a.group < loads && a.group < 32) a.group *= 2;
  const int j = (loads + 31) / 32;
  if (wide) {
    if (j <= 1) return balance_launch<T, VE, 1, SUM, GRAD>(a, ctas, stream);
    if (j <= 2) return balance_launch<T, VE, 2, SUM, GRAD>(a, ctas, stream);
    if (j <= 4) return balance_launch<T, VE, 4, SUM, GRAD>(a, ctas, stream);
    return balance_launch<T, VE, 8, SUM, GRAD>(a, ctas, stream);
  }
  if (j <= 1) return balance_launch<T, 1, 1, SUM, GRAD>(a, ctas, stream);
  if (j <= 4) return balance_launch<T, 1, 4, SUM, GRAD>(a, ctas, stream);
  if (j <= 16) return balance_launch<T, 1, 16, SUM, GRAD>(a, ctas, stream);
  return balance_launch<T, 1, 32, SUM, GRAD>(a, ctas, stream);
}

template <bool SUM, bool GRAD>
static int balance_run(const lpmm_b200_balance* b, void* stream_) {
  const int bad = balance_check(b, SUM, GRAD);
  if (bad) return bad;
  cudaStream_t stream = (cudaStream_t)stream_;
  const BalanceLayout l = balance_layout(b->tokens, b->experts, b->sequences);
  char* work = reinterpret_cast<char*>(b->work);
  BalanceArgs a = {};
  a.logits = b->logits, a.grad = b->grad, a.index = b->index, a.valid = b->valid, a.offsets = b->offsets;
  a.upstream = b->upstream, a.loss = b->loss, a.factor = b->factor;
  a.counts = reinterpret_cast<unsigned long long*>(b->counts);
  if (SUM) {
    a.sizes = reinterpret_cast<unsigned long long*>(work);
    a.bad = reinterpret_cast<int*>(work + l.bad_at);
    a.psum = reinterpret_cast<float*>(work + l.psum_at);
    a.partial = reinterpret_cast<float*>(work + l.partial_at);
  }
  a.tokens = b->tokens, a.inner = b->inner, a.outer_stride = b->outer_stride, a.inner_stride = b->inner_stride;
  a.sequences = b->sequences, a.tile = l.tile;
  a.experts = (int)b->experts, a.k = (int)b->k, a.index_bits = b->index_bits, a.offset_bits = b->offset_bits;
  a.sigmoid = b->score == LPMM_B200_SCORE_SIGMOID;
  a.scale = b->grad_scale;
  if (SUM) {
    LPMM_CUDA_TRY(cudaMemsetAsync(b->counts, 0, sizeof(int64_t) * b->sequences * b->experts, stream));
    LPMM_CUDA_TRY(cudaMemsetAsync(work, 0, l.psum_at, stream));
    balance_count_kernel<<<(unsigned)l.ctas, WARPS * 32, b->sequences == 1 ? sizeof(int) * b->experts : 0, stream>>>(a);
    LPMM_CUDA_TRY(cudaGetLastError());
  }
  if (b->tokens) {
    if (b->dtype == LPMM_B200_DTYPE_FP32)
      LPMM_CUDA_TRY((balance_shape<float, SUM, GRAD>(a, l.ctas, stream)));
    else if (b->dtype == LPMM_B200_DTYPE_BF16)
      LPMM_CUDA_TRY((balance_shape<__nv_bfloat16, SUM, GRAD>(a, l.ctas, stream)));
    else
      LPMM_CUDA_TRY((balance_shape<__half, SUM, GRAD>(a, l.ctas, stream)));
  }
  if (SUM) {
    balance_loss_kernel<<<(unsigned)b->sequences, 256, 0, stream>>>(a);
    LPMM_CUDA_TRY(cudaGetLastError());
  }
  return LPMM_B200_OK;
}

}  // namespace lpmm_b200

using namespace lpmm_b200;

extern "C" int64_t lpmm_b200_balance_work_bytes(int64_t tokens, int64_t experts, int64_t sequences) {
  if (tokens < 0 || experts < 1 || sequences < 1 || tokens > (1ll << 40) || experts > LPMM_B200_BALANCE_MAX_EXPERTS ||
      sequences >= (1ll << 31) - 1)
    return LPMM_B200_ERR_BAD_SIZE;
  return balance_layout(tokens, experts, sequences).bytes;
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
