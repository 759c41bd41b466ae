// K8 answers as log-probabilities: per row of logits x the log-probability of given labels, the entropy and the k most
// likely classes.
//
//   m = max x_j     s = sum e^(x_j - m)     t = sum e^(x_j - m) (x_j - m)
//   logp(j) = x_j - m - log s               entropy = log s - t / s
//
// One pass: a lane keeps (m, s, t) of the elements it has seen and rescales s and t when its maximum grows, so a logit
// is read once and memory bounds the kernel. The differences x - m are taken before the change to base 2: masks of the
// type's lowest value stay finite, and -inf gives e = 0.
//
// The k best come out of the same pass. A lane also keeps its best chunk (8 consecutive logits; the first one with the
// lane's maximum). The k-th largest of the lanes' (maximum, chunk) pairs bounds the k-th best logit from below, so only
// the k lanes at or above it hold candidates: their chunks are read again (from cache), what reaches the bound is put
// into LDS, and each candidate's rank is the number of candidates before it. Ties go to the lower class. If more
// candidates come than LDS has room for (their order on the row is adverse), k rounds over the row find one each.
//
// A row of few, long rows is split over `splits` workgroups, whose (m, s, t) and k best are joined by a second launch.
#include "mx.h"

namespace {

constexpr int T = 256, WAVES = T / 64, KMAX = 64, CAP = 1024, SPLITS_MAX = 64;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LOWEST = -3.402823466e38f;
constexpr float FAR = -200.f;  // e^FAR is 0 in 32 bits; keeps 0 * (x - m) from being 0 * -inf

struct Stat {
  float m, s, t;
};

__device__ __forceinline__ float exp_(float d) { return __builtin_amdgcn_exp2f(d * LOG2E); }

// both parts' sums, relative to the larger maximum
__device__ __forceinline__ Stat join(const Stat& a, const Stat& b) {
  const float m = fmaxf(a.m, b.m);
  const float da = a.m - m, db = b.m - m, fa = exp_(da), fb = exp_(db);
  return {m, a.s * fa + b.s * fb, fa * (a.t + fmaxf(da, FAR) * a.s) + fb * (b.t + fmaxf(db, FAR) * b.s)};
}

__device__ __forceinline__ Stat wave_join(Stat v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const Stat w = {__shfl_xor(v.m, o, 64), __shfl_xor(v.s, o, 64), __shfl_xor(v.t, o, 64)};
    v = join(v, w);
  }
  return v;
}

// larger value first, then the lower class
__device__ __forceinline__ bool before(float a, int ia, float b, int ib) { return a > b || (a == b && ia < ib); }

// floats (no NaN) in the order of unsigned integers; -0 as 0
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t b = __float_as_uint(v + 0.f);
  return b ^ (static_cast<uint32_t>(static_cast<int>(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t o) {
  return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}

template <int DT>
__device__ __forceinline__ void load_chunk(const typename mx_elem<DT>::type* x, int c, int n, float (&f)[8]) {
  if (c + 8 <= n)
    mx_floats<DT>(mx_load8<DT>(x + c), f);
  else
    mx_load8_tail<DT>(x + c, n - c, -INFINITY, f);
}

struct Shared {
  Stat stat[WAVES];
  uint32_t key[T];     // each lane's maximum (ordered; 0: it has seen nothing over -inf) and chunk
  int chunk[T];
  uint32_t bound;      // the k-th largest of the keys, and among equal ones the last chunk that counts
  int bound_chunk;
  int lanes[KMAX];     // lanes at or over the bound
  int n_lanes, n_cand;
  float value[CAP];
  int index[CAP];
  float round_value[WAVES];
  int round_index[WAVES];
};

// the k-th largest (key, lower chunk first) of the T lanes, by the first wave: the key bit by bit, then the chunk
__device__ __forceinline__ void find_bound(Shared& sh, int k) {
  const int lane = threadIdx.x;
  uint32_t key[WAVES];
  int chunk[WAVES];
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    key[w] = sh.key[lane + 64 * w];
    chunk[w] = sh.chunk[lane + 64 * w];
  }
  uint32_t bound = 0;
  for (int b = 31; b >= 0; --b) {
    const uint32_t c = bound | (1u << b);
    int n = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) n += __popcll(__ballot(key[w] >= c));
    if (n >= k) bound = c;
  }
  int last = 0x7fffffff;
  if (bound) {
    int over = 0, equal = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      over += __popcll(__ballot(key[w] > bound));
      equal += __popcll(__ballot(key[w] == bound));
    }
    if (over + equal > k) {  // the smallest `last` with k - over equal keys at or before it
      last = 0;
      for (int b = 30; b >= 0; --b) {
        const int c = last + (1 << b);  // with fewer than k - over before c, the answer is c or later
        int n = 0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) n += __popcll(__ballot(key[w] == bound && chunk[w] < c));
        if (n < k - over) last = c;
      }
    }
  }
  if (lane == 0) {
    sh.bound = bound;
    sh.bound_chunk = last;
  }
}

// (m, s, t) of x[0, n), and its k best in sh.value / sh.index [0, k) in order, index -1 where there are no more; classes
// are counted from `first`. Every thread returns the same Stat.
template <int DT>
__device__ Stat row_part(const typename mx_elem<DT>::type* __restrict__ x, int n, int first, int k, Shared& sh) {
  const int tid = threadIdx.x, chunks = (n + 7) / 8;
  Stat st = {LOWEST, 0.f, 0.f};
  float best = -INFINITY;
  int best_chunk = 0;
  for (int c = tid; c < chunks; c += T) {
    float f[8];
    load_chunk<DT>(x, c * 8, n, f);
    float cm = f[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) cm = fmaxf(cm, f[i]);
    best_chunk = cm > best ? c : best_chunk;
    best = fmaxf(best, cm);
    const float m = fmaxf(st.m, best), d = st.m - m, r = exp_(d);
    st.t = r * (st.t + fmaxf(d, FAR) * st.s);
    st.s *= r;
    st.m = m;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float u = f[i] - m, e = exp_(u);
      st.s += e;
      st.t = fmaf(e, fmaxf(u, FAR), st.t);
    }
  }
  const Stat w = wave_join(st);
  if ((tid & 63) == 0) sh.stat[tid >> 6] = w;
  sh.key[tid] = best > -INFINITY ? ordered(best) : 0;
  sh.chunk[tid] = best_chunk;
  if (tid == 0) sh.n_lanes = sh.n_cand = 0;
  __syncthreads();
  Stat all = sh.stat[0];
#pragma unroll
  for (int i = 1; i < WAVES; ++i) all = join(all, sh.stat[i]);
  if (k == 0) return all;

  if (tid < 64) find_bound(sh, k);
  __syncthreads();
  const uint32_t bound = sh.bound;
  const int bound_chunk = sh.bound_chunk;
  {
    const uint32_t key = sh.key[tid];
    if (key && (key > bound || (key == bound && best_chunk <= bound_chunk))) sh.lanes[atomicAdd(&sh.n_lanes, 1)] = tid;
  }
  __syncthreads();
  const int per_lane = (chunks + T - 1) / T, items = sh.n_lanes * per_lane;
  const float least = bound ? unordered(bound) : -INFINITY;
  for (int it = tid; it < items; it += T) {
    const int j = it / per_lane, c = sh.lanes[j] + (it - j * per_lane) * T;
    if (c >= chunks) continue;
    float f[8];
    load_chunk<DT>(x, c * 8, n, f);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (f[i] > least || (f[i] == least && bound && c <= bound_chunk)) {
        const int at = atomicAdd(&sh.n_cand, 1);
        if (at < CAP) {
          sh.value[at] = f[i];
          sh.index[at] = first + c * 8 + i;
        }
      }
  }
  __syncthreads();
  const int cand = sh.n_cand;
  if (cand <= CAP) {
    float v[CAP / T];
    int id[CAP / T], rank[CAP / T];
#pragma unroll
    for (int q = 0; q < CAP / T; ++q) {
      const int a = tid + q * T;
      v[q] = a < cand ? sh.value[a] : 0.f;
      id[q] = a < cand ? sh.index[a] : 0;
      rank[q] = a < cand ? 0 : KMAX;
    }
    for (int b = 0; b < cand; ++b) {
      const float bv = sh.value[b];
      const int bi = sh.index[b];
#pragma unroll
      for (int q = 0; q < CAP / T; ++q) rank[q] += before(bv, bi, v[q], id[q]);
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < CAP / T; ++q)
      if (rank[q] < k) {
        sh.value[rank[q]] = v[q];
        sh.index[rank[q]] = id[q];
      }
    if (tid >= cand && tid < k) {
      sh.value[tid] = -INFINITY;
      sh.index[tid] = -1;
    }
  } else {
    float pv = INFINITY;  // the class that the last round found
    int pi = -1;
    for (int r = 0; r < k; ++r) {
      float bv = -INFINITY;
      int bi = 0x7fffffff;
      for (int c = tid; c < chunks; c += T) {
        float f[8];
        load_chunk<DT>(x, c * 8, n, f);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int id = first + c * 8 + i;
          if (f[i] > -INFINITY && before(pv, pi, f[i], id) && before(f[i], id, bv, bi)) {
            bv = f[i];
            bi = id;
          }
        }
      }
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) {
        const float ov = __shfl_xor(bv, o, 64);
        const int oi = __shfl_xor(bi, o, 64);
        if (before(ov, oi, bv, bi)) {
          bv = ov;
          bi = oi;
        }
      }
      __syncthreads();  // the last round's (or the candidates') slots have been read
      if ((tid & 63) == 0) {
        sh.round_value[tid >> 6] = bv;
        sh.round_index[tid >> 6] = bi;
      }
      __syncthreads();
      pv = sh.round_value[0];
      pi = sh.round_index[0];
#pragma unroll
      for (int w2 = 1; w2 < WAVES; ++w2)
        if (before(sh.round_value[w2], sh.round_index[w2], pv, pi)) {
          pv = sh.round_value[w2];
          pi = sh.round_index[w2];
        }
      if (tid == 0) {
        sh.value[r] = pv;
        sh.index[r] = pi;
      }
    }
  }
  __syncthreads();
  return all;
}

struct Out {
  float* logp;
  float* entropy;
  int* top_idx;
  float* top_logp;
};

// what a row answers. No finite logit: nothing is possible (log-probabilities -inf, entropy 0). A NaN or +inf among
// them: no distribution (NaN, classes -1).
template <int DT, typename L>
__device__ __forceinline__ void answer(const Stat& st, const typename mx_elem<DT>::type* x, int c, const L* labels,
                                       int n_labels, long row, int k, const float* value, const int* index,
                                       const Out& out) {
  const float log_s = logf(st.s);
  const bool none = st.s == 0.f, bad = !(st.s < INFINITY);
  const float nan = __uint_as_float(0x7fc00000u);
  const int tid = threadIdx.x;
  if (tid == 0) out.entropy[row] = none ? 0.f : bad ? nan : log_s - st.t / st.s;
  for (int j = tid; j < n_labels; j += T) {
    const long l = static_cast<long>(labels[row * n_labels + j]);
    float v;
    if (l < 0)
      v = 0.f;  // no label
    else if (l >= c || bad)
      v = nan;
    else
      v = none ? -INFINITY : (mx_elem<DT>::one(x[l]) - st.m) - log_s;
    out.logp[row * n_labels + j] = v;
  }
  for (int r = tid; r < k; r += T) {
    out.top_idx[row * k + r] = bad ? -1 : index[r];
    out.top_logp[row * k + r] = bad ? nan : index[r] < 0 ? -INFINITY : (value[r] - st.m) - log_s;
  }
}

template <int DT, typename L>
__global__ __launch_bounds__(T) void logprobs_kernel(const typename mx_elem<DT>::type* __restrict__ x, long ld, long rows,
                                                     int c, const L* __restrict__ labels, int n_labels, int k, Out out) {
  __shared__ Shared sh;
  for (long row = blockIdx.x; row < rows; row += gridDim.x) {
    const auto* xr = x + row * ld;
    const Stat st = row_part<DT>(xr, c, 0, k, sh);
    answer<DT, L>(st, xr, c, labels, n_labels, row, k, sh.value, sh.index, out);
    __syncthreads();  // the next row writes the shared parts
  }
}

// part p of a row: classes [p * len, (p + 1) * len); ws holds Stat [rows, splits], then k values and k classes of each
template <int DT>
__global__ __launch_bounds__(T) void logprobs_part_kernel(const typename mx_elem<DT>::type* __restrict__ x, long ld,
                                                          int c, int splits, int len, int k, float* __restrict__ ws,
                                                          float* __restrict__ wv, int* __restrict__ wi) {
  __shared__ Shared sh;
  const int row = blockIdx.x / splits, p = blockIdx.x - row * splits;
  const int c0 = p * len, n = min(len, c - c0);
  const Stat st = row_part<DT>(x + row * ld + c0, n, c0, k, sh);
  if (threadIdx.x == 0) {
    ws[blockIdx.x * 3] = st.m;
    ws[blockIdx.x * 3 + 1] = st.s;
    ws[blockIdx.x * 3 + 2] = st.t;
  }
  if (static_cast<int>(threadIdx.x) < k) {
    wv[blockIdx.x * k + threadIdx.x] = sh.value[threadIdx.x];
    wi[blockIdx.x * k + threadIdx.x] = sh.index[threadIdx.x];
  }
}

template <int DT, typename L>
__global__ __launch_bounds__(T) void logprobs_join_kernel(const typename mx_elem<DT>::type* __restrict__ x, long ld,
                                                          int c, const L* __restrict__ labels, int n_labels, int splits,
                                                          int k, const float* __restrict__ ws,
                                                          const float* __restrict__ wv, const int* __restrict__ wi,
                                                          Out out) {
  __shared__ float value[SPLITS_MAX * KMAX];
  __shared__ int index[SPLITS_MAX * KMAX];
  __shared__ float top_value[KMAX];
  __shared__ int top_index[KMAX];
  const int row = blockIdx.x, tid = threadIdx.x, n = splits * k;
  const float* w = ws + static_cast<long>(row) * splits * 3;
  Stat st = {w[0], w[1], w[2]};
  for (int p = 1; p < splits; ++p) st = join(st, {w[p * 3], w[p * 3 + 1], w[p * 3 + 2]});
  for (int a = tid; a < n; a += T) {
    value[a] = wv[static_cast<long>(row) * n + a];
    index[a] = wi[static_cast<long>(row) * n + a];
  }
  if (tid < k) {
    top_value[tid] = -INFINITY;
    top_index[tid] = -1;
  }
  __syncthreads();
  for (int a = tid; a < n; a += T) {
    const float v = value[a];
    const int id = index[a];
    if (id < 0) continue;
    int rank = 0;
    for (int b = 0; b < n && rank < k; ++b) rank += index[b] >= 0 && before(value[b], index[b], v, id);
    if (rank < k) {
      top_value[rank] = v;
      top_index[rank] = id;
    }
  }
  __syncthreads();
  answer<DT, L>(st, x + static_cast<long>(row) * ld, c, labels, n_labels, row, k, top_value, top_index, out);
}

// Parts per row: a row of fewer than 1024 is cut until 1024 workgroups are there or a part has 4096 classes.
int splits_of(long rows, int c) {
  const long want = (1024 + rows - 1) / rows, most = (c + 4095) / 4096;
  const long n = want < most ? want : most;
  return static_cast<int>(n < 1 ? 1 : n > SPLITS_MAX ? SPLITS_MAX : n);
}

template <int DT, typename L>
void launch(const void* x, long ld, long rows, int c, const void* labels, int n_labels, int k, const Out& out, void* ws,
            hipStream_t s) {
  const auto* xp = static_cast<const typename mx_elem<DT>::type*>(x);
  const auto* lp = static_cast<const L*>(labels);
  const int splits = splits_of(rows, c);
  if (splits == 1) {
    hipLaunchKernelGGL((logprobs_kernel<DT, L>), dim3(static_cast<unsigned>(rows < (1 << 20) ? rows : (1 << 20))), dim3(T),
                       0, s, xp, ld, rows, c, lp, n_labels, k, out);
    return;
  }
  const int parts = static_cast<int>(rows) * splits, len = ((c + splits - 1) / splits + 7) / 8 * 8;
  float* st = static_cast<float*>(ws);
  float* wv = st + parts * 3;
  int* wi = reinterpret_cast<int*>(wv + parts * k);
  hipLaunchKernelGGL((logprobs_part_kernel<DT>), dim3(parts), dim3(T), 0, s, xp, ld, c, splits, len, k, st, wv, wi);
  hipLaunchKernelGGL((logprobs_join_kernel<DT, L>), dim3(static_cast<unsigned>(rows)), dim3(T), 0, s, xp, ld, c, lp, n_labels,
                     splits, k, st, wv, wi, out);
}

}  // namespace

// 4-byte words of workspace that ai4e_label_logprobs takes (0: none)
AI4E_API int ai4e_label_logprobs_ws(long rows, int c, int k) {
  if (rows <= 0 || c <= 0) return 0;
  const int splits = splits_of(rows, c);
  return splits == 1 ? 0 : static_cast<int>(rows) * splits * (3 + 2 * k);
}

// logits [rows, ld] of type dt (0 bf16, 1 fp16, 2 fp32), c valid columns; labels [rows, n_labels] int64 (wide) or int32;
// logp [rows, n_labels], entropy [rows], top_idx / top_logp [rows, k], k <= 64 and <= c.
AI4E_API int ai4e_label_logprobs(const void* logits, long ld, long rows, int c, int dt, const void* labels, int wide,
                                 int n_labels, int k, void* logp, void* entropy, void* top_idx, void* top_logp, void* ws,
                                 hipStream_t s) {
  if (!logits || !entropy || c <= 0 || c > (1 << 30) || ld < c || rows < 0 || dt < 0 || dt > 2 || k < 0 || k > KMAX || k > c ||
      n_labels < 0 || (n_labels && (!labels || !logp)) || (k && (!top_idx || !top_logp)))
    return AI4E_EINVAL;
  if (rows == 0) return AI4E_OK;
  if (splits_of(rows, c) > 1 && !ws) return AI4E_EINVAL;
  const Out out = {static_cast<float*>(logp), static_cast<float*>(entropy), static_cast<int*>(top_idx),
                   static_cast<float*>(top_logp)};
#define GO(DT)                                                                                       \
  if (wide) launch<DT, int64_t>(logits, ld, rows, c, labels, n_labels, k, out, ws, s);               \
  else launch<DT, int32_t>(logits, ld, rows, c, labels, n_labels, k, out, ws, s)
  if (dt == MX_BF16) { GO(MX_BF16); }
  else if (dt == MX_F16) { GO(MX_F16); }
  else { GO(MX_F32); }
#undef GO
  return hipGetLastError() == hipSuccess ? AI4E_OK : AI4E_ELAUNCH;
}
