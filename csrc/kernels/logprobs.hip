// K8 answers as log-probabilities: per row of logits x the log-probability of given labels, the entropy and the k most
// likely classes.
//
//   m = max x_j     s = sum e^(x_j - m)     t = sum e^(x_j - m) (x_j - m)
//   logp(j) = x_j - m - log s               entropy = log s - t / s
//
// One pass: a lane keeps its maximum, s and t of the elements it has seen and rescales s and t when the maximum grows, so
// a logit is read once. The pass works in base 2, s = sum 2^d and t = sum 2^d d with d = x log2 e - mu in one fused
// operation, mu the rounded m log2 e: what mu lost, at most 2^-8, is put back at the end. -inf gives 2^d = 0. From
// |m| = 2^16 on mu would lose more, up to what 2^d cannot hold: there it lies over m log2 e, so that no d is over 0 and a
// lane that has seen nothing but such a mask adds 0 to its row, and a row whose maximum lies there is summed again from
// differences x - m.
//
// The k best come out of the same pass (logprobs_kernel). A lane also keeps its best chunk (8 consecutive logits; the
// first one with the lane's maximum) and the maxima of SEGMENTS parts of its chunks. The k-th largest of 256 groups'
// (maximum, chunk) pairs bounds the k-th best logit from below, so only the k groups at or above it hold candidates, and of
// their parts those that reach it: these are read again, what reaches the bound is put into LDS, and each candidate's rank is
// the number of candidates before it. Ties go to the lower class.
// If more candidates come than LDS has room for (their order on the row is adverse), k rounds over the row find one each.
// Short rows with few alternatives stay in one wave's registers (logprobs_wave_kernel).
#include <type_traits>

#include "mx.h"

namespace {

constexpr int KMAX = 64, CAP = 1024, GROUPS = 256, SEGMENTS = 8;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float LOWEST = -3.402823466e38f;
constexpr float OUTER = 65536.f;  // logits from here on are summed from differences (fp16 has none)
constexpr float FAR = -200.f;  // 2^FAR is 0 in 32 bits; keeps 0 * d from being 0 * -inf

// the largest logit (-inf: none yet) and the sums relative to it
struct Stat {
  float m, s, t;
};

__device__ __forceinline__ float mu_of(float m) {
  const float p = m * LOG2E, a = fabsf(m);
  return fmaxf(a < OUTER ? p : fmaf(a, 0x1p-20f, p), LOWEST);  // 2^-20 m is over the two roundings of m log2 e
}

// v's sums (base 2), taken relative to mu, relative to a maximum m >= v.m, whose reference is to_mu
__device__ __forceinline__ Stat rescaled(const Stat& v, float mu, float m, float to_mu) {
  // the minimum only makes a number of inf - inf (both references are over 32 bits: the sums are 0); at m = -OUTER, where
  // mu steps up, the difference may be as large as 2^-4
  const float d = fminf(mu - to_mu, 1.f), f = __builtin_amdgcn_exp2f(d);
  return {m, v.s * f, f * (v.t + fmaxf(d, FAR) * v.s)};
}
__device__ __forceinline__ Stat rescaled(const Stat& v, float m) { return rescaled(v, mu_of(v.m), m, mu_of(m)); }

// lane i's value from lane i ^ 1, i ^ 2, 7 - i of 8, 15 - i of 16: four steps that join 16 lanes
template <int STEP>
__device__ __forceinline__ int dpp(int v) {
  constexpr int CTRL[4] = {0xB1, 0x4E, 0x141, 0x140};
  return __builtin_amdgcn_mov_dpp(v, CTRL[STEP], 0xF, 0xF, true);
}
template <int STEP>
__device__ __forceinline__ float dpp(float v) {
  return __int_as_float(dpp<STEP>(__float_as_int(v)));
}
template <typename V, typename F>
__device__ __forceinline__ V wave_all(V v, F op) {
  v = op(v, dpp<0>(v));
  v = op(v, dpp<1>(v));
  v = op(v, dpp<2>(v));
  v = op(v, dpp<3>(v));
  const int b = __builtin_bit_cast(int, v);
  const V v0 = __builtin_bit_cast(V, __builtin_amdgcn_readlane(b, 0)), v1 = __builtin_bit_cast(V, __builtin_amdgcn_readlane(b, 16));
  const V v2 = __builtin_bit_cast(V, __builtin_amdgcn_readlane(b, 32)), v3 = __builtin_bit_cast(V, __builtin_amdgcn_readlane(b, 48));
  return op(op(v0, v1), op(v2, v3));
}
__device__ __forceinline__ float wave_max(float v) {
  return wave_all(v, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float wave_sum(float v) {
  return wave_all(v, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ int wave_min(int v) {
  return wave_all(v, [](int a, int b) { return min(a, b); });
}
__device__ __forceinline__ Stat wave_join(const Stat& v) {
  const Stat r = rescaled(v, wave_max(v.m));
  return {r.m, wave_sum(r.s), wave_sum(r.t)};
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

// v_max3_f32 as such: from raw bits the compiler would quiet every operand first, an instruction each
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
__device__ __forceinline__ float max8(const float (&f)[8]) {
  const float a = max3(f[0], f[1], f[2]), b = max3(f[3], f[4], f[5]);
  return max3(max3(a, f[6], f[7]), b, b);
}

// s and t of 8 logits, base 2, relative to mu
__device__ __forceinline__ void add8(Stat& st, const float (&f)[8], float mu) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float d = fmaf(f[i], LOG2E, -mu), e = __builtin_amdgcn_exp2f(d);
    st.s += e;
    st.t = fmaf(e, fmaxf(d, FAR), st.t);
  }
}
// the same from differences, base e: for any finite maximum
__device__ __forceinline__ void add8_differences(Stat& st, const float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float u = f[i] - st.m, e = __builtin_amdgcn_exp2f(u * LOG2E);
    st.s += e;
    st.t = fmaf(e, fmaxf(u, FAR), st.t);
  }
}

struct Out {
  float* logp;
  float* entropy;
  int* top_idx;
  float* top_logp;
};

// label j of a row: its logit, and whether it is below 0 (the row has none) or over the classes
struct Label {
  float x;
  int kind;
};
// the labels of all rows, n of each, int64 or int32
struct Labels {
  const void* p;
  int n;
  bool wide;
};
template <int DT>
__device__ __forceinline__ Label label(const typename mx_elem<DT>::type* x, int c, const Labels& lab, int j, long row) {
  Label v = {0.f, -1};
  if (j < lab.n) {
    const long at = row * lab.n + j;
    const long l = lab.wide ? static_cast<const int64_t*>(lab.p)[at] : static_cast<const int32_t*>(lab.p)[at];
    v.kind = l < 0 ? -1 : l >= c ? 1 : 0;
    if (v.kind == 0) v.x = mx_elem<DT>::one(x[l]);
  }
  return v;
}

// What a row answers, from its sums. No finite logit: nothing is possible (log-probabilities -inf, entropy 0). A NaN or
// +inf among them: no distribution (NaN, classes -1).
struct Answer {
  float m, log_s, entropy;
  bool none, bad;
  __device__ Answer(const Stat& st, bool differences)
      : m(st.m), none(st.m == -INFINITY), bad(!(st.s < INFINITY)) {
    const float ln = logf(st.s);
    log_s = differences ? ln : ln - fmaf(m, LOG2E, -mu_of(m)) * LN2;
    entropy = differences ? ln - st.t / st.s : ln - st.t / st.s * LN2;
  }
  static __device__ float nan() { return __uint_as_float(0x7fc00000u); }
  __device__ float logp(float v) const { return bad ? nan() : none ? -INFINITY : (v - m) - log_s; }
  // the entropy and the labels, by the lanes of one wave; `first` holds the first 64 labels' logits
  template <int DT>
  __device__ void labels(const Label& first, const typename mx_elem<DT>::type* x, int c, const Labels& lab, long row,
                         const Out& out) const {
    const int lane = threadIdx.x & 63;
    if (lane == 0) out.entropy[row] = bad ? nan() : none ? 0.f : entropy;
    Label v = first;
    for (int j = lane; j < lab.n; j += 64) {
      if (j >= 64) v = label<DT>(x, c, lab, j, row);
      out.logp[row * lab.n + j] = v.kind < 0 ? 0.f : v.kind > 0 ? nan() : logp(v.x);
    }
  }
  // alternative r: (v, class), class < 0 where there is none
  __device__ void top(int r, float v, int id, long row, int k, const Out& out) const {
    out.top_idx[row * k + r] = bad ? -1 : id;
    out.top_logp[row * k + r] = id < 0 && !bad ? -INFINITY : logp(v);
  }
};

template <int WAVES>
struct Shared {
  Stat stat[WAVES];
  uint32_t key[GROUPS];  // each group's maximum (ordered; 0: it has seen nothing over -inf) and chunk
  int chunk[GROUPS];
  float least;           // the bound: a logit over it is a candidate, one equal to it up to chunk `last`
  int last;
  int groups[KMAX];      // the groups at or over the bound
  float part[SEGMENTS][WAVES * 64];  // each lane's maxima of the parts of its chunks
  uint16_t parts[KMAX * (WAVES * 64 / GROUPS) * SEGMENTS];  // those groups' parts that reach the bound: lane, part
  int n_groups, n_parts, n_cand;
  uint64_t cand[CAP];    // candidates: the ordered logit, then the class counted down
  float round_value[WAVES];
  int round_index[WAVES];
};

// The bound that the k best groups (larger key, then the lower chunk, first) reach, and which they are, by one wave: the
// key bit by bit, until exactly k groups reach it, then the chunk among equal keys.
template <int WAVES>
__device__ __forceinline__ void find_bound(Shared<WAVES>& sh, int k) {
  constexpr int PER = GROUPS / 64;
  const int lane = threadIdx.x & 63;
  uint32_t key[PER];
  int chunk[PER];
#pragma unroll
  for (int w = 0; w < PER; ++w) {
    key[w] = sh.key[lane + 64 * w];
    chunk[w] = sh.chunk[lane + 64 * w];
  }
  uint32_t bound = 0;
  int reach = 0;
  for (int b = 31; b >= 0 && reach != k; --b) {
    const uint32_t c = bound | (1u << b);
    int n = 0;
#pragma unroll
    for (int w = 0; w < PER; ++w) n += __popcll(__ballot(key[w] >= c));
    if (n >= k) {
      bound = c;
      reach = n;
    }
  }
  int last = 0x7fffffff;
  if (bound && reach > k) {  // equal keys: the smallest `last` with enough of them at or before it
    int over = 0;
#pragma unroll
    for (int w = 0; w < PER; ++w) over += __popcll(__ballot(key[w] > bound));
    last = 0;
    for (int b = 30; b >= 0; --b) {
      const int c = last + (1 << b);  // with fewer than k - over before c, the answer is c or later
      int n = 0;
#pragma unroll
      for (int w = 0; w < PER; ++w) n += __popcll(__ballot(key[w] == bound && chunk[w] < c));
      if (n < k - over) last = c;
    }
  }
  int at = 0;
#pragma unroll
  for (int w = 0; w < PER; ++w) {
    const bool in = key[w] && (key[w] > bound || (key[w] == bound && chunk[w] <= last));
    const unsigned long long mask = __ballot(in);
    if (in) sh.groups[at + __popcll(mask & ((1ull << lane) - 1))] = lane + 64 * w;
    at += __popcll(mask);
  }
  if (lane == 0) {
    sh.least = bound ? unordered(bound) : -INFINITY;
    sh.last = bound ? last : -1;
    sh.n_groups = at;
    sh.n_parts = 0;
    sh.n_cand = 0;
  }
}

// A workgroup of WAVES waves per row. PAST: the pass reads past the caches (see launch).
template <int DT, int WAVES, bool PAST>
__global__ __launch_bounds__(WAVES * 64) void logprobs_kernel(const typename mx_elem<DT>::type* __restrict__ x, long ld,
                                                              long rows, int c, Labels labels, int k, Out out) {
  constexpr int T = WAVES * 64, MEMBERS = T / GROUPS;
  constexpr int U = 2;  // chunks per step and lane, the next step's in flight
  __shared__ Shared<WAVES> sh;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int full = c / 8, chunks = (c + 7) / 8;
  // a lane's chunks, `per` of them T apart, in at most SEGMENTS parts of whole steps
  const int per = (chunks + T - 1) / T, length = U * ((per + U * SEGMENTS - 1) / (U * SEGMENTS));
  for (long row = blockIdx.x; row < rows; row += gridDim.x) {
    const auto* xr = x + row * ld;
    Label first = {0.f, -1};
    if (wave == 1) first = label<DT>(xr, c, labels, lane, row);
    Stat st = {-INFINITY, 0.f, 0.f};
    float mu = LOWEST;  // st's reference, mu_of(st.m)
    int best_chunk = 0;
    float part = -INFINITY;
    typedef mx_raw8<DT> Pack;
    // N chunks' logits, one rescaling for all
    auto take = [&](auto count, const Pack* q, int at) {
      constexpr int N = decltype(count)::value;
      float f[N][8], m = st.m;
#pragma unroll
      for (int u = 0; u < N; ++u) {
        mx_floats<DT>(q[u], f[u]);
        const float cm = max8(f[u]);
        best_chunk = cm > m ? at + u * T : best_chunk;
        m = fmaxf(m, cm);
        part = fmaxf(part, cm);
      }
      const float to_mu = mu_of(m);
      st = rescaled(st, mu, m, to_mu);
      mu = to_mu;
#pragma unroll
      for (int u = 0; u < N; ++u) add8(st, f[u], mu);
    };
    const int steps = full / (U * T);
    if (steps > 0) {
      Pack q[U];
      auto fetch = [&](Pack(&p)[U], int step) {
#pragma unroll
        for (int u = 0; u < U; ++u) p[u] = mx_load8<DT, PAST>(xr + ((step * U + u) * T + tid) * 8l);
      };
      fetch(q, 0);
      int end = length, p = 0;
      for (int i = 0; i < steps; ++i) {
        Pack next[U];
        if (i + 1 < steps) fetch(next, i + 1);
        take(std::integral_constant<int, U>{}, q, i * U * T + tid);
#pragma unroll
        for (int u = 0; u < U; ++u) q[u] = next[u];
        if ((i + 1) * U == end) {
          sh.part[p++][tid] = part;
          part = -INFINITY;
          end += length;
        }
      }
    }
    for (int at = steps * U * T + tid; at < full; at += T) {
      const Pack q = mx_load8<DT>(xr + at * 8l);
      take(std::integral_constant<int, 1>{}, &q, at);
    }
    if (chunks > full && tid == full % T) {
      float f[8];
      mx_load8_tail<DT>(xr + full * 8l, c - full * 8, -INFINITY, f);
      const float cm = max8(f);
      best_chunk = cm > st.m ? full : best_chunk;
      part = fmaxf(part, cm);
      st = rescaled(st, fmaxf(st.m, cm));
      add8(st, f, mu_of(st.m));
    }
    if (steps * U < per || steps * U % length) sh.part[steps * U / length][tid] = part;  // the last, unfinished part
    float best = st.m;
    const Stat w = wave_join(st);
    if (lane == 0) sh.stat[wave] = w;
    if constexpr (MEMBERS == 4) {  // a group is four neighbouring lanes
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const float ob = s ? dpp<1>(best) : dpp<0>(best);
        const int oc = s ? dpp<1>(best_chunk) : dpp<0>(best_chunk);
        if (before(ob, oc, best, best_chunk)) {
          best = ob;
          best_chunk = oc;
        }
      }
    }
    if (tid % MEMBERS == 0) {
      sh.key[tid / MEMBERS] = best > -INFINITY ? ordered(best) : 0;
      sh.chunk[tid / MEMBERS] = best_chunk;
    }
    __syncthreads();
    // the second wave finishes the labels while the first looks for the bound
    if (wave == 0 && k > 0) find_bound(sh, k);
    Stat all = {-INFINITY, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < WAVES; ++i) all.m = fmaxf(all.m, sh.stat[i].m);
#pragma unroll
    for (int i = 0; i < WAVES; ++i) {
      const Stat r = rescaled(sh.stat[i], all.m);
      all.s += r.s;
      all.t += r.t;
    }
    const bool again = fabsf(all.m) >= OUTER && fabsf(all.m) < INFINITY;
    if (again) {
      Stat d = {all.m, 0.f, 0.f};
      for (int at = tid; at < chunks; at += T) {
        float f[8];
        load_chunk<DT>(xr, at * 8, c, f);
        add8_differences(d, f);
      }
      d.s = wave_sum(d.s);
      d.t = wave_sum(d.t);
      __syncthreads();  // every wave has read the first sums
      if (lane == 0) sh.stat[wave] = d;
      __syncthreads();
      all.s = all.t = 0.f;
#pragma unroll
      for (int i = 0; i < WAVES; ++i) {
        all.s += sh.stat[i].s;
        all.t += sh.stat[i].t;
      }
    }
    const Answer ans(all, again);
    if (wave == 1) ans.labels<DT>(first, xr, c, labels, row, out);
    if (k > 0) {
      __syncthreads();
      const float least = sh.least;
      const int last = sh.last;
      const int nparts = (per + length - 1) / length, all_parts = sh.n_groups * MEMBERS * nparts;
      for (int it = tid; it < all_parts; it += T) {
        const int g = it / nparts, p = it - g * nparts, from = sh.groups[g / MEMBERS] * MEMBERS + g % MEMBERS;
        if (sh.part[p][from] >= least) sh.parts[atomicAdd(&sh.n_parts, 1)] = static_cast<uint16_t>(from * SEGMENTS + p);
      }
      __syncthreads();
      const int items = sh.n_parts * length;
      for (int it = tid; it < items; it += T) {
        const int i = it / length, j = sh.parts[i] % SEGMENTS * length + it - i * length;
        const int at = sh.parts[i] / SEGMENTS + j * T;
        if (j >= per || at >= chunks) continue;
        float f[8];
        load_chunk<DT>(xr, at * 8, c, f);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (f[i] > least || (f[i] == least && at <= last)) {
            const int to = atomicAdd(&sh.n_cand, 1);
            if (to < CAP) sh.cand[to] = static_cast<uint64_t>(ordered(f[i])) << 32 | ~static_cast<uint32_t>(at * 8 + i);
          }
      }
      __syncthreads();
      const int cand = sh.n_cand;
      if (cand <= CAP) {
        for (int a = tid; a < cand; a += T) {
          const uint64_t key = sh.cand[a];
          int rank = 0;
          for (int b = 0; b < cand; b += 8) {  // read together; what lies behind the last candidate does not count
            uint64_t other[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) other[i] = sh.cand[b + i];
#pragma unroll
            for (int i = 0; i < 8; ++i) rank += b + i < cand && other[i] > key;
          }
          if (rank < k) ans.top(rank, unordered(key >> 32), ~static_cast<uint32_t>(key), row, k, out);
        }
        if (tid >= cand && tid < k) ans.top(tid, 0.f, -1, row, k, out);
      } else {
        float pv = INFINITY;  // the class that the last round found
        int pi = -1;
        for (int r = 0; r < k; ++r) {
          float bv = -INFINITY;
          int bi = 0x7fffffff;
          for (int at = tid; at < chunks; at += T) {
            float f[8];
            load_chunk<DT>(xr, at * 8, c, f);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int id = at * 8 + i;
              if (f[i] > -INFINITY && before(pv, pi, f[i], id) && before(f[i], id, bv, bi)) {
                bv = f[i];
                bi = id;
              }
            }
          }
          const float wv = wave_max(bv);
          const int wi = wave_min(bv == wv ? bi : 0x7fffffff);
          __syncthreads();  // the last round's slots have been read
          if (lane == 0) {
            sh.round_value[wave] = wv;
            sh.round_index[wave] = wi;
          }
          __syncthreads();
          pv = sh.round_value[0];
          pi = sh.round_index[0];
#pragma unroll
          for (int i = 1; i < WAVES; ++i)
            if (before(sh.round_value[i], sh.round_index[i], pv, pi)) {
              pv = sh.round_value[i];
              pi = sh.round_index[i];
            }
          if (tid == 0) ans.top(r, pv, pi, row, k, out);
        }
      }
    }
    __syncthreads();  // the next row writes the shared parts
  }
}

// A wave per row of at most 512 CH classes, all in registers; an alternative is a wave's maximum, then retired
template <int DT, int CH>
__global__ __launch_bounds__(256) void logprobs_wave_kernel(const typename mx_elem<DT>::type* __restrict__ x, long ld,
                                                            long rows, int c, Labels labels, int k, Out out) {
  const int lane = threadIdx.x & 63;
  const long row = static_cast<long>(blockIdx.x) * (blockDim.x >> 6) + (threadIdx.x >> 6);
  if (row >= rows) return;
  const auto* xr = x + row * ld;
  const Label first = label<DT>(xr, c, labels, lane, row);
  float f[CH][8];
#pragma unroll
  for (int j = 0; j < CH; ++j) {
    const int at = (j * 64 + lane) * 8;
    if (at < c)
      load_chunk<DT>(xr, at, c, f[j]);
    else
#pragma unroll
      for (int i = 0; i < 8; ++i) f[j][i] = -INFINITY;
  }
  Stat st = {-INFINITY, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < CH; ++j) st.m = fmaxf(st.m, max8(f[j]));
  st.m = wave_max(st.m);
  if (st.m == -INFINITY) {  // nothing but -inf and NaN: a difference would be NaN for either
#pragma unroll
    for (int j = 0; j < CH; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) st.s += f[j][i] == -INFINITY ? 0.f : f[j][i];
  } else {
#pragma unroll
    for (int j = 0; j < CH; ++j) add8_differences(st, f[j]);
  }
  st.s = wave_sum(st.s);
  st.t = wave_sum(st.t);
  const Answer ans(st, true);
  ans.labels<DT>(first, xr, c, labels, row, out);
  for (int r = 0; r < k; ++r) {
    float bv = -INFINITY;
    int bi = 0x7fffffff;
#pragma unroll
    for (int j = 0; j < CH; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (f[j][i] > bv) {
          bv = f[j][i];
          bi = (j * 64 + lane) * 8 + i;
        }
    const float wv = wave_max(bv);
    const int wi = wave_min(bv == wv ? bi : 0x7fffffff);
    if (lane == 0) ans.top(r, wv, wv > -INFINITY ? wi : -1, row, k, out);
#pragma unroll
    for (int j = 0; j < CH; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if ((j * 64 + lane) * 8 + i == wi) f[j][i] = -INFINITY;
  }
}

template <int DT>
void launch(const void* x, long ld, long rows, int c, const Labels& labels, int k, const Out& out, hipStream_t s) {
  const auto* xp = static_cast<const typename mx_elem<DT>::type*>(x);
#define GO(GRID, BLOCK, ...) \
  hipLaunchKernelGGL((__VA_ARGS__), dim3(static_cast<unsigned>(GRID)), dim3(BLOCK), 0, s, xp, ld, rows, c, labels, k, out)
  if (c <= 2048 && k <= 16 && rows <= (1 << 24)) {
    const int per = rows < 1024 ? 1 : 4;  // rows per workgroup
    const long grid = (rows + per - 1) / per;
    if (c <= 512) GO(grid, per * 64, logprobs_wave_kernel<DT, 1>);
    else if (c <= 1024) GO(grid, per * 64, logprobs_wave_kernel<DT, 2>);
    else GO(grid, per * 64, logprobs_wave_kernel<DT, 4>);
    return;
  }
  const long grid = rows < (1 << 20) ? rows : (1 << 20);
  // 16 waves per row where there are too few rows to fill the CUs with 4 (1 x 131072: 14.6 us against 18.3, 256 x 131072
  // 24.3 against 30.4, 256 x 9000 12.1 against 11.2); with more rows their phases cost more (512 x 131072 47.2 against 45.7,
  // 333 x 50001 fp32 26.2 against 18.3, 1024 x 32768 48.9 against 23.8)
  if (rows <= 256 && c >= 8192) GO(grid, 1024, logprobs_kernel<DT, 16, false>);
  // Logits are often what the last kernel wrote, so they are read through the caches (333 x 50001 fp32 18.5 us, past them
  // 28). No cache holds 512 MB of them: 16-bit ones then come faster past the caches (4096 x 131072 212 us, past them 193),
  // 32-bit ones do not (2048 x 131072 195, 199).
  else if (DT != MX_F32 && rows * c >= (256l << 20)) GO(grid, 256, logprobs_kernel<DT, 4, DT != MX_F32>);
  else GO(grid, 256, logprobs_kernel<DT, 4, false>);
#undef GO
}

}  // namespace

// logits [rows, ld] of type dt (0 bf16, 1 fp16, 2 fp32), c valid columns; labels [rows, n_labels] int64 (wide) or int32;
// logp [rows, n_labels], entropy [rows], top_idx / top_logp [rows, k], k <= 64 and <= c.
AI4E_API int ai4e_label_logprobs(const void* logits, long ld, long rows, int c, int dt, const void* labels, int wide,
                                 int n_labels, int k, void* logp, void* entropy, void* top_idx, void* top_logp,
                                 hipStream_t s) {
  if (c <= 0 || c > (1 << 30) || ld < c || rows < 0 || dt < 0 || dt > 2 || k < 0 || k > KMAX || k > c || n_labels < 0 ||
      n_labels > (1 << 30))
    return AI4E_EINVAL;
  if (rows == 0) return AI4E_OK;  // tensors without elements have no memory
  if (!logits || !entropy || (n_labels && (!labels || !logp)) || (k && (!top_idx || !top_logp))) return AI4E_EINVAL;
  const Out out = {static_cast<float*>(logp), static_cast<float*>(entropy), static_cast<int*>(top_idx),
                   static_cast<float*>(top_logp)};
  const Labels lab = {labels, n_labels, wide != 0};
  if (dt == MX_BF16) launch<MX_BF16>(logits, ld, rows, c, lab, k, out, s);
  else if (dt == MX_F16) launch<MX_F16>(logits, ld, rows, c, lab, k, out, s);
  else launch<MX_F32>(logits, ld, rows, c, lab, k, out, s);
  return hipGetLastError() == hipSuccess ? AI4E_OK : AI4E_ELAUNCH;
}
