// RMS norm with the residual's addition, written as MX e4m3 (formats: mx.h).
//
//   h = x + residual            y = h / sqrt(mean(h^2) + eps) * gamma            (e4m3, scales) = mx(y), h kept
//
// The row stays in registers between the sum of squares and the products, so memory is what bounds it: per value 2 + 2 B
// in, 2 B (h) and 1.03 B (codes, scales) out for 16-bit rows. A workgroup per row, or for narrow rows the 16, 32 or 64
// lanes that its chunks of 8 fill.
// A value next to the border of two 8-bit neighbours falls to either side by the last bit of y, so y is computed to one
// rounding: squares and the row's factor in double, h as the rounded sum and, of 32-bit rows, what the rounding lost, the
// factor as a float and its remainder, and each product with its error. Where the last rounding ends on a border it is
// taken back by a bit towards y, so that the 8-bit rounding sees y's side of it. 16384 x 8192 bf16 with a residual 172 us
// (5.5 TB/s, a copy's rate).
// Sums of 16-bit rows are 32-bit numbers: all of them fit but where x and the residual are 2^13 (fp16) or 2^16 (bf16) and
// more apart, and of such elements one in some 10^6 falls to the other side by what is lost. With it 16384 x 8192 bf16 took
// 180 us instead of 167.
#include "mx.h"

namespace {

// sum over a row's LANES lanes
template <int LANES>
__device__ __forceinline__ double row_sum(double s, double* lds) {
#pragma unroll
  for (int o = (LANES < 64 ? LANES : 64) / 2; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if constexpr (LANES > 64) {
    __syncthreads();  // the last row's sums have been read
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
    __syncthreads();
    s = 0;
#pragma unroll
    for (int w = 0; w < LANES / 64; ++w) s += lds[w];
  }
  return s;
}

// 1 / sqrt(d): the float estimate and a Newton step in double (to 2^-44) where the estimate is in range
__device__ __forceinline__ double inv_sqrt(double d) {
  if (!(d > 1e-30 && d < 1e38)) return 1.0 / sqrt(d);
  const double r = __builtin_amdgcn_rsqf(static_cast<float>(d));
  return r * (1.5 - 0.5 * d * r * r);
}

// h of 8 columns, those below n, and for 32-bit rows what its rounding lost
template <int DT>
__device__ __forceinline__ void load_h(const typename mx_elem<DT>::type* x, const typename mx_elem<DT>::type* r, int n,
                                       float (&h)[8], float (&low)[8]) {
  float g[8] = {};
  if (n >= 8) {
    mx_floats<DT>(mx_load8<DT>(x), h);
    if (r) mx_floats<DT>(mx_load8<DT>(r), g);
  } else {
    mx_load8_tail<DT>(x, n, 0.f, h);
    if (r) mx_load8_tail<DT>(r, n, 0.f, g);
  }
  if (!r) {
#pragma unroll
    for (int i = 0; i < 8; ++i) low[i] = 0.f;
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float s = h[i] + g[i], b = s - h[i];
    low[i] = DT == MX_F32 && fabsf(s) < INFINITY ? (h[i] - (s - b)) + (g[i] - b) : 0.f;
    h[i] = s;
  }
}

// LANES lanes per row; CH > 0: the row's chunks of 8 per lane, kept in registers; CH == 0: any width, read a second time
template <int DT, int LANES, int CH>
__global__ __launch_bounds__(LANES > 256 ? LANES : 256) void rms_norm_mx8_kernel(
    const typename mx_elem<DT>::type* __restrict__ x, long ldx, const typename mx_elem<DT>::type* __restrict__ res,
    long ldr, const float* __restrict__ gamma, float eps, double inv_c, long rows, int c, int cp,
    typename mx_elem<DT>::type* __restrict__ hout, uint8_t* __restrict__ data, uint8_t* __restrict__ scale) {
  constexpr int T = LANES > 256 ? LANES : 256, ROWS = T / LANES;
  static_assert(LANES <= 64 || ROWS == 1, "rows of several waves share no workgroup: they meet at its barriers");
  constexpr int KEEP = CH > 0 ? CH : 1;
  __shared__ double lds[T / 64];
  const int tid = threadIdx.x % LANES;
  const int nch = CH > 0 ? CH : (cp / 8 + LANES - 1) / LANES;
  for (long row = static_cast<long>(blockIdx.x) * ROWS + threadIdx.x / LANES; row < rows; row += static_cast<long>(gridDim.x) * ROWS) {
    const auto* xr = x + row * ldx;
    const auto* rr = res ? res + row * ldr : nullptr;
    float h[KEEP][8], low[KEEP][8];
    double sq = 0;  // in 64 bits, which the unit adds at the same rate: no square leaves its range
#pragma unroll
    for (int j = 0; j < nch; ++j) {
      const int col = (j * LANES + tid) * 8;
      float(&v)[8] = h[CH > 0 ? j : 0], (&lv)[8] = low[CH > 0 ? j : 0];
      load_h<DT>(xr + col, rr ? rr + col : nullptr, c - col, v, lv);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const double d = DT == MX_F32 ? static_cast<double>(v[i]) + lv[i] : v[i];
        sq = fma(d, d, sq);
      }
      if (hout) mx_store8_quad<DT>(hout + row * c, col, c, v);
    }
    const double factor = inv_sqrt(row_sum<LANES>(sq, lds) * inv_c + static_cast<double>(eps));
    const float fh = static_cast<float>(factor), fl = static_cast<float>(factor - static_cast<double>(fh));
#pragma unroll
    for (int j = 0; j < nch; ++j) {
      const int col = (j * LANES + tid) * 8;
      if (col >= cp) break;  // cp is a multiple of 128: a block's four lanes leave together
      float(&v)[8] = h[CH > 0 ? j : 0], (&lv)[8] = low[CH > 0 ? j : 0];
      if (CH == 0) load_h<DT>(xr + col, rr ? rr + col : nullptr, c - col, v, lv);
      float g[8], y[8];
      if (col + 8 <= c)
        mx_floats<MX_F32>(mx_load8<MX_F32>(gamma + col), g);
      else
        mx_load8_tail<MX_F32>(gamma + col, c - col, 0.f, g);
      auto product = [&](int i, float fa, float& rest) {  // h * factor * gamma in one rounding, and what it left
        const float a = v[i] * fa;
        float part = fmaf(v[i], fl, fmaf(v[i], fa, -a));
        if (DT == MX_F32) part = fmaf(lv[i], fa, part);
        const float e = part * g[i], p = fmaf(a, g[i], e);
        rest = fmaf(a, g[i], -p) + e;
        return p;
      };
      bool border = false;  // values of few significant bits, the 8-bit format's borders among them: 1 in 65536
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float rest;
        y[i] = col + i < c ? product(i, fh, rest) : 0.f;  // also where the factor is not finite
        const uint32_t b = __float_as_uint(y[i]);
        border |= (b & 0xffffu) == 0 && b << 1 != 0;
      }
      if (border) {
        float again = fh;
        asm("" : "+v"(again));  // computed again: kept for this branch, the parts took a sixth of the waves (177 -> 210 us)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t b = __float_as_uint(y[i]);
          float rest;
          product(i, again, rest);
          if ((b & 0xffffu) == 0 && b << 1 != 0 && fabsf(y[i]) < INFINITY && rest != 0.f)
            y[i] = __uint_as_float((rest > 0.f) == (y[i] > 0.f) ? b + 1 : b - 1);
        }
      }
      const int code = mx_scale_code<MX_E4M3>(mx_quad_max(mx_abs_bits8(y)));
      const long at = row * cp + col;
      mx_store_past(reinterpret_cast<uint2*>(data + at), mx_pack_e4m3(y, code));
      if ((tid & 3) == 0) scale[at >> 5] = static_cast<uint8_t>(code);
    }
  }
}

}  // namespace

// x [rows, ldx] and residual [rows, ldr] (or null) of type dt (0 bf16, 1 fp16, 2 fp32), c valid columns; gamma [c] fp32;
// hout [rows, c] of type dt (or null); data [rows, cp], scale [rows, cp / 32], cp = c up to a multiple of 128.
AI4E_API int ai4e_rms_norm_mx8(const void* x, long ldx, const void* residual, long ldr, const void* gamma, float eps,
                               long rows, int c, int dt, void* hout, void* data, void* scale, hipStream_t s) {
  if (c <= 0 || c > (1 << 30) || rows < 0 || dt < 0 || dt > 2 || ldx < c || (residual && ldr < c) || !(eps > 0.f))
    return AI4E_EINVAL;
  if (rows == 0) return AI4E_OK;  // tensors without elements have no memory
  if (!x || !gamma || !data || !scale) return AI4E_EINVAL;
  const int cp = ai4e_cdiv(c, MX_ALIGN) * MX_ALIGN;
#define GO(DT, LANES, CH)                                                                                        \
  {                                                                                                              \
    constexpr int T = LANES > 256 ? LANES : 256;                                                                 \
    const long blocks = (rows + T / LANES - 1) / (T / LANES);                                                    \
    hipLaunchKernelGGL((rms_norm_mx8_kernel<DT, LANES, CH>), dim3(static_cast<unsigned>(blocks < (1 << 20) ? blocks : (1 << 20))), \
                       dim3(T), 0, s, static_cast<const mx_elem<DT>::type*>(x), ldx,                             \
                       static_cast<const mx_elem<DT>::type*>(residual), ldr, static_cast<const float*>(gamma), eps, 1.0 / c, \
                       rows, c, cp, static_cast<mx_elem<DT>::type*>(hout), static_cast<uint8_t*>(data),          \
                       static_cast<uint8_t*>(scale));                                                            \
  }
// up to 8192 values a row takes as few lanes as hold it in two chunks each: 16384 x 8192 bf16 with 256 lanes x 4 chunks
// 184 us, 512 x 2 173, 1024 x 1 243; 4096 x 4096 256 x 2 21.8, 512 x 1 22.9
#define PICK(DT)                       \
  if (cp <= 128) GO(DT, 16, 1)         \
  else if (cp <= 256) GO(DT, 32, 1)    \
  else if (cp <= 512) GO(DT, 64, 1)    \
  else if (cp <= 2048) GO(DT, 256, 1)  \
  else if (cp <= 4096) GO(DT, 256, 2)  \
  else if (cp <= 8192) GO(DT, 512, 2)  \
  else if (cp <= 16384) GO(DT, 512, 4) \
  else GO(DT, 512, 0)
  if (dt == MX_BF16) { PICK(MX_BF16); }
  else if (dt == MX_F16) { PICK(MX_F16); }
  else { PICK(MX_F32); }
#undef PICK
#undef GO
  return hipGetLastError() == hipSuccess ? AI4E_OK : AI4E_ELAUNCH;
}
