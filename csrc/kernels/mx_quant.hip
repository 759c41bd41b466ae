// MX quantisation and its reverse (formats: mx.h).
//
// y = round(x / 2^e) per block of 32, e from the block's largest |x|: nothing but a maximum over 32 values stands between
// a load and a store, so both directions are bound by memory. A thread takes 8 values (16 B of 16-bit input) twice, four
// neighbouring lanes a block: the maximum is two DPP steps, and a wave's stores are contiguous. 16384 x 8192 bf16 to e2m1
// 59 us (5.75 TB/s; 67 with one group per thread, 60 with four), back 66 us with the codes out of memory (5.2 TB/s) and 48
// where the memory-side cache still holds them (through L2 108).
#include "mx.h"

namespace {

constexpr int THREADS = 256, PER = 2;  // groups of 8 values per thread, one workgroup's width apart

// group g of 8 stored elements -> (row, group in the row); a workgroup's first is divided in 64 bits once, as a scalar,
// and the lanes only divide what is left
struct Place {
  long row;
  int col8;
};
__device__ __forceinline__ Place place(int per_row, int i) {
  const long g0 = static_cast<long>(blockIdx.x) * THREADS * PER;
  const long r0 = g0 / per_row;
  const uint32_t q = static_cast<uint32_t>(g0 - r0 * per_row) + threadIdx.x + THREADS * i;
  const uint32_t dr = q / static_cast<uint32_t>(per_row);
  return {r0 + dr, static_cast<int>(q - dr * per_row)};
}

template <int DT, int FMT>
__global__ __launch_bounds__(THREADS) void quantize_kernel(const typename mx_elem<DT>::type* __restrict__ x, long ldx,
                                                           long rows, int k, int kp, uint8_t* __restrict__ data,
                                                           uint8_t* __restrict__ scale) {
  const int per_row = kp / 8;
  Place at[PER];
  float f[PER][8];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    at[i] = place(per_row, i);
    if (at[i].row >= rows) continue;  // per_row is a multiple of 16: a block's four lanes go together
    const int c = at[i].col8 * 8;
    const auto* p = x + at[i].row * ldx + c;
    if (c + 8 <= k)
      mx_floats<DT>(mx_load8<DT>(p), f[i]);
    else
      mx_load8_tail<DT>(p, k - c, 0.f, f[i]);
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (at[i].row >= rows) continue;
    const int code = mx_scale_code<FMT>(mx_quad_max(mx_abs_bits8(f[i])));
    const long g = at[i].row * per_row + at[i].col8;
    if constexpr (FMT == MX_E4M3)
      mx_store_past(reinterpret_cast<uint2*>(data) + g, mx_pack_e4m3(f[i], code));
    else
      mx_store_past(reinterpret_cast<uint32_t*>(data) + g, mx_pack_e2m1(f[i], code));
    if ((threadIdx.x & 3) == 0) scale[g >> 2] = static_cast<uint8_t>(code);
  }
}

__device__ __forceinline__ float scale_value(int code) {
  return code == 255 ? __uint_as_float(0x7fc00000u)
                     : (code == 0 ? __uint_as_float(0x00400000u) : __uint_as_float(static_cast<uint32_t>(code) << 23));
}

template <int DT, int FMT>
__global__ __launch_bounds__(THREADS) void dequantize_kernel(const uint8_t* __restrict__ data,
                                                             const uint8_t* __restrict__ scale, long rows, int k, int kp,
                                                             typename mx_elem<DT>::type* __restrict__ y) {
  const int per_row = kp / 8;
  Place at[PER];
  uint2 q[PER];
  int code[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    at[i] = place(per_row, i);
    if (at[i].row >= rows) continue;
    const long g = at[i].row * per_row + at[i].col8;
    code[i] = scale[g >> 2];
    if constexpr (FMT == MX_E4M3)
      q[i] = reinterpret_cast<const uint2*>(data)[g];
    else
      q[i].x = reinterpret_cast<const uint32_t*>(data)[g];
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int c = at[i].col8 * 8;
    if (at[i].row >= rows) continue;
    const float s = scale_value(code[i]);
    float f[8];
    if constexpr (FMT == MX_E4M3) {
      f[0] = __builtin_amdgcn_cvt_f32_fp8(q[i].x, 0); f[1] = __builtin_amdgcn_cvt_f32_fp8(q[i].x, 1);
      f[2] = __builtin_amdgcn_cvt_f32_fp8(q[i].x, 2); f[3] = __builtin_amdgcn_cvt_f32_fp8(q[i].x, 3);
      f[4] = __builtin_amdgcn_cvt_f32_fp8(q[i].y, 0); f[5] = __builtin_amdgcn_cvt_f32_fp8(q[i].y, 1);
      f[6] = __builtin_amdgcn_cvt_f32_fp8(q[i].y, 2); f[7] = __builtin_amdgcn_cvt_f32_fp8(q[i].y, 3);
    } else {
      f32x2_t v;
      v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[i].x, 1.f, 0); f[0] = v[0]; f[1] = v[1];
      v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[i].x, 1.f, 1); f[2] = v[0]; f[3] = v[1];
      v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[i].x, 1.f, 2); f[4] = v[0]; f[5] = v[1];
      v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[i].x, 1.f, 3); f[6] = v[0]; f[7] = v[1];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] *= s;
    mx_store8_quad<DT>(y + at[i].row * k, c, k, f);
  }
}

// a launch has fewer than 2^32 threads
bool bad_shape(long rows, int k) {
  return rows < 0 || k <= 0 || k > (1 << 30) ||
         rows > ((1L << 32) - THREADS) * PER / (static_cast<long>(ai4e_cdiv(k, MX_ALIGN)) * (MX_ALIGN / 8));
}

}  // namespace

#define AI4E_MX_EACH(DT, FMT, DO)                               \
  if (DT == MX_BF16 && FMT == MX_E4M3) DO(MX_BF16, MX_E4M3)     \
  else if (DT == MX_BF16) DO(MX_BF16, MX_E2M1)                  \
  else if (DT == MX_F16 && FMT == MX_E4M3) DO(MX_F16, MX_E4M3)  \
  else if (DT == MX_F16) DO(MX_F16, MX_E2M1)                    \
  else if (FMT == MX_E4M3) DO(MX_F32, MX_E4M3)                  \
  else DO(MX_F32, MX_E2M1)

// x [rows, ldx] of type dt (0 bf16, 1 fp16, 2 fp32), k valid columns; kp = k up to a multiple of 128:
// data [rows, kp] (fmt 0, e4m3) or [rows, kp / 2] (fmt 1, e2m1), scale [rows, kp / 32].
AI4E_API int ai4e_mx_quantize(const void* x, long ldx, long rows, int k, int dt, int fmt, void* data, void* scale,
                              hipStream_t s) {
  if (dt < 0 || dt > 2 || fmt < 0 || fmt > 1 || bad_shape(rows, k) || ldx < k) return AI4E_EINVAL;
  if (rows == 0) return AI4E_OK;  // tensors without elements have no memory
  if (!x || !data || !scale) return AI4E_EINVAL;
  const int kp = ai4e_cdiv(k, MX_ALIGN) * MX_ALIGN;
  const dim3 grid(ai4e_cdiv(rows * (kp / 8), THREADS * PER)), block(THREADS);
#define DO(DT, FMT)                                                                                               \
  hipLaunchKernelGGL((quantize_kernel<DT, FMT>), grid, block, 0, s, static_cast<const mx_elem<DT>::type*>(x), ldx, \
                     rows, k, kp, static_cast<uint8_t*>(data), static_cast<uint8_t*>(scale));
  AI4E_MX_EACH(dt, fmt, DO)
#undef DO
  return hipGetLastError() == hipSuccess ? AI4E_OK : AI4E_ELAUNCH;
}

// the values that codes stand for: y [rows, k] contiguous, of type dt
AI4E_API int ai4e_mx_dequantize(const void* data, const void* scale, long rows, int k, int dt, int fmt, void* y,
                                hipStream_t s) {
  if (dt < 0 || dt > 2 || fmt < 0 || fmt > 1 || bad_shape(rows, k)) return AI4E_EINVAL;
  if (rows == 0) return AI4E_OK;
  if (!data || !scale || !y) return AI4E_EINVAL;
  const int kp = ai4e_cdiv(k, MX_ALIGN) * MX_ALIGN;
  const dim3 grid(ai4e_cdiv(rows * (kp / 8), THREADS * PER)), block(THREADS);
#define DO(DT, FMT)                                                                                                   \
  hipLaunchKernelGGL((dequantize_kernel<DT, FMT>), grid, block, 0, s, static_cast<const uint8_t*>(data),              \
                     static_cast<const uint8_t*>(scale), rows, k, kp, static_cast<mx_elem<DT>::type*>(y));
  AI4E_MX_EACH(dt, fmt, DO)
#undef DO
  return hipGetLastError() == hipSuccess ? AI4E_OK : AI4E_ELAUNCH;
}
