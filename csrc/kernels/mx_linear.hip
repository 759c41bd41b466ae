// y = x . w^T + bias over MX operands (formats: mx.h): x e4m3 or e2m1, w e2m1, both [rows, k].
#include "mx.h"

namespace {

typedef int i32x8_t __attribute__((ext_vector_type(8)));

// v_mfma_scale_f32_32x32x64: D[32 x 32] += A[32 x 64] . B[32 x 64]^T, a scale for each row and block of 32.
// Lane l holds row l & 31. Its 32 elements are k = 32 (l >> 5) .. + 31 of e2m1, and k = 16 (l >> 5) .. + 15 and
// 32 + 16 (l >> 5) .. + 15 of e4m3; its scale is that of block l >> 5 in both (measured).
// Of D it holds column l & 31, rows 8 (i >> 2) + 4 (l >> 5) + (i & 3) for i = 0..15.
template <int FMT>
__device__ __forceinline__ i32x8_t load_frag(const uint8_t* row, int k0, int half) {
  i32x8_t v = {};
  if constexpr (FMT == MX_E4M3) {
    const uint4 a = *reinterpret_cast<const uint4*>(row + k0 + 16 * half);
    const uint4 b = *reinterpret_cast<const uint4*>(row + k0 + 32 + 16 * half);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    const uint4 a = *reinterpret_cast<const uint4*>(row + (k0 >> 1) + 16 * half);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  }
  return v;
}

// one 32 x 32 tile of y per wave: rows of w are the matrix instruction's first operand, so a lane ends with four
// consecutive outputs of one row of x
template <int FX, int DT>
__global__ __launch_bounds__(256) void mx_linear_kernel(const uint8_t* __restrict__ x, const uint8_t* __restrict__ xs,
                                                        const uint8_t* __restrict__ w, const uint8_t* __restrict__ ws,
                                                        const float* __restrict__ bias, int m, int n, int kp,
                                                        typename mx_elem<DT>::type* __restrict__ y) {
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int tiles_n = (n + 31) / 32;
  const long tile = static_cast<long>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int tm = static_cast<int>(tile / tiles_n), tn = static_cast<int>(tile % tiles_n);
  if (tm * 32 >= m) return;
  const int rx = min(tm * 32 + (lane & 31), m - 1), rw = min(tn * 32 + (lane & 31), n - 1);
  const uint8_t* xr = x + static_cast<long>(rx) * (FX == MX_E4M3 ? kp : kp / 2);
  const uint8_t* wr = w + static_cast<long>(rw) * (kp / 2);
  const uint8_t* xsr = xs + static_cast<long>(rx) * (kp / 32);
  const uint8_t* wsr = ws + static_cast<long>(rw) * (kp / 32);
  f32x16_t acc = {};
  for (int k0 = 0; k0 < kp; k0 += 64) {
    const i32x8_t a = load_frag<MX_E2M1>(wr, k0, half), b = load_frag<FX>(xr, k0, half);
    acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, acc, 4, FX == MX_E4M3 ? 0 : 4, 0,
                                                          wsr[(k0 >> 5) + half], 0, xsr[(k0 >> 5) + half]);
  }
  const int row = tm * 32 + (lane & 31);
  if (row >= m) return;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int col = tn * 32 + 8 * (i >> 2) + 4 * half + (i & 3);
    if (col < n) y[static_cast<long>(row) * n + col] = mx_elem<DT>::from(acc[i] + (bias ? bias[col] : 0.f));
  }
}

}  // namespace

// x: data [m, kp] (fx 0, e4m3) or [m, kp / 2] (fx 1, e2m1), xs [m, kp / 32]; w: [n, kp / 2], ws [n, kp / 32];
// bias [n] fp32 or null; y [m, n] of type dt (0 bf16, 1 fp16, 2 fp32). kp is a multiple of 128.
AI4E_API int ai4e_mx_linear(const void* x, const void* xs, int fx, const void* w, const void* ws, const void* bias,
                            int m, int n, int kp, void* y, int dt, hipStream_t s) {
  if (!x || !xs || !w || !ws || !y || m < 0 || n <= 0 || kp <= 0 || kp % MX_ALIGN || fx < 0 || fx > 1 || dt < 0 || dt > 2 ||
      n > (1 << 30) || m > (1 << 30) || static_cast<long>((m + 31) / 32) * ((n + 31) / 32) > (1L << 25))
    return AI4E_EINVAL;
  if (m == 0) return AI4E_OK;
  const dim3 grid(ai4e_cdiv(static_cast<long>((m + 31) / 32) * ((n + 31) / 32), 4)), block(256);
#define GO(FX, DT)                                                                                                     \
  hipLaunchKernelGGL((mx_linear_kernel<FX, DT>), grid, block, 0, s, static_cast<const uint8_t*>(x),                    \
                     static_cast<const uint8_t*>(xs), static_cast<const uint8_t*>(w), static_cast<const uint8_t*>(ws), \
                     static_cast<const float*>(bias), m, n, kp, static_cast<mx_elem<DT>::type*>(y))
  if (fx == MX_E4M3) {
    if (dt == MX_BF16) GO(MX_E4M3, MX_BF16); else if (dt == MX_F16) GO(MX_E4M3, MX_F16); else GO(MX_E4M3, MX_F32);
  } else {
    if (dt == MX_BF16) GO(MX_E2M1, MX_BF16); else if (dt == MX_F16) GO(MX_E2M1, MX_F16); else GO(MX_E2M1, MX_F32);
  }
#undef GO
  return hipGetLastError() == hipSuccess ? AI4E_OK : AI4E_ELAUNCH;
}
