// Block-scaled ("MX") 8- and 4-bit formats, shared by the kernels that write and read them.
//
// 32 consecutive values of a row share a scale 2^(code - 127); an element is the value / scale rounded to nearest even:
//   e4m3  1 byte, largest 448 = 1.75 * 2^8          e2m1  4 bits, largest 6 = 1.5 * 2^2 (even element in the low half)
// The code is the smallest that needs no clipping: max|x| <= largest * 2^(code - 127), at least 0. A block with a NaN or
// an infinity has code 255 (the scale's NaN) and zero elements. A row is stored up to a multiple of 128 elements, the
// depth of one matrix instruction, with zeros and code 0 behind the last value.
#pragma once
#include "common.h"

enum { MX_BF16 = 0, MX_F16 = 1, MX_F32 = 2 };   // element types of plain tensors at the C entries
enum { MX_E4M3 = 0, MX_E2M1 = 1 };
constexpr int MX_BLOCK = 32, MX_ALIGN = 128;

// 8 consecutive values as floats; rows of odd widths start at any element, so the loads assume element alignment
// only (global memory takes wide accesses at any address on gfx950).
template <int DT>
struct mx_elem;
template <>
struct mx_elem<MX_BF16> {
  typedef uint16_t type;
  static __device__ __forceinline__ float one(uint16_t v) { return bf16_to_f32(v); }
  static __device__ __forceinline__ uint16_t from(float f) { return f32_to_bf16(f); }
};
template <>
struct mx_elem<MX_F16> {
  typedef uint16_t type;
  static __device__ __forceinline__ float one(uint16_t v) { return static_cast<float>(__builtin_bit_cast(_Float16, v)); }
  static __device__ __forceinline__ uint16_t from(float f) {
    return __builtin_bit_cast(uint16_t, static_cast<_Float16>(f));
  }
};
template <>
struct mx_elem<MX_F32> {
  typedef float type;
  static __device__ __forceinline__ float one(float v) { return v; }
  static __device__ __forceinline__ float from(float f) { return f; }
};

// Results go past L2 (non-temporal): they are read by a later kernel on any XCD, and would push inputs out of it (RMS norm
// of 16384 x 8192 bf16: 196 us through L2, 173 past it). Inputs come through the caches, which often still hold what the
// last kernel wrote (RMS norm of 1003 x 5000 fp32 15.0 us, with loads past them 20.6; of 16384 x 8192 bf16 181 and 179).
typedef int mx_i32x4_t __attribute__((ext_vector_type(4), aligned(2)));
typedef int mx_i32x2_t __attribute__((ext_vector_type(2)));

// as loaded: kept in whole registers until they are taken apart, so that a load can be in flight
template <int DT>
struct mx_raw8 {
  mx_i32x4_t v[DT == MX_F32 ? 2 : 1];
};

template <int DT, bool PAST = false>
__device__ __forceinline__ mx_raw8<DT> mx_load8(const typename mx_elem<DT>::type* p) {
  mx_raw8<DT> w;
#pragma unroll
  for (int i = 0; i < (DT == MX_F32 ? 2 : 1); ++i) {
    const auto* q = reinterpret_cast<const mx_i32x4_t*>(p) + i;
    w.v[i] = PAST ? __builtin_nontemporal_load(q) : *q;
  }
  return w;
}

// the first n (0..8) of them, `fill` behind
template <int DT>
__device__ __forceinline__ void mx_load8_tail(const typename mx_elem<DT>::type* p, int n, float fill, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = i < n ? mx_elem<DT>::one(p[i]) : fill;
}

template <int DT>
__device__ __forceinline__ void mx_floats(const mx_raw8<DT>& q, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == MX_F32) {
      f[i] = __int_as_float(q.v[0][i]);
      f[4 + i] = __int_as_float(q.v[1][i]);
    } else {
      unpack2<DT == MX_F16>(static_cast<uint32_t>(q.v[0][i]), f[2 * i], f[2 * i + 1]);
    }
  }
}

__device__ __forceinline__ void mx_store_past(uint2* p, const uint2& v) {
  __builtin_nontemporal_store(mx_i32x2_t{static_cast<int>(v.x), static_cast<int>(v.y)}, reinterpret_cast<mx_i32x2_t*>(p));
}
__device__ __forceinline__ void mx_store_past(uint32_t* p, uint32_t v) { __builtin_nontemporal_store(v, p); }

// 8 values, those below n
template <int DT>
__device__ __forceinline__ void mx_store8(typename mx_elem<DT>::type* p, const float (&f)[8], int n) {
  struct Pack { typename mx_elem<DT>::type v[8]; } q;
#pragma unroll
  for (int i = 0; i < 8; ++i) q.v[i] = mx_elem<DT>::from(f[i]);
  if (n >= 8) {
    struct Words { mx_i32x4_t v[sizeof(Pack) / 16]; };
    const Words w = __builtin_bit_cast(Words, q);
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(Pack) / 16); ++i)
      __builtin_nontemporal_store(w.v[i], reinterpret_cast<mx_i32x4_t*>(p) + i);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = q.v[i];
  }
}

// Row[col .. col + 8) of k values, where four neighbouring lanes hold 32 consecutive columns: in 32 bits a lane's 32 B are
// passed around the four lanes so that each store fills 64 B (dequantised 16384 x 8192: 144 us, 214 as 16-B pieces).
template <int DT>
__device__ __forceinline__ void mx_store8_quad(typename mx_elem<DT>::type* row, int col, int k, const float (&f)[8]) {
  if constexpr (DT == MX_F32) {
    if ((col & ~31) + 32 <= k) {
      const bool odd = threadIdx.x & 1;
      mx_i32x4_t a, b;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int lo = __float_as_int(f[i]), hi = __float_as_int(f[4 + i]);
        const int a0 = __builtin_amdgcn_mov_dpp(lo, 0x50, 0xF, 0xF, true), a1 = __builtin_amdgcn_mov_dpp(hi, 0x50, 0xF, 0xF, true);
        const int b0 = __builtin_amdgcn_mov_dpp(lo, 0xFA, 0xF, 0xF, true), b1 = __builtin_amdgcn_mov_dpp(hi, 0xFA, 0xF, 0xF, true);
        a[i] = odd ? a1 : a0;  // lanes 0, 0, 1, 1
        b[i] = odd ? b1 : b0;  // lanes 2, 2, 3, 3
      }
      auto* to = reinterpret_cast<mx_i32x4_t*>(row + (col & ~31)) + (threadIdx.x & 3);
      __builtin_nontemporal_store(a, to);
      __builtin_nontemporal_store(b, to + 4);
      return;
    }
  }
  if (col < k) mx_store8<DT>(row + col, f, k - col);
}

// |x| as ordered bits: a NaN is above every number, so one integer maximum finds the largest value and what is not finite
__device__ __forceinline__ uint32_t mx_abs_bits8(const float (&f)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(f[i]) & 0x7fffffffu);
  return m;
}

// maximum over the 4 neighbouring lanes that hold one block (8 values each)
__device__ __forceinline__ uint32_t mx_quad_max(uint32_t m) {
  m = max(m, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(m), 0xB1, 0xF, 0xF, true)));  // lane ^ 1
  m = max(m, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(m), 0x4E, 0xF, 0xF, true)));  // lane ^ 2
  return m;
}

// scale code from the block's largest |x| (bits): exponent - 8 (e4m3) or - 2 (e2m1), one more where the significand is
// over the format's largest (1.75, 1.5)
template <int FMT>
__device__ __forceinline__ int mx_scale_code(uint32_t amax) {
  const int e = static_cast<int>(amax >> 23);
  const uint32_t m = amax & 0x7fffffu;
  const int code = FMT == MX_E4M3 ? e - 8 + (m > 0x600000u) : e - 2 + (m > 0x400000u);
  return e == 255 ? 255 : max(code, 0);
}

// 2^(127 - code); finite blocks have codes up to 247 (e4m3) or 253 (e2m1)
__device__ __forceinline__ float mx_inv_scale(int code) {
  return __uint_as_float(static_cast<uint32_t>(254 - code) << 23);
}

// 8 values -> 8 e4m3 bytes / 8 e2m1 halves of a byte (the conversions round to nearest even; nothing exceeds the format)
__device__ __forceinline__ uint2 mx_pack_e4m3(const float (&f)[8], int code) {
  const float s = mx_inv_scale(code);
  int a = 0, b = 0;
  a = __builtin_amdgcn_cvt_pk_fp8_f32(f[0] * s, f[1] * s, a, false);
  a = __builtin_amdgcn_cvt_pk_fp8_f32(f[2] * s, f[3] * s, a, true);
  b = __builtin_amdgcn_cvt_pk_fp8_f32(f[4] * s, f[5] * s, b, false);
  b = __builtin_amdgcn_cvt_pk_fp8_f32(f[6] * s, f[7] * s, b, true);
  return code == 255 ? make_uint2(0, 0) : make_uint2(a, b);
}
__device__ __forceinline__ uint32_t mx_pack_e2m1(const float (&f)[8], int code) {
  const float s = mx_inv_scale(code);
  uint32_t a = 0;
  a = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(a, f[0] * s, f[1] * s, 1.f, 0);
  a = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(a, f[2] * s, f[3] * s, 1.f, 1);
  a = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(a, f[4] * s, f[5] * s, 1.f, 2);
  a = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(a, f[6] * s, f[7] * s, 1.f, 3);
  return code == 255 ? 0u : a;
}
