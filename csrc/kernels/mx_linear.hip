// y = x . w^T + bias over MX operands (formats: mx.h): x e4m3 or e2m1, w e2m1, both [rows, k].
//
// gfx950's block-scaled matrix instructions take both formats and their scales as they lie in memory. The rows of w are
// the first operand and the rows of x the second, so a lane ends with four consecutive outputs of one row of x.
//
// v_mfma_scale_f32_32x32x64: D[32 x 32] += A[32 x 64] . B[32 x 64]^T, a scale for each row and block of 32 (measured):
//   lane l holds row l & 31; its 32 elements are k = 32 (l >> 5) .. + 31 of e2m1, and 16 (l >> 5) .. + 15 and
//   32 + 16 (l >> 5) .. + 15 of e4m3; its scale is that of block l >> 5 in both
//   of D it holds column l & 31 (a row of x), rows 8 (i >> 2) + 4 (l >> 5) + (i & 3), i = 0..15 (rows of w)
// Operands of registers alone run at 4.4 PFLOP/s with e4m3 on one side and 8.0 with e2m1 on both, whose 32 x 32 x 64
// form is twice as fast as the 16 x 16 x 128 one; hence the large tiles are made of it.
// The accumulators are 32 bits wide. Inside one instruction products of e2m1 are added exactly, products with e4m3 to some 17
// bits (measured: relative 5e-6 of normally distributed values): the unit's own width, which the 4.4 PFLOP/s come with. 16-bit
// results are as far from 64-bit ones as those of 32-bit sums (0.0017 in both for bf16, 4096 x 16384 x 8192), 32-bit results
// are not, so x in e4m3 has none.
#include <atomic>
#include <type_traits>

#include "conv_common.h"
#include "mx.h"

namespace {

typedef int i32x8_t __attribute__((ext_vector_type(8)));
typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef i32x4_t __attribute__((aligned(2))) Chunk16;  // 16 B of outputs: rows of odd n start at any element

// 16 B per lane from base + off to LDS at (wave-uniform lds + 16 * lane); completion is counted by vmcnt.
// M0 is put back: the compiler reserves it. PAST: past the caches, for what is read once.
template <bool PAST = false>
__device__ __forceinline__ void dma16(const void* base, uint32_t off, uint32_t lds) {
  uint32_t keep;
  if constexpr (PAST)
    asm volatile(
        "s_mov_b32 %0, m0\n\t"
        "s_mov_b32 m0, %3\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %1, %2 nt\n\t"
        "s_mov_b32 m0, %0"
        : "=&s"(keep)
        : "v"(off), "s"(base), "s"(lds)
        : "memory");
  else
    asm volatile(
        "s_mov_b32 %0, m0\n\t"
        "s_mov_b32 m0, %3\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %1, %2\n\t"
        "s_mov_b32 m0, %0"
        : "=&s"(keep)
        : "v"(off), "s"(base), "s"(lds)
        : "memory");
}

// Dynamic LDS over 64 KB is allowed per kernel and device, before its first launch there. `devices`: where it is.
bool allow_lds(const void* kernel, int bytes, std::atomic<uint64_t>& devices) {
  int d = 0;
  if (hipGetDevice(&d) != hipSuccess) return false;
  const uint64_t bit = 1ull << (d & 63);
  if (devices.load(std::memory_order_acquire) & bit) return true;
  if (hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess) return false;
  devices.fetch_or(bit, std::memory_order_release);
  return true;
}

// four consecutive outputs of a row, those below n
template <int DT>
__device__ __forceinline__ void store4(typename mx_elem<DT>::type* yr, int col, int n, const float* bias, const f32x4_t& v) {
  typedef typename mx_elem<DT>::type E;
  struct __attribute__((packed, aligned(sizeof(E)))) Four { E v[4]; } o;
  if (col + 4 <= n) {
#pragma unroll
    for (int p = 0; p < 4; ++p) o.v[p] = mx_elem<DT>::from(v[p] + (bias ? bias[col + p] : 0.f));
    *reinterpret_cast<Four*>(yr + col) = o;
  } else {
#pragma unroll
    for (int p = 0; p < 4; ++p)
      if (col + p < n) yr[col + p] = mx_elem<DT>::from(v[p] + (bias ? bias[col + p] : 0.f));
  }
}

// Rows of a tile in LDS, 128 elements each: 128 B (e4m3) or 64 B (e2m1). A DMA writes 1024 consecutive bytes, 8 or 16
// rows; the 16-B chunks of a row are permuted by the row so that the fragment reads of neighbouring rows fall into
// different banks, which is done by permuting the source addresses.
template <int FMT>
struct TileRow {
  static constexpr int BYTES = FMT == MX_E4M3 ? 128 : 64, CHUNKS = BYTES / 16, PER_DMA = 1024 / BYTES;
  static __device__ __forceinline__ int swizzle(int row) { return FMT == MX_E4M3 ? (row >> 1) & 7 : ai4e_conv::swz(row); }
};

// The tile kernel: BX x BW outputs per workgroup, WX x WW waves of TX x TW fragments of 32 x 32. Steps of 128 along k go
// through a ring of STAGES stages in LDS, written by DMA STAGES - 1 steps ahead; a barrier per step. Fragments are read half a
// step before the matrix instructions that take them. SHORT: for fewer than 4 steps, m and n at least 4.
template <int FX, int DT, int WX, int WW, int TX, int TW, int STAGES, bool SHORT>
__global__ __launch_bounds__(WX* WW * 64) void mx_tile_kernel(
    const uint8_t* __restrict__ x, const uint8_t* __restrict__ xs, const uint8_t* __restrict__ w,
    const uint8_t* __restrict__ ws, const float* __restrict__ bias, int m, int n, int kp, int tiles_x, int tiles_w,
    typename mx_elem<DT>::type* __restrict__ y) {
  constexpr int NW = WX * WW, BX = WX * TX * 32, BW = WW * TW * 32;
  typedef TileRow<FX> XR;
  typedef TileRow<MX_E2M1> WR;
  constexpr int X_BYTES = BX * XR::BYTES, W_BYTES = BW * WR::BYTES, S_BYTES = (BX + BW) * 16;
  constexpr int STAGE = X_BYTES + W_BYTES, SCALES = STAGE * STAGES;
  // DMAs per stage; the waves that a tile's DMAs do not divide among bring some twice
  constexpr int X_ALL = X_BYTES / 1024, W_ALL = W_BYTES / 1024, S_ALL = S_BYTES / 1024;
  constexpr int X_DMA = (X_ALL + NW - 1) / NW, W_DMA = (W_ALL + NW - 1) / NW, S_DMA = (S_ALL + NW - 1) / NW;
  constexpr int PER_STAGE = X_DMA + W_DMA;
  static_assert(X_BYTES % 1024 == 0 && W_BYTES % 1024 == 0 && S_BYTES % 1024 == 0, "");
  static_assert(SCALES + 2 * S_BYTES <= 160 * 1024 && STAGES >= 2 && STAGES <= 4, "");
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];

  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // neighbouring workgroups of one XCD take tiles of a block of 4 rows of tiles, which shares x and w in its L2
  const int t = xcd_remap(blockIdx.x, gridDim.x);
  constexpr int GROUP = 4;
  const int group = t / (GROUP * tiles_w), g0 = group * GROUP, gh = min(GROUP, tiles_x - g0);
  const int in = t - group * GROUP * tiles_w;
  const int x0 = (g0 + in % gh) * BX, w0 = (in / gh) * BW;

  const int px = FX == MX_E4M3 ? kp : kp / 2, pw = kp / 2, ps = kp / 32;  // row pitches in bytes
  uint32_t xoff[X_DMA], woff[W_DMA];
#pragma unroll
  for (int j = 0; j < X_DMA; ++j) {
    const int row = (wave * X_DMA + j) % X_ALL * XR::PER_DMA + lane / XR::CHUNKS;
    xoff[j] = static_cast<uint32_t>(min(row, m - 1 - x0)) * px + ((lane % XR::CHUNKS) ^ XR::swizzle(row)) * 16;
  }
#pragma unroll
  for (int j = 0; j < W_DMA; ++j) {
    const int row = (wave * W_DMA + j) % W_ALL * WR::PER_DMA + lane / WR::CHUNKS;
    woff[j] = static_cast<uint32_t>(min(row, n - 1 - w0)) * pw + ((lane % WR::CHUNKS) ^ WR::swizzle(row)) * 16;
  }
  uint32_t soff[S_DMA];  // a DMA brings the scales of 64 rows, first x's, then w's
#pragma unroll
  for (int j = 0; j < S_DMA; ++j) {
    const int p = (wave + j * NW) % S_ALL;
    soff[j] = static_cast<uint32_t>(p < BX / 64 ? min(p * 64 + lane, m - 1 - x0) : min(p * 64 - BX + lane, n - 1 - w0)) * ps;
    if (SHORT) {  // the 16 B from a row on pass its end; those of the last rows end with the tensor
      const int back = p < BX / 64 ? (x0 ? 16 : 0) : (w0 ? 16 : 0);
      soff[j] = back + min(static_cast<int>(soff[j]), min(p < BX / 64 ? m - x0 : n - w0, 1024) * ps - 16);
    }
  }
  const uint8_t* xb = x + static_cast<long>(x0) * px;
  const uint8_t* wb = w + static_cast<long>(w0) * pw;
  const uint8_t* xsb = xs + static_cast<long>(x0) * ps - (SHORT && x0 ? 16 : 0);
  const uint8_t* wsb = ws + static_cast<long>(w0) * ps - (SHORT && w0 ? 16 : 0);

  const int nk = kp / MX_ALIGN;
  // Where nobody else reads the same rows of w, each workgroup starts elsewhere along k: rows a power of two apart would
  // else have all workgroups in the same memory channels at once (64 x 32768 x 8192, weights out of memory: 41.0 us, so 38.8). Whole groups of scales.
  const int rot = tiles_x > 1 || nk % 4 ? 0 : w0 / BW * 5 * 4 % nk;
  auto place = [&](int k) { return k + rot < nk ? k + rot : k + rot - nk; };
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(
      (__attribute__((address_space(3))) uint8_t*)lds));
  // scales come 16 B of a row at a time, for 4 steps: as 4-B pieces they would be as many requests to L2 as the data
  // (measured: the rate of requests was what bound the kernel). Two slots; the last group ends with the row.
  auto scales = [&](int g) {
#pragma unroll
    for (int j = 0; j < S_DMA; ++j) {
      const int p = (wave + j * NW) % S_ALL;
      dma16((p < BX / 64 ? xsb : wsb) + (SHORT ? 0 : static_cast<long>(place(min(4 * g, nk - 4))) * 4), soff[j],
            lds0 + SCALES + (g & 1) * S_BYTES + p * 1024);
    }
  };
  // piece j of step kt; past the end the last step is brought again, into a slot that nobody reads
  auto issue = [&](int kt, uint32_t slot, int j) {
    const int k = place(min(kt, nk - 1));
    const uint32_t base = lds0 + slot * STAGE;
    if (j < X_DMA)
      dma16(xb + static_cast<long>(k) * XR::BYTES, xoff[j], base + (wave * X_DMA + j) % X_ALL * 1024);
    else
      dma16(wb + static_cast<long>(k) * WR::BYTES, woff[j - X_DMA], base + X_BYTES + (wave * W_DMA + j - X_DMA) % W_ALL * 1024);
  };

  const int wx = wave % WX, ww = wave / WX;
  const int r = lane & 31;
  const int xrow = wx * TX * 32 + r, wrow = ww * TW * 32 + r;
  const uint32_t xa = xrow * XR::BYTES + (half ^ XR::swizzle(xrow)) * 16;
  const uint32_t wa = X_BYTES + wrow * WR::BYTES + (half ^ WR::swizzle(wrow)) * 16;
  const uint32_t sa = r * 16;

  i32x8_t fx[2][TX], fw[2][TW];
  int sx[TX], sw[TW], nx[TX], nw[TW];
  typedef __attribute__((address_space(3))) const i32x4_t* Lds16;
  typedef __attribute__((address_space(3))) const int* Lds4;
  // piece p of the fragments of half step u of the stage at LDS address st: first w's, then x's (two per row of e4m3)
  constexpr int PIECES = TW + TX * XR::BYTES / 64;
  auto read = [&](uint32_t st, int u, int p) {
    if (p < TW) {
      const i32x4_t a = *reinterpret_cast<Lds16>(((st + wa) ^ (32 * u)) + p * 32 * WR::BYTES);
      fw[u][p] = __builtin_shufflevector(a, i32x4_t{}, 0, 1, 2, 3, 4, 5, 6, 7);
    } else if constexpr (FX == MX_E4M3) {
      const int i = (p - TW) / 2, hi = (p - TW) & 1;
      const i32x4_t a = *reinterpret_cast<Lds16>(((st + xa) ^ (64 * u + 32 * hi)) + i * 32 * XR::BYTES);
      fx[u][i] = hi ? __builtin_shufflevector(fx[u][i], __builtin_shufflevector(a, a, 0, 1, 2, 3, 0, 1, 2, 3), 0, 1, 2, 3, 8, 9, 10, 11)
                    : __builtin_shufflevector(a, i32x4_t{}, 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
      const int i = p - TW;
      const i32x4_t a = *reinterpret_cast<Lds16>(((st + xa) ^ (32 * u)) + i * 32 * XR::BYTES);
      fx[u][i] = __builtin_shufflevector(a, i32x4_t{}, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  };
  // a row's four scale bytes of step kt, shifted so that bytes 0 and 2 are those of this half's blocks
  auto late = [&](int row, int rows) {  // how much earlier than its row a piece of scales begins
    return SHORT ? max(0, 16 - (min(rows, 1024) - min(row, rows - 1)) * ps) : 0;
  };
  auto read_scales = [&](int kt, int(&ax)[TX], int(&aw)[TW]) {
    const uint32_t st = lds0 + SCALES + (SHORT ? kt * 4 : ((kt >> 2) & 1) * S_BYTES + (kt - min(kt & ~3, nk - 4)) * 4) + sa;
#pragma unroll
    for (int i = 0; i < TX; ++i) ax[i] = *reinterpret_cast<Lds4>(st + wx * TX * 512 + i * 512 + late(xrow + i * 32, m - x0));
#pragma unroll
    for (int j = 0; j < TW; ++j)
      aw[j] = *reinterpret_cast<Lds4>(st + BX * 16 + ww * TW * 512 + j * 512 + late(wrow + j * 32, n - w0));
  };
  auto shift_scales = [&]() {
#pragma unroll
    for (int i = 0; i < TX; ++i) sx[i] = nx[i] >> (8 * half);
#pragma unroll
    for (int j = 0; j < TW; ++j) sw[j] = nw[j] >> (8 * half);
  };
  f32x16_t acc[TX][TW] = {};
  constexpr int Q = TX * TW, READS = PIECES <= 2 * Q ? 2 : (PIECES + Q - 1) / Q;  // pieces read after each instruction
#define MX_MMA(U, N)                                                                                           \
  acc[(N) / TW][(N) % TW] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(                                   \
      fw[U][(N) % TW], fx[U][(N) / TW], acc[(N) / TW][(N) % TW], 4, FX == MX_E4M3 ? 0 : 4, 2 * U, sw[(N) % TW], \
      2 * U, sx[(N) / TW]);

#pragma unroll
  for (int s = 0; s < STAGES; ++s) {
    if (s == 0) scales(0);
#pragma unroll
    for (int j = 0; j < PER_STAGE; ++j) issue(s, s, j);
  }
  ai4e_conv::wait_vmcnt<(STAGES - 1) * PER_STAGE>();
  __builtin_amdgcn_s_barrier();
  read_scales(0, nx, nw);
#pragma unroll
  for (int p = 0; p < PIECES; ++p) read(lds0, 0, p);
  uint32_t slot = 0;
  // At step kt its first half's fragments and its scales are in registers. Reads and DMAs go out between the matrix
  // instructions, which keep their unit busy meanwhile; the order is fixed by scheduling barriers.
  for (int kt = 0; kt < nk; ++kt) {
    shift_scales();
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      MX_MMA(0, q)
#pragma unroll
      for (int p = READS * q; p < READS * (q + 1) && p < PIECES; ++p) read(lds0 + slot * STAGE, 1, p);
      __builtin_amdgcn_sched_barrier(0);
    }
    // this wave's part of step kt + 1 is there and it has read all of step kt: after the barrier step kt + 1 is
    // complete and step kt's slot free
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((STAGES - 2) * PER_STAGE) : "memory");
    __builtin_amdgcn_s_barrier();
    const uint32_t free = slot;
    slot = slot + 1 == STAGES ? 0 : slot + 1;
    if (!SHORT && ((kt + STAGES) & 3) == 0) scales((kt + STAGES) / 4);
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      MX_MMA(1, q)
      if (q == 0) read_scales(min(kt + 1, nk - 1), nx, nw);
#pragma unroll
      for (int p = READS * q; p < READS * (q + 1) && p < PIECES; ++p) read(lds0 + slot * STAGE, 0, p);
#pragma unroll
      for (int j = PER_STAGE * q / Q; j < PER_STAGE * (q + 1) / Q; ++j) issue(kt + STAGES, free, j);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  ai4e_conv::wait_vmcnt<0>();
#undef MX_MMA

  // The wave's outputs go through its own part of the idle ring, 32 rows at a time, so that stores fill whole lines:
  // straight from the accumulators they are 16-B pieces of 32 rows, whose requests took L2 longer than the data does
  // (4096 x 16384 x 8192: 55 of 414 us).
  __builtin_amdgcn_s_barrier();  // every wave has read its last fragments, every DMA has landed
  typedef typename mx_elem<DT>::type E;
  constexpr int COLS = TW * 32, CHUNK = 16 / sizeof(E), CHUNKS = COLS / CHUNK;  // 16-B chunks of a row of outputs
  static_assert(NW * 32 * COLS * sizeof(E) <= SCALES, "");
  uint8_t* mine = lds + wave * 32 * COLS * sizeof(E);
  const int c0 = w0 + ww * COLS;
#pragma unroll
  for (int i = 0; i < TX; ++i) {
#pragma unroll
    for (int j = 0; j < TW; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int col = j * 32 + 8 * q + 4 * half;
        typedef int Four __attribute__((ext_vector_type(sizeof(E))));  // 4 outputs
        struct { E v[4]; } o;
#pragma unroll
        for (int p = 0; p < 4; ++p)
          o.v[p] = mx_elem<DT>::from(acc[i][j][4 * q + p] + (bias && c0 + col + p < n ? bias[c0 + col + p] : 0.f));
        const int chunk = (col / CHUNK) ^ (r & (CHUNKS - 1));
        *reinterpret_cast<Four*>(mine + (r * CHUNKS + chunk) * 16 + col % CHUNK * sizeof(E)) = __builtin_bit_cast(Four, o);
      }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int it = 0; it < 32 * CHUNKS / 64; ++it) {
      const int rr = (it * 64 + lane) / CHUNKS, ch = (it * 64 + lane) % CHUNKS;
      const int row = x0 + (wx * TX + i) * 32 + rr, col = c0 + ch * CHUNK;
      struct Chunk { E v[CHUNK]; };
      const Chunk o = __builtin_bit_cast(
          Chunk, *reinterpret_cast<const i32x4_t*>(mine + (rr * CHUNKS + (ch ^ (rr & (CHUNKS - 1)))) * 16));
      if (row < m) {
        E* to = y + static_cast<long>(row) * n + col;
        if (col + CHUNK <= n) {
          // past L2: the outputs would push x and w out of it
          __builtin_nontemporal_store(__builtin_bit_cast(Chunk16, o), reinterpret_cast<Chunk16*>(to));
        } else {
#pragma unroll
          for (int p = 0; p < CHUNK; ++p)
            if (col + p < n) to[p] = o.v[p];
        }
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

template <int FX, int DT, int WX, int WW, int TX, int TW, int STAGES, bool SHORT = false>
int launch_tile(const void* x, const void* xs, const void* w, const void* ws, const void* bias, int m, int n, int kp, void* y,
                hipStream_t s) {
  constexpr int BX = WX * TX * 32, BW = WW * TW * 32;
  constexpr int LDS = STAGES * (BX * TileRow<FX>::BYTES + BW * TileRow<MX_E2M1>::BYTES) +
                      2 * (BX + BW) * 16;
  const int tx = ai4e_cdiv(m, BX), tw = ai4e_cdiv(n, BW);
  auto* kernel = mx_tile_kernel<FX, DT, WX, WW, TX, TW, STAGES, SHORT>;
  static std::atomic<uint64_t> devices{0};
  if (!allow_lds(reinterpret_cast<const void*>(kernel), LDS, devices)) return AI4E_ELAUNCH;
  hipLaunchKernelGGL(kernel, dim3(tx * tw), dim3(WX * WW * 64), LDS, s, static_cast<const uint8_t*>(x),
                     static_cast<const uint8_t*>(xs), static_cast<const uint8_t*>(w), static_cast<const uint8_t*>(ws),
                     static_cast<const float*>(bias), m, n, kp, tx, tw, static_cast<typename mx_elem<DT>::type*>(y));
  return hipGetLastError() == hipSuccess ? AI4E_OK : AI4E_ELAUNCH;
}

// The few-rows kernel: up to 32 rows of x by 128 rows of w (at least as many) per workgroup of 4 waves, a fragment of 32 x 32 each. What
// bounds it is how w comes out of memory: a DMA brings 256 consecutive bytes of 4 rows, four steps of k, since pieces of one
// step (64 B) of many rows take longer (16 x 32768 x 8192 31.5 us, so 30.2), and past the caches, since a model's weights come by
// once per token (26.9; weights that a cache still holds 25.5 us, through it 24.0). Such groups of four steps go through a
// ring of three, two of them in flight, a barrier per group, from one tile of a workgroup to its next.
template <int FX, int DT>
struct FewLds {
  static constexpr int X_ROW = 4 * TileRow<FX>::BYTES, W_ROW = 4 * TileRow<MX_E2M1>::BYTES;  // bytes of a row of a group
  static constexpr int X_BYTES = 32 * X_ROW, W_BYTES = 128 * W_ROW, S_BYTES = (64 + 128) * 16;
  static constexpr int GROUP = X_BYTES + W_BYTES + S_BYTES, RING = 3, ALL = RING * GROUP;
  static_assert(ALL <= 160 * 1024, "");
};

template <int FX, int DT>
__global__ __launch_bounds__(256) void mx_few_kernel(
    const uint8_t* __restrict__ x, const uint8_t* __restrict__ xs, const uint8_t* __restrict__ w,
    const uint8_t* __restrict__ ws, const float* __restrict__ bias, int m, int n, int kp, int tiles,
    typename mx_elem<DT>::type* __restrict__ y) {
  typedef FewLds<FX, DT> S;
  constexpr int X_DMA = S::X_BYTES / 1024 / 4, W_DMA = S::W_BYTES / 1024 / 4, PER_GROUP = X_DMA + W_DMA + 1;
  constexpr int X_CHUNKS = S::X_ROW / 16, W_CHUNKS = S::W_ROW / 16;  // of 16 B; stored at their place ^ (row & 15)
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  const int lane = threadIdx.x & 63, half = lane >> 5, r = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int px = FX == MX_E4M3 ? kp : kp / 2, pw = kp / 2, ps = kp / 32;
  uint32_t xoff[X_DMA], woff[W_DMA];
#pragma unroll
  for (int j = 0; j < X_DMA; ++j) {
    const int row = ((wave * X_DMA + j) * 64 + lane) / X_CHUNKS;
    xoff[j] = static_cast<uint32_t>(min(row, m - 1)) * px + ((lane % X_CHUNKS) ^ (row & 15)) * 16;
  }
#pragma unroll
  for (int j = 0; j < W_DMA; ++j) {
    const int row = ((wave * W_DMA + j) * 64 + lane) / W_CHUNKS;
    woff[j] = static_cast<uint32_t>(row) * pw + ((lane % W_CHUNKS) ^ (row & 15)) * 16;
  }
  // scales of 64 rows per DMA: w's two halves, x's rows, and those once more
  const uint32_t soff = static_cast<uint32_t>(wave < 2 ? wave * 64 + lane : min(lane, m - 1)) * ps;
  const uint32_t sto = S::X_BYTES + S::W_BYTES + (wave < 2 ? wave : 2) * 1024;

  // the workgroup's tiles one after the other, all the groups of each; a workgroup's first group lies elsewhere along k
  // than its neighbours', since rows a power of two apart would else be in the same memory channels at once
  const int nk = kp / MX_ALIGN, groups = (nk + 3) / 4;
  const int mine = (tiles - static_cast<int>(blockIdx.x) + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x);
  struct Place {
    int tile, group;
  };
  const int rot = blockIdx.x * 5 % groups;
  Place next = {0, 0}, now = {0, 0};  // the group to fetch, the group at work: tile of this workgroup, turn in the tile
  auto advance = [&](Place& p) {
    if (++p.group == groups) {
      p.group = 0;
      ++p.tile;
    }
  };
  auto place = [&](const Place& p) { return p.group + rot < groups ? p.group + rot : p.group + rot - groups; };
  // a tile's first row of w: n is at least 128, and the last tile ends with w
  auto start = [&](int t) { return min(static_cast<int>(blockIdx.x + t * gridDim.x) * 128, n - 128); };
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(
      (__attribute__((address_space(3))) uint8_t*)lds));
  auto issue = [&](uint32_t slot) {  // past the end the last tile's groups are brought again, into slots that nobody reads
    const int k = __builtin_amdgcn_readfirstlane(min(4 * place(next), nk - 4));  // the last group ends with the row
    const int w0 = start(min(next.tile, mine - 1));
    advance(next);
    const uint32_t base = lds0 + slot * S::GROUP;
    dma16((wave < 2 ? ws + static_cast<long>(w0) * ps : xs) + k * 4l, soff, base + sto);
    const uint8_t* wb = w + static_cast<long>(w0) * pw + k * 64l;
#pragma unroll
    for (int j = 0; j < W_DMA; ++j) dma16<true>(wb, woff[j], base + S::X_BYTES + (wave * W_DMA + j) * 1024);
#pragma unroll
    for (int j = 0; j < X_DMA; ++j)
      dma16(x + k * static_cast<long>(TileRow<FX>::BYTES), xoff[j], base + (wave * X_DMA + j) * 1024);
  };
  typedef __attribute__((address_space(3))) const i32x4_t* Lds16;
  typedef __attribute__((address_space(3))) const int* Lds4;
  const uint32_t xa = r * S::X_ROW, wa = S::X_BYTES + (wave * 32 + r) * S::W_ROW;
  const uint32_t sa = S::X_BYTES + S::W_BYTES + (wave * 32 + r) * 16;
  f32x16_t acc = {};
  issue(0);
  issue(1);
  uint32_t slot = 0;
  while (now.tile < mine) {
    // this wave's part of the group is there and it has read all of the last one: after the barrier the group is complete
    // and the last one's slot free
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(PER_GROUP) : "memory");
    __builtin_amdgcn_s_barrier();
    issue(slot == 0 ? 2 : slot - 1);
    const uint32_t st = lds0 + slot * S::GROUP;
    const int p0 = max(0, 4 * place(now) - (nk - 4));  // steps that the last group shares with the one before it
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      if (p < p0) continue;
      const int sw = *reinterpret_cast<Lds4>(st + sa + p * 4) >> (8 * half);
      const int sx = *reinterpret_cast<Lds4>(st + S::X_BYTES + S::W_BYTES + 2048 + r * 16 + p * 4) >> (8 * half);
      i32x8_t fx[2], fw[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const i32x4_t a = *reinterpret_cast<Lds16>(st + wa + ((4 * p + 2 * u + half) ^ (r & 15)) * 16);
        fw[u] = __builtin_shufflevector(a, i32x4_t{}, 0, 1, 2, 3, 4, 5, 6, 7);
        if constexpr (FX == MX_E4M3) {
          const i32x4_t b = *reinterpret_cast<Lds16>(st + xa + ((8 * p + 4 * u + half) ^ (r & 15)) * 16);
          const i32x4_t c = *reinterpret_cast<Lds16>(st + xa + ((8 * p + 4 * u + 2 + half) ^ (r & 15)) * 16);
          fx[u] = __builtin_shufflevector(b, c, 0, 1, 2, 3, 4, 5, 6, 7);
        } else {
          const i32x4_t b = *reinterpret_cast<Lds16>(st + xa + ((4 * p + 2 * u + half) ^ (r & 15)) * 16);
          fx[u] = __builtin_shufflevector(b, i32x4_t{}, 0, 1, 2, 3, 4, 5, 6, 7);
        }
      }
      acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fw[0], fx[0], acc, 4, FX == MX_E4M3 ? 0 : 4, 0, sw, 0, sx);
      acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fw[1], fx[1], acc, 4, FX == MX_E4M3 ? 0 : 4, 2, sw, 2, sx);
    }
    slot = slot == 2 ? 0 : slot + 1;
    if (now.group == groups - 1) {
      const int w0 = start(now.tile) + wave * 32, from = (blockIdx.x + now.tile * gridDim.x) * 128;
      if (r < m)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int col = w0 + 8 * q + 4 * half;
          const f32x4_t v = {acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]};
          if (col >= from) {
            store4<DT>(y + static_cast<long>(r) * n, col, n, bias, v);
          } else {  // columns below `from` are the tile's before this one
#pragma unroll
            for (int p = 0; p < 4; ++p)
              if (col + p >= from) y[static_cast<long>(r) * n + col + p] = mx_elem<DT>::from(v[p] + (bias ? bias[col + p] : 0.f));
          }
        }
      acc = f32x16_t{};
    }
    advance(now);
  }
  ai4e_conv::wait_vmcnt<0>();  // the ring is the workgroup's until the last DMA has landed
}

template <int FX, int DT>
int launch_few(const void* x, const void* xs, const void* w, const void* ws, const void* bias, int m, int n, int kp, void* y,
               hipStream_t s) {
  constexpr int LDS = FewLds<FX, DT>::ALL;
  auto* kernel = mx_few_kernel<FX, DT>;
  static std::atomic<uint64_t> devices{0};
  if (!allow_lds(reinterpret_cast<const void*>(kernel), LDS, devices)) return AI4E_ELAUNCH;
  const int tiles = ai4e_cdiv(n, 128);
  hipLaunchKernelGGL(kernel, dim3(tiles < 256 ? tiles : 256), dim3(256), LDS, s, static_cast<const uint8_t*>(x),
                     static_cast<const uint8_t*>(xs), static_cast<const uint8_t*>(w), static_cast<const uint8_t*>(ws),
                     static_cast<const float*>(bias), m, n, kp, tiles, static_cast<typename mx_elem<DT>::type*>(y));
  return hipGetLastError() == hipSuccess ? AI4E_OK : AI4E_ELAUNCH;
}

// The slice kernel: 16 MT rows of x by 16 NT rows of w per workgroup, k cut over its 8 waves: for the fewest rows, where
// latency counts, and for k below 512. Operands go from memory to registers, in steps of v_mfma_scale_f32_16x16x128: lane l
// holds row l & 15, k = 32 (l >> 4) .. + 31 of e2m1, 16 (l >> 4) .. + 15 and 64 + 16 (l >> 4) .. + 15 of e4m3, the scale
// of block l >> 4; of D column l & 15, rows 4 (l >> 4) + i. Four steps' loads go out together, their scales as one 16-B
// load per row. The waves' sums are added in LDS, always in the same order.
constexpr int SLICES = 8;

template <int FX, int DT, int MT, int NT>
__global__ __launch_bounds__(SLICES * 64) void mx_slice_kernel(
    const uint8_t* __restrict__ x, const uint8_t* __restrict__ xs, const uint8_t* __restrict__ w,
    const uint8_t* __restrict__ ws, const float* __restrict__ bias, int m, int n, int kp, int tiles_m,
    typename mx_elem<DT>::type* __restrict__ y) {
  __shared__ f32x4_t part[SLICES][MT * NT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4;
  const int t = xcd_remap(blockIdx.x, gridDim.x);  // the row blocks of one w block follow each other: its L2 serves them
  const int m0 = (t % tiles_m) * 16 * MT, n0 = (t / tiles_m) * 16 * NT;
  const int nk = kp / MX_ALIGN, k0 = nk * wave / SLICES, k1 = nk * (wave + 1) / SLICES;
  const long px = FX == MX_E4M3 ? kp : kp / 2, pw = kp / 2, ps = kp / 32;
  const uint8_t *xr[MT], *xsr[MT], *wr[NT], *wsr[NT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int row = min(m0 + 16 * i + (lane & 15), m - 1);
    xr[i] = x + row * px + 16 * g;
    xsr[i] = xs + row * ps;
  }
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int row = min(n0 + 16 * j + (lane & 15), n - 1);
    wr[j] = w + row * pw + 16 * g;
    wsr[j] = ws + row * ps;
  }
  f32x4_t acc[MT][NT] = {};
  auto steps = [&](int kt, auto count) {
    constexpr int S = decltype(count)::value;
    struct __attribute__((packed, aligned(4))) Scales { int v[S]; };
    Scales sx[MT], sw[NT];
    i32x4_t b[NT][S], a0[MT][S], a1[MT][S];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      sw[j] = *reinterpret_cast<const Scales*>(wsr[j] + kt * 4);
#pragma unroll
      for (int s = 0; s < S; ++s) b[j][s] = *reinterpret_cast<const i32x4_t*>(wr[j] + (kt + s) * 64l);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      sx[i] = *reinterpret_cast<const Scales*>(xsr[i] + kt * 4);
#pragma unroll
      for (int s = 0; s < S; ++s) {
        a0[i][s] = *reinterpret_cast<const i32x4_t*>(xr[i] + (kt + s) * static_cast<long>(TileRow<FX>::BYTES));
        if constexpr (FX == MX_E4M3) a1[i][s] = *reinterpret_cast<const i32x4_t*>(xr[i] + (kt + s) * 128l + 64);
        else a1[i][s] = i32x4_t{};
      }
    }
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < MT; ++i)
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
              __builtin_shufflevector(b[j][s], i32x4_t{}, 0, 1, 2, 3, 4, 5, 6, 7),
              __builtin_shufflevector(a0[i][s], a1[i][s], 0, 1, 2, 3, 4, 5, 6, 7), acc[i][j], 4, FX == MX_E4M3 ? 0 : 4, 0,
              sw[j].v[s] >> (8 * g), 0, sx[i].v[s] >> (8 * g));
  };
  int kt = k0;
  for (; kt + 4 <= k1; kt += 4) steps(kt, std::integral_constant<int, 4>{});
  for (; kt < k1; ++kt) steps(kt, std::integral_constant<int, 1>{});
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) part[wave][i * NT + j][lane] = acc[i][j];
  __syncthreads();
  for (int f = wave; f < MT * NT; f += SLICES) {
    f32x4_t v = part[0][f][lane];
#pragma unroll
    for (int p = 1; p < SLICES; ++p) v += part[p][f][lane];
    const int row = m0 + 16 * (f / NT) + (lane & 15), col = n0 + 16 * (f % NT) + 4 * g;
    if (row < m) store4<DT>(y + static_cast<long>(row) * n, col, n, bias, v);
  }
}

template <int FX, int DT, int MT, int NT>
int launch_slice(const void* x, const void* xs, const void* w, const void* ws, const void* bias, int m, int n, int kp, void* y,
                 hipStream_t s) {
  const int tm = ai4e_cdiv(m, 16 * MT);
  hipLaunchKernelGGL((mx_slice_kernel<FX, DT, MT, NT>), dim3(tm * ai4e_cdiv(n, 16 * NT)), dim3(SLICES * 64), 0, s,
                     static_cast<const uint8_t*>(x), static_cast<const uint8_t*>(xs), static_cast<const uint8_t*>(w),
                     static_cast<const uint8_t*>(ws), static_cast<const float*>(bias), m, n, kp, tm,
                     static_cast<typename mx_elem<DT>::type*>(y));
  return hipGetLastError() == hipSuccess ? AI4E_OK : AI4E_ELAUNCH;
}

// The stream kernel: 32 rows of x by 32 TW rows of w per workgroup, k cut over its 4 waves, each of which runs its steps
// through a ring of its own in LDS: no barrier until the waves' sums are added, always in the same order. For outputs
// too few to give every CU a tile of 64 x 64, whose single workgroup would wait out every step's latency (333 x 5000 x
// 1000: 12.9 us, so 8.2).
constexpr int STREAMS = 4;

template <int FX, int TW, int STAGES>
struct StreamLds {
  static constexpr int X_BYTES = 32 * TileRow<FX>::BYTES, W_BYTES = 32 * TW * TileRow<MX_E2M1>::BYTES;
  static constexpr int S_ROWS = (32 + 32 * TW + 63) / 64 * 64, S_BYTES = S_ROWS * 16;  // 4 steps' scales: x's rows, w's
  static constexpr int STAGE = X_BYTES + W_BYTES, SCALES = STAGES * STAGE, WAVE = SCALES + 2 * S_BYTES;
  static constexpr int SUMS = STREAMS * TW * 16 * 64 * 4;
  static constexpr int ALL = STREAMS * WAVE > SUMS ? STREAMS * WAVE : SUMS;
  static_assert(STAGES >= 2 && STAGES <= 4 && ALL <= 160 * 1024 && WAVE % 128 == 0, "");
};

template <int FX, int DT, int TW, int STAGES>
__global__ __launch_bounds__(STREAMS * 64) void mx_stream_kernel(
    const uint8_t* __restrict__ x, const uint8_t* __restrict__ xs, const uint8_t* __restrict__ w,
    const uint8_t* __restrict__ ws, const float* __restrict__ bias, int m, int n, int kp, int tiles_x,
    typename mx_elem<DT>::type* __restrict__ y) {
  typedef TileRow<FX> XR;
  typedef TileRow<MX_E2M1> WR;
  typedef StreamLds<FX, TW, STAGES> S;
  constexpr int BW = TW * 32, S_DMA = S::S_ROWS / 64, X_DMA = S::X_BYTES / 1024, W_DMA = S::W_BYTES / 1024;
  constexpr int PER_STAGE = X_DMA + W_DMA;
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  const int lane = threadIdx.x & 63, half = lane >> 5, r = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int t = xcd_remap(blockIdx.x, gridDim.x);  // the row blocks of one w block follow each other: its L2 serves them
  const int x0 = t % tiles_x * 32, w0 = t / tiles_x * BW;
  const int px = FX == MX_E4M3 ? kp : kp / 2, pw = kp / 2, ps = kp / 32;
  uint32_t xoff[X_DMA], woff[W_DMA];
#pragma unroll
  for (int j = 0; j < X_DMA; ++j) {
    const int row = j * XR::PER_DMA + lane / XR::CHUNKS;
    xoff[j] = static_cast<uint32_t>(min(row, m - 1 - x0)) * px + ((lane % XR::CHUNKS) ^ XR::swizzle(row)) * 16;
  }
#pragma unroll
  for (int j = 0; j < W_DMA; ++j) {
    const int row = j * WR::PER_DMA + lane / WR::CHUNKS;
    woff[j] = static_cast<uint32_t>(min(row, n - 1 - w0)) * pw + ((lane % WR::CHUNKS) ^ WR::swizzle(row)) * 16;
  }
  const uint8_t* xb = x + static_cast<long>(x0) * px;
  const uint8_t* wb = w + static_cast<long>(w0) * pw;
  const uint8_t* sp[S_DMA];
#pragma unroll
  for (int j = 0; j < S_DMA; ++j) {
    const int p = j * 64 + lane;
    sp[j] = p < 32 ? xs + static_cast<long>(min(x0 + p, m - 1)) * ps
                   : ws + static_cast<long>(min(w0 + min(p - 32, BW - 1), n - 1)) * ps;
  }
  // whole groups of 4 steps per wave; the last group's scales end with the row
  const int nk = kp / MX_ALIGN, groups = (nk + 3) / 4;
  const int k0 = groups * wave / STREAMS * 4, k1 = min(groups * (wave + 1) / STREAMS * 4, nk);
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(
      (__attribute__((address_space(3))) uint8_t*)lds)) + wave * S::WAVE;
  // step kt into a slot; past the wave's end its last step is brought again, into a slot that nobody reads
  auto issue = [&](int kt, uint32_t slot) {
    const int k = __builtin_amdgcn_readfirstlane(min(kt, k1 - 1));
    const uint32_t base = lds0 + slot * S::STAGE;
    if ((kt & 3) == 0) {
      const long at = min(k & ~3, nk - 4) * 4l;
#pragma unroll
      for (int j = 0; j < S_DMA; ++j)
        ai4e_conv::glds16(sp[j] + at, lds0 + S::SCALES + ((kt >> 2) & 1) * S::S_BYTES + j * 1024);
    }
#pragma unroll
    for (int j = 0; j < X_DMA; ++j) dma16(xb + static_cast<long>(k) * XR::BYTES, xoff[j], base + j * 1024);
#pragma unroll
    for (int j = 0; j < W_DMA; ++j) dma16(wb + static_cast<long>(k) * WR::BYTES, woff[j], base + S::X_BYTES + j * 1024);
  };
  const uint32_t xa = r * XR::BYTES + (half ^ XR::swizzle(r)) * 16;
  const uint32_t wa = S::X_BYTES + r * WR::BYTES + (half ^ WR::swizzle(r)) * 16;
  typedef __attribute__((address_space(3))) const i32x4_t* Lds16;
  typedef __attribute__((address_space(3))) const int* Lds4;
  f32x16_t acc[TW] = {};
  if (k0 < k1) {
#pragma unroll
    for (int s = 0; s < STAGES; ++s) issue(k0 + s, s);
    uint32_t slot = 0;
    for (int kt = k0; kt < k1; ++kt) {
      ai4e_conv::wait_vmcnt<(STAGES - 1) * PER_STAGE>();  // step kt is there, and its scales, which went out before it
      const uint32_t st = lds0 + slot * S::STAGE;
      const uint32_t sa = lds0 + S::SCALES + ((kt >> 2) & 1) * S::S_BYTES + (kt - min(kt & ~3, nk - 4)) * 4 + r * 16;
      i32x8_t fx[2], fw[2][TW];
      int sw[TW];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if constexpr (FX == MX_E4M3) {
          const i32x4_t a = *reinterpret_cast<Lds16>((st + xa) ^ (64 * u));
          const i32x4_t b = *reinterpret_cast<Lds16>((st + xa) ^ (64 * u + 32));
          fx[u] = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        } else {
          const i32x4_t a = *reinterpret_cast<Lds16>((st + xa) ^ (32 * u));
          fx[u] = __builtin_shufflevector(a, i32x4_t{}, 0, 1, 2, 3, 4, 5, 6, 7);
        }
#pragma unroll
        for (int j = 0; j < TW; ++j) {
          const i32x4_t a = *reinterpret_cast<Lds16>(((st + wa) ^ (32 * u)) + j * 32 * WR::BYTES);
          fw[u][j] = __builtin_shufflevector(a, i32x4_t{}, 0, 1, 2, 3, 4, 5, 6, 7);
        }
      }
      const int sx = *reinterpret_cast<Lds4>(sa) >> (8 * half);
#pragma unroll
      for (int j = 0; j < TW; ++j) sw[j] = *reinterpret_cast<Lds4>(sa + (1 + j) * 512) >> (8 * half);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the slot has been read
      issue(kt + STAGES, slot);
      slot = slot + 1 == STAGES ? 0 : slot + 1;
#pragma unroll
      for (int j = 0; j < TW; ++j)
        acc[j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fw[0][j], fx[0], acc[j], 4, FX == MX_E4M3 ? 0 : 4, 0,
                                                                 sw[j], 0, sx);
#pragma unroll
      for (int j = 0; j < TW; ++j)
        acc[j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fw[1][j], fx[1], acc[j], 4, FX == MX_E4M3 ? 0 : 4, 2,
                                                                 sw[j], 2, sx);
    }
    ai4e_conv::wait_vmcnt<0>();
  }
  __syncthreads();  // every wave is through with its ring
  f32x4_t* part = reinterpret_cast<f32x4_t*>(lds);  // [wave][TW][4][lane]
#pragma unroll
  for (int j = 0; j < TW; ++j)
#pragma unroll
    for (int q = 0; q < 4; ++q)
      part[((wave * TW + j) * 4 + q) * 64 + lane] =
          f32x4_t{acc[j][4 * q], acc[j][4 * q + 1], acc[j][4 * q + 2], acc[j][4 * q + 3]};
  __syncthreads();
  for (int f = wave; f < TW * 4; f += STREAMS) {
    f32x4_t v = part[f * 64 + lane];
#pragma unroll
    for (int p = 1; p < STREAMS; ++p) v += part[(p * TW * 4 + f) * 64 + lane];
    const int row = x0 + r;
    if (row < m) store4<DT>(y + static_cast<long>(row) * n, w0 + f / 4 * 32 + 8 * (f % 4) + 4 * half, n, bias, v);
  }
}

template <int FX, int DT, int TW, int STAGES>
int launch_stream(const void* x, const void* xs, const void* w, const void* ws, const void* bias, int m, int n, int kp, void* y,
                  hipStream_t s) {
  constexpr int LDS = StreamLds<FX, TW, STAGES>::ALL;
  const int tx = ai4e_cdiv(m, 32), tw = ai4e_cdiv(n, 32 * TW);
  auto* kernel = mx_stream_kernel<FX, DT, TW, STAGES>;
  static std::atomic<uint64_t> devices{0};
  if (!allow_lds(reinterpret_cast<const void*>(kernel), LDS, devices)) return AI4E_ELAUNCH;
  hipLaunchKernelGGL(kernel, dim3(tx * tw), dim3(STREAMS * 64), LDS, s, static_cast<const uint8_t*>(x),
                     static_cast<const uint8_t*>(xs), static_cast<const uint8_t*>(w), static_cast<const uint8_t*>(ws),
                     static_cast<const float*>(bias), m, n, kp, tx, static_cast<typename mx_elem<DT>::type*>(y));
  return hipGetLastError() == hipSuccess ? AI4E_OK : AI4E_ELAUNCH;
}

// Which kernel: the largest tile that still gives most of the 256 CUs one, since a larger tile moves fewer bytes per
// product; where even 64 x 64 does not, the streams that need one round of workgroups, and for the fewest rows slices.
// Measured at the borders (us, e4m3; the first kernel's time first; weights from memory where a row names 16 rows of x,
// else from the memory-side cache):
//   256 x 256 / 128 x 128   1024 x 8192 x 8192 (128 / 512 tiles) 77.7 / 61.8    4096 x 4096 x 4096 (256 / 1024) 55 / 70
//   128 x 128 / 64 x 128    512 x 4096 x 4096 (128 / 256 tiles) 17.6 / 12.5     512 x 8192 x 8192 (256 / 512) 38.5 / 45.0
//   64 x 128 / 64 x 64      256 x 4096 x 4096 (128 / 256 tiles) 12.5 / 10.9     256 x 8192 x 8192 (256 / 512) 26.4 / 33.0
//   64 x 64 / stream 2      128 x 4096 x 4096 (128 / 256) 10.6 / 7.8            200 x 3000 x 4096 (188 / 329) 11.0 / 11.4
//   few rows / stream 2     16 x 20480 x 4096 (160 / 320) 14.9 / 17.9           16 x 16384 x 4096 (128 / 256) 13.4 / 11.0
//   stream 2 / stream 1     64 x 6144 x 4096 (192 / 384) 9.6 / 11.4             64 x 4096 x 4096 (128 / 256) 7.3 / 6.1
//   stream 1 / slices       1 x 4096 x 4096 5.6 / 4.4                           16 x 4096 x 4096 5.7 / 5.9
// and with k below 512, where latency counts more than bytes do:
//   128 x 128 / 64 x 64     4096 x 16384 x 384 (4096 / 16384 tiles) 52 / 65     1024 x 4096 x 384 (256 / 1024) 7.1 / 6.2
//   64 x 64 / slices        64 x 16384 x 384 (256 / 512) 3.9 / 5.7              4096 x 16384 x 384 65 / 286
template <int FX, int DT>
int launch(const void* x, const void* xs, const void* w, const void* ws, const void* bias, int m, int n, int kp, void* y,
           hipStream_t s) {
#define ARGS x, xs, w, ws, bias, m, n, kp, y, s
  const auto blocks = [&](int bm, int bn) { return static_cast<long>(ai4e_cdiv(m, bm)) * ai4e_cdiv(n, bn); };
  constexpr long FILL = 192, ROUND = 320;
  if (kp < 512) {  // the others' scales come four steps of 128 at a time
    if (m > 64 && n >= 4 && blocks(128, 128) >= 4 * 256) return launch_tile<FX, DT, 2, 2, 2, 2, 2, true>(ARGS);
    if (m > 32 && n >= 4 && blocks(64, 64) >= FILL) return launch_tile<FX, DT, 2, 2, 1, 1, 2, true>(ARGS);
    return blocks(16, 16) <= ROUND ? launch_slice<FX, DT, 1, 1>(ARGS) : launch_slice<FX, DT, 2, 4>(ARGS);
  }
  if (m <= 8 && blocks(16, 16) <= ROUND) return launch_slice<FX, DT, 1, 1>(ARGS);
  if (m > 128 && blocks(256, 256) >= FILL) return launch_tile<FX, DT, 4, 2, 2, 4, FX == MX_E4M3 ? 3 : 4>(ARGS);
  if (m > 64 && blocks(128, 128) >= FILL) return launch_tile<FX, DT, 2, 2, 2, 2, FX == MX_E4M3 ? 3 : 4>(ARGS);
  if (m > 32 && blocks(64, 128) >= FILL) return launch_tile<FX, DT, 2, 2, 1, 2, 4>(ARGS);
  if (m > 32 && blocks(64, 64) >= FILL) return launch_tile<FX, DT, 2, 2, 1, 1, 4>(ARGS);
  if (blocks(32, 32) <= ROUND) return launch_stream<FX, DT, 1, 2>(ARGS);
  if (blocks(32, 64) <= (m > 32 ? ROUND : 256)) return launch_stream<FX, DT, 2, 2>(ARGS);
  return m <= 32 ? launch_few<FX, DT>(ARGS) : launch_tile<FX, DT, 2, 2, 1, 1, 4>(ARGS);
#undef ARGS
}

// What a launch of fewer than 2^32 threads holds: 2^22 tiles of 128 x 128; of slices (`launch`: short k, few rows or
// outputs) fewer than 2^23 of 32 x 64.
bool fits(int m, int n, int kp) {
  const auto blocks = [&](int bm, int bn) { return static_cast<long>(ai4e_cdiv(m, bm)) * ai4e_cdiv(n, bn); };
  return kp <= (1 << 23) && n <= (1 << 30) && m <= (1 << 30) && blocks(128, 128) <= (1L << 22) &&
         (kp >= 512 || (m > 32 && n >= 4) || blocks(32, 64) < (1L << 23));
}

}  // namespace

// x: data [m, kp] (fx 0, e4m3) or [m, kp / 2] (fx 1, e2m1), xs [m, kp / 32]; w: [n, kp / 2], ws [n, kp / 32];
// bias [n] fp32 or null; y [m, n] of type dt (0 bf16, 1 fp16, 2 fp32: of e2m1 x only). kp is a multiple of 128.
AI4E_API int ai4e_mx_linear(const void* x, const void* xs, int fx, const void* w, const void* ws, const void* bias,
                            int m, int n, int kp, void* y, int dt, hipStream_t s) {
  if (m < 0 || n <= 0 || kp <= 0 || kp % MX_ALIGN || fx < 0 || fx > 1 || dt < 0 || dt > 2 ||
      (fx == MX_E4M3 && dt == MX_F32) || !fits(m, n, kp))
    return AI4E_EINVAL;
  if (m == 0) return AI4E_OK;  // tensors without elements have no memory
  if (!x || !xs || !w || !ws || !y) return AI4E_EINVAL;
#define GO(FX, DT) return launch<FX, DT>(x, xs, w, ws, bias, m, n, kp, y, s)
  if (fx == MX_E4M3) {
    if (dt == MX_BF16) GO(MX_E4M3, MX_BF16);
    GO(MX_E4M3, MX_F16);
  }
  if (dt == MX_BF16) GO(MX_E2M1, MX_BF16);
  if (dt == MX_F16) GO(MX_E2M1, MX_F16);
  GO(MX_E2M1, MX_F32);
#undef GO
}
