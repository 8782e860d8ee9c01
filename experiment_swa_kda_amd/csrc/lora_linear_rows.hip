// y_m = W x_m + B_a u_m for a few rows (a batch of requests' token step), with u = s A x from
// lora_shrink_rows_kernel before it: the projection and every row's own adapter in one kernel.
//
// A workgroup takes 16 outputs of 16 MT rows; its waves take 64 columns of the contraction at a time
// each and their partial tiles meet in LDS.  Every workgroup reads all its rows of x for its 16 outputs,
// so these loads are most of its work, and an MFMA fragment loaded directly (16 rows in 16 neighbouring
// lanes) takes 64 cycles of address processing for its 1 KB: lanes load along rows instead, 8 to a
// 128-byte line (16 cycles), and pass them through an LDS stage of the wave's own, without a barrier.
//
// Rows of different adapters share no product, so a thread forms the adapter's part of one output of
// one row with f32 FMAs: the 16 outputs' factors are 32 R contiguous bytes, and their loads are issued
// ahead of the main loop.
//
// Bound by the latency of the two launches, and for many rows by the adapters' bytes.  With the shrink,
// rank 16, against the library's product without adapters: 8 rows, 384 -> 1536: 5.5 / 3.9 us; 64 rows,
// 2048 -> 2048, an adapter each: 8.6 / 7.6 us (fragments loaded directly, and the adapters' factors by
// MFMA fragment lanes: 19.2); 8 rows, 384 -> 32768: 10.0 / 6.4.
#include "kda_device.hpp"
#include "kda_host.hpp"
#include "lora_rows.hpp"

namespace kda {

constexpr int kFewAhead = 2;  // 64-column steps of a wave in flight

template <int MT, int WAVES>
__global__ __launch_bounds__(WAVES * kWave, 4) void lora_linear_rows_kernel(LoraRows rows, int N, int K, int R, long ldx,
                                                                         const bf16* __restrict__ x,
                                                                         const bf16* __restrict__ w,
                                                                         const bf16* __restrict__ u,
                                                                         const bf16* __restrict__ b,
                                                                         bf16* __restrict__ y) {
  constexpr int STAGE = (16 * MT + 16) * 128;  // rows of 64 columns: x's, then W's
  constexpr int RG = 2;                        // vectors of 8 ranks whose loads are in flight
  static_assert(16 * MT * kWave <= STAGE, "a wave's partial tiles fit its stage");
  static_assert(256 * MT <= WAVES * kWave, "a thread for every row and output");
  __shared__ __attribute__((aligned(16))) char smem[WAVES * STAGE];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid % kWave;
  const int lr = lane % 16, kg = lane / 16, row8 = lane / 8, chunk8 = lane % 8;
  const int n0 = 16 * blockIdx.x, m0 = 16 * MT * blockIdx.y;

  const int pm = tid / 16, pn = tid % 16, m = m0 + pm, n = n0 + pn;
  const int a = pm < 16 * MT && n < N ? rows.id(m) : -1;
  const bf16* pu = u + (a >= 0 ? (size_t)m * R : (size_t)0);
  const bf16* pb = b + (a >= 0 ? ((size_t)a * N + n) * R : (size_t)0);
  const size_t plane = a >= 0 ? (size_t)rows.M * R : (size_t)0;
  bf16x8 fb[RG], fu[RG][2];  // (two parts of u: the sum is rounded to bf16)
  auto load_adapter = [&](int r0) {
#pragma unroll
    for (int g = 0; g < RG; ++g) {
      const int r = r0 + 8 * g;
      const bool in = a >= 0 && r < R;
      fb[g] = keep8(*(const bf16x8*)(pb + (in ? r : 0)), in);
#pragma unroll
      for (int k = 0; k < 2; ++k) fu[g][k] = keep8(*(const bf16x8*)(pu + k * plane + (in ? r : 0)), in);
    }
  };
  load_adapter(0);

  f32x4 acc[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) acc[t] = zero4();
  char* sx = smem + wave * STAGE;
  char* sw = sx + 16 * MT * 128;
  const int groups = (K + 63) / 64;  // of 64 columns; wave v takes v, v + WAVES, ...
  for (int s0 = wave; s0 < groups; s0 += kFewAhead * WAVES) {
    bf16x8 vx[kFewAhead][2 * MT], vw[kFewAhead][2];
#pragma unroll
    for (int q = 0; q < kFewAhead; ++q) {
      const int k = 64 * (s0 + q * WAVES) + 8 * chunk8;
      const bool ok = k < K;
#pragma unroll
      for (int v = 0; v < 2; ++v)
        vw[q][v] = keep8(*(const bf16x8*)(w + (size_t)min(n0 + 8 * v + row8, N - 1) * K + (ok ? k : 0)), ok);
#pragma unroll
      for (int v = 0; v < 2 * MT; ++v)
        vx[q][v] = keep8(*(const bf16x8*)(x + (size_t)min(m0 + 8 * v + row8, rows.M - 1) * ldx + (ok ? k : 0)), ok);
    }
#pragma unroll
    for (int q = 0; q < kFewAhead; ++q) {
      asm volatile("" ::: "memory");
#pragma unroll
      for (int v = 0; v < 2; ++v) *(bf16x8*)(sw + row64_off(8 * v + row8, chunk8)) = vw[q][v];
#pragma unroll
      for (int v = 0; v < 2 * MT; ++v) *(bf16x8*)(sx + row64_off(8 * v + row8, chunk8)) = vx[q][v];
      asm volatile("" ::: "memory");
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const bf16x8 fw = *(const bf16x8*)(sw + row64_off(lr, 4 * h + kg));
#pragma unroll
        for (int t = 0; t < MT; ++t)
          acc[t] = mfma16(fw, *(const bf16x8*)(sx + row64_off(16 * t + lr, 4 * h + kg)), acc[t]);
      }
    }
  }
  asm volatile("" ::: "memory");  // the wave's stage becomes its partial tiles
#pragma unroll
  for (int t = 0; t < MT; ++t) reinterpret_cast<f32x4*>(sx)[t * kWave + lane] = acc[t];
  float sum = 0.f;
  for (int r0 = 0;;) {
#pragma unroll
    for (int g = 0; g < RG; ++g)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        sum = fmaf((float)fu[g][0][e] + (float)fu[g][1][e], (float)fb[g][e], sum);
    r0 += 8 * RG;
    if (r0 >= R) break;
    load_adapter(r0);
  }
  __syncthreads();
  if (pm >= 16 * MT || m >= rows.M || n >= N) return;
  // accumulator: output 4 kg + i, row lr
  const int at = (pm / 16 * kWave + 16 * (pn / 4) + pm % 16) * 4 + pn % 4;
#pragma unroll
  for (int q = 0; q < WAVES; ++q) sum += reinterpret_cast<const float*>(smem + q * STAGE)[at];
  y[(size_t)m * N + n] = to_bf16(sum);
}

}  // namespace kda

extern "C" int kda_lora_linear_rows(int32_t rows, int32_t out_dim, int32_t in_dim, int32_t R, int32_t n,
                                    const int32_t* ids, int64_t rows_per_id, const void* x, int64_t x_row_stride,
                                    const void* weight, const void* lora_a, const void* lora_b, const float* scale,
                                    void* u, void* y, hipStream_t stream) {
  using namespace kda;
  KDA_REQUIRE(rows >= 0 && rows <= 512, "lora_linear_rows: at most 512 rows");
  KDA_REQUIRE(out_dim > 0 && out_dim % 8 == 0, "lora_linear_rows: out_dim must be a multiple of 8");
  int rc = check_lora("lora_linear_rows", rows, in_dim, R, n, ids, rows_per_id);
  if (rc != KDA_OK) return rc;
  KDA_REQUIRE(x_row_stride >= in_dim && x_row_stride % 8 == 0, "lora_linear_rows: x rows must be 16-byte aligned");
  if (rows == 0) return KDA_OK;
  KDA_REQUIRE(x && weight && lora_a && lora_b && u && y && aligned16(x, weight, lora_a, lora_b, u, y),
              "lora_linear_rows: null or unaligned pointer");
  const LoraRows lr{rows, n, ids, (int)rows_per_id};
  hipLaunchKernelGGL(lora_shrink_rows_kernel<4>, dim3((unsigned)rows, (unsigned)((R + 3) / 4)), dim3(256), 0, stream, lr,
                     in_dim, R, (const bf16*)x, (long)x_row_stride, (const bf16*)lora_a, scale, (bf16*)u);
  KDA_LAUNCH_CHECK("lora_shrink_rows");
  auto go = [&](auto kern, int tile, int waves) {
    hipLaunchKernelGGL(kern, dim3((unsigned)((out_dim + 15) / 16), (unsigned)((rows + tile - 1) / tile)),
                       dim3(waves * kWave), 0, stream, lr, out_dim, in_dim, R, (long)x_row_stride, (const bf16*)x,
                       (const bf16*)weight, (const bf16*)u, (const bf16*)lora_b, (bf16*)y);
  };
  // Four waves hold a contraction of 512 in flight, a longer one takes eight (16 rows, 2048 -> 2048: 6.7 us
  // against 9.7).  Tiles of 32 rows read W half as often, but halve the workgroups: they pay where a CU
  // has one all the same (64 rows, 1024 -> 4096: 8.3 us against 9.9 with 16 rows; 32 rows, 2048 -> 2048:
  // 7.6 against 7.1; 64 rows, 384 -> 1536: 6.2 either way).
  const int64_t tiles = (int64_t)((out_dim + 15) / 16) * ((rows + 31) / 32);
  if (in_dim <= 512)
    go(lora_linear_rows_kernel<1, 4>, 16, 4);
  else if (rows <= 16 || tiles < 256)
    go(lora_linear_rows_kernel<1, 8>, 16, 8);
  else
    go(lora_linear_rows_kernel<2, 8>, 32, 8);
  KDA_LAUNCH_CHECK("lora_linear_rows");
  return KDA_OK;
}
