// The rows of a call with low-rank adapters, and its checks (lora.hip, lora_linear.hip, lora_linear_rows.hip).
#pragma once

#include "kda_device.hpp"
#include "kda_host.hpp"

namespace kda {

// row m's adapter: ids[m / rows_per_id], -1 where that is none of the n
struct LoraRows {
  int M, n;
  const int32_t* ids;
  int rows_per_id;
  __device__ __forceinline__ int id(int m) const {
    if (m >= M) return -1;
    const int a = ids[m / rows_per_id];
    return a >= 0 && a < n ? a : -1;
  }
};

constexpr int kNoAdapter = 0x7fffffff;
// the smallest adapter above `prev` among the lanes' ids, kNoAdapter if there is none (lane steps
// as group_sum's)
__device__ __forceinline__ int next_adapter(int id, int prev) {
  int v = id > prev ? id : kNoAdapter;
  v = min(v, __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xf, 0xf, false));
  v = min(v, __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xf, 0xf, false));
  v = min(v, __builtin_amdgcn_update_dpp(0, v, 0x141, 0xf, 0xf, false));
  v = min(v, __builtin_amdgcn_update_dpp(0, v, 0x140, 0xf, 0xf, false));
  const auto r = __builtin_amdgcn_permlane16_swap((unsigned)v, (unsigned)v, false, false);
  v = min((int)r[0], (int)r[1]);
  const auto q = __builtin_amdgcn_permlane32_swap((unsigned)v, (unsigned)v, false, false);
  return __builtin_amdgcn_readfirstlane(min((int)q[0], (int)q[1]));
}

// eight bf16 of a buffer at a byte offset (kDropOffset: zeros) and a wave-uniform one
__device__ __forceinline__ bf16x8 buffer8(__amdgpu_buffer_rsrc_t rs, int off, int uniform) {
  typedef int i4 __attribute__((ext_vector_type(4)));
  const i4 v = __builtin_amdgcn_raw_buffer_load_b128(rs, off, uniform, 0);
  return __builtin_bit_cast(bf16x8, v);
}

// A row of 64 bf16 in LDS is 128 bytes; its 16-byte chunk c sits in slot c ^ (row % 8), so that the
// same chunk of eight neighbouring rows, and all chunks of one, fall on different banks.
__device__ __forceinline__ int row64_off(int row, int chunk) { return row * 128 + ((chunk ^ (row & 7)) << 4); }

// u [3, M, R]: an f32 value as the sum of three bf16 parts, each the rounding of what the ones before
// leave (24 bits together), so that the matrix cores take it as it lies: two parts where the result
// is rounded to bf16 (16 bits of u), three where it stays f32.
__device__ __forceinline__ void split3(float v, bf16& a, bf16& b, bf16& c) {
  a = to_bf16(v);
  v = __builtin_isinf((float)a) ? 0.f : v - (float)a;  // (an infinity is whole in its first part)
  b = to_bf16(v);
  v -= (float)b;
  c = to_bf16(v);
}

// v, or zeros
__device__ __forceinline__ bf16x8 keep8(bf16x8 v, bool ok) {
  const unsigned k = ok ? 0xffffffffu : 0u;
  uint4 u = __builtin_bit_cast(uint4, v);
  u.x &= k; u.y &= k; u.z &= k; u.w &= k;
  return __builtin_bit_cast(bf16x8, u);
}

// u[m, r] = scale_a (A_a x_m)_r, one wave per (row, rank): 64 lanes walk K in 16-byte vectors,
// AHEAD of them in flight.
template <int AHEAD>
__global__ __launch_bounds__(256) void lora_shrink_rows_kernel(LoraRows rows, int K, int R, const bf16* __restrict__ x,
                                                               long ldx, const bf16* __restrict__ a,
                                                               const float* __restrict__ scale,
                                                               bf16* __restrict__ u) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave;
  const int m = blockIdx.x, r = 4 * blockIdx.y + wave;
  if (r >= R) return;
  const int id = rows.id(m);
  float s = 0.f;
  if (id >= 0) {
    const bf16* px = x + (size_t)m * ldx;
    const bf16* pa = a + ((size_t)id * R + r) * K;
    for (int k0 = 8 * lane; k0 < K; k0 += 8 * kWave * AHEAD) {
      bf16x8 vx[AHEAD], va[AHEAD];
#pragma unroll
      for (int q = 0; q < AHEAD; ++q) {
        const int k = k0 + q * 8 * kWave;
        vx[q] = keep8(*(const bf16x8*)(px + (k < K ? k : 0)), k < K);
        va[q] = keep8(*(const bf16x8*)(pa + (k < K ? k : 0)), k < K);
      }
#pragma unroll
      for (int q = 0; q < AHEAD; ++q)
#pragma unroll
        for (int e = 0; e < 8; ++e) s = fmaf((float)vx[q][e], (float)va[q][e], s);
    }
    s = wave_sum(s) * (scale ? scale[id] : 1.f);
  }
  if (lane == 0) {
    const size_t at = (size_t)m * R + r, plane = (size_t)rows.M * R;
    split3(s, u[at], u[plane + at], u[2 * plane + at]);
  }
}

inline int check_lora(const char* what, int64_t M, int32_t J, int32_t R, int32_t n, const void* ids,
                      int64_t rows_per_id) {
  KDA_REQUIRE(M >= 0 && M <= (1 << 30), "%s: invalid row count", what);
  KDA_REQUIRE(J > 0 && J % 8 == 0 && J <= (1 << 24), "%s: feature dimensions must be positive multiples of 8", what);
  KDA_REQUIRE(R > 0 && R % 8 == 0 && R <= 128, "%s: the rank must be a multiple of 8 and at most 128", what);
  KDA_REQUIRE(n > 0 && n <= 65535, "%s: the number of adapters must be in [1, 65535]", what);
  KDA_REQUIRE(M == 0 || ids, "%s: null ids", what);
  KDA_REQUIRE(rows_per_id > 0 && rows_per_id <= (1 << 30), "%s: invalid rows per id", what);
  return KDA_OK;
}

}  // namespace kda
