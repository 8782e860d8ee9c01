// The shared projection with every row's adapter in one product: y_m = W x_m + F_a u_m, the
// adapter's part added to the accumulators (with the first two bf16 parts of u, 16 bits: the sum is
// rounded to 8), so y is written once and rounded once.
// WT false: W [N, K] and F [n, N, R] (the forward, F = B, u = s A x); WT true: W [K, N] and F [n, R, N]
// (the input gradient, y = dx, x = dy, F = A, u = t; N and K are then the output and contraction
// dimensions of this product).
//
// 128 x 128 output tiles, four compute waves of 64 x 64 each; two loader waves stream 32-deep steps
// of x and W into LDS (global -> LDS buffer loads), kGlStages - 1 steps ahead, one barrier a step.
// Stages are 16 KB, so two workgroups share a CU and one's epilogue hides behind the other's steps.
// Tiles of the same rows are neighbours on one XCD, whose L2 then holds x's rows and all of a small W.
// A tile of several adapters adds each of them to its own rows.
#include "kda_device.hpp"
#include "kda_host.hpp"
#include "lora_rows.hpp"

namespace kda {

constexpr int kGlTile = 128, kGlDepth = 32, kGlStages = 4, kGlCompute = 4;
constexpr int kGlThreads = (kGlCompute + 2) * kWave;
constexpr int kGlPart = kGlTile * kGlDepth * 2;  // 8 KB: one operand's step
constexpr int kGlStage = 2 * kGlPart;
constexpr int kGlLoads = kGlPart / 1024;         // loads of a step and loader
constexpr int kGlAdPitch = 64 + 4;               // a wave's 32 x 64 piece of F (WT)
static_assert(64 * 128 <= kGlStage / 2, "a wave's 64 x 64 results fit half a stage");
static_assert((kGlStages - 2) * kGlLoads < 64, "vmcnt range");
static_assert(32 * kGlAdPitch * 2 <= kGlStage / 2, "a wave's piece of F fits half a stage");

// A step of a row-major operand whose rows run along the contraction: 128 rows of 64 bytes.  The
// 16-byte chunk c of row r sits in slot c ^ (r / 2 % 4), so that eight neighbouring rows' reads of
// one chunk fall on different banks.
__device__ __forceinline__ bf16x8 gl_row_frag(const char* part, int r0, int lane) {
  const int r = r0 + lane % 16;
  return *reinterpret_cast<const bf16x8*>(part + r * 64 + (((lane / 16) ^ (r >> 1 & 3)) << 4));
}
// A step of an operand whose rows are the contraction's: 32 rows of 256 bytes, chunk c of row r in
// slot c ^ (2 (r % 4)); fragments run down the columns (two transposing reads).
__device__ __forceinline__ bf16x8 gl_col_frag(const char* part, int c0, int lane) {
  const int lr = lane % 16, kg = lane / 16, r = 8 * kg + lr / 4, col = c0 + 4 * (lr % 4);
  const char* p = part + r * 256 + (((col >> 3) ^ (2 * (r & 3))) << 4) + ((col >> 2) & 1) * 8;
  const short4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_t*)p);
  const short4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_t*)(p + 4 * 256));
  return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

template <bool WT>
__global__ __launch_bounds__(kGlThreads, 3) void lora_linear_kernel(LoraRows rows, int N, int K, int R,
                                                                    const bf16* __restrict__ x, long ldx,
                                                                    const bf16* __restrict__ w,
                                                                    const bf16* __restrict__ u,
                                                                    const bf16* __restrict__ f, bf16* __restrict__ y,
                                                                    int tiles_n, int items) {
  __shared__ __attribute__((aligned(16))) char smem[kGlStages * kGlStage];
  const int per_xcd = (items + kXcds - 1) / kXcds;
  const int item = (blockIdx.x % kXcds) * per_xcd + blockIdx.x / kXcds;
  if (blockIdx.x / kXcds >= per_xcd || item >= items) return;  // grid rounding (the whole workgroup)
  const int m0 = (item / tiles_n) * kGlTile, n0 = (item % tiles_n) * kGlTile;
  const int nsteps = (K + kGlDepth - 1) / kGlDepth;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave;
  constexpr int P = kGlStages - 1;

  if (wave >= kGlCompute) {
    // ---- loader waves: wave 4 moves rows of x, wave 5 W ----
    const bool isx = wave == kGlCompute;
    auto issue = [&](int q) {
      char* st = smem + (q % kGlStages) * kGlStage + (isx ? 0 : kGlPart);
      const int k0 = kGlDepth * q;
      if (WT && !isx) {
        const __amdgpu_buffer_rsrc_t rs = raw_rsrc(w + (size_t)k0 * N + n0);
#pragma unroll
        for (int i = 0; i < kGlLoads; ++i) {
          const int r = 4 * i + lane / 16, c = 8 * ((lane % 16) ^ (2 * (r & 3)));
          const bool ok = k0 + r < K && n0 + c < N;
          __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)(st + i * 1024), 16,
                                                   ok ? (r * N + c) * 2 : kDropOffset, 0, 0, 0);
        }
      } else {
        const long ld = isx ? ldx : (long)K;
        const int r0 = isx ? m0 : n0, rn = isx ? rows.M : N;
        const __amdgpu_buffer_rsrc_t rs = raw_rsrc((isx ? x : w) + (size_t)r0 * ld);
#pragma unroll
        for (int i = 0; i < kGlLoads; ++i) {
          const int r = 16 * i + lane / 4, k = k0 + 8 * ((lane % 4) ^ (r >> 1 & 3));
          const bool ok = r0 + r < rn && k < K;
          __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)(st + i * 1024), 16,
                                                   ok ? (int)((r * ld + k) * 2) : kDropOffset, 0, 0, 0);
        }
      }
    };
    auto wait_landed = [&](int later) {  // all but the last `later` steps issued have landed
      switch (later) {
        case 2: wait_vmcnt<2 * kGlLoads>(); break;
        case 1: wait_vmcnt<kGlLoads>(); break;
        default: wait_vmcnt<0>(); break;
      }
    };
    for (int q = 0; q < P && q < nsteps; ++q) issue(q);
    wait_landed(min(P - 1, nsteps - 1));
    ring_barrier();  // B0: step 0 visible
    for (int q = 0; q < nsteps; ++q) {
      wait_landed(max(0, min(P - 2, nsteps - 2 - q)));
      ring_barrier();  // A(q): step q + 1 visible; step q's slot is free
      if (q + P < nsteps) issue(q + P);
    }
    return;
  }

  // ---- compute wave (wm, wn): rows m0 + 64 wm .., columns n0 + 64 wn .. ----
  const int wm = wave / 2, wn = wave % 2, lr = lane % 16, kg = lane / 16;
  f32x4 acc[4][4];  // [column tile][row tile]
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int t = 0; t < 4; ++t) acc[c][t] = zero4();
  ring_barrier();  // B0
  for (int q = 0; q < nsteps; ++q) {
    const char* st = smem + (q % kGlStages) * kGlStage;
    bf16x8 fx[4], fw[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) fx[t] = gl_row_frag(st, 64 * wm + 16 * t, lane);
#pragma unroll
    for (int c = 0; c < 4; ++c)
      fw[c] = WT ? gl_col_frag(st + kGlPart, 64 * wn + 16 * c, lane) : gl_row_frag(st + kGlPart, 64 * wn + 16 * c, lane);
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int t = 0; t < 4; ++t) acc[c][t] = mfma16(fw[c], fx[t], acc[c][t]);
    ring_barrier();  // A(q)
  }

  // ---- the adapters of the wave's 64 rows, one after another ----
  const int mw = m0 + 64 * wm, nw = n0 + 64 * wn;
  const int row_id = rows.id(mw + lane);
  const size_t plane = (size_t)rows.M * R;
  // (buffers from the wave's first row or column: 32-bit offsets, and what is outside reads as zero)
  const __amdgpu_buffer_rsrc_t rhi = raw_rsrc(u + (size_t)mw * R), rlo = raw_rsrc(u + plane + (size_t)mw * R);
  // half a stage per wave, of stages that nobody reads any more (the last step's is not among them):
  // pieces of F (WT), and the result
  bf16* piece = reinterpret_cast<bf16*>(smem + ((nsteps + wave / 2) % kGlStages) * kGlStage + (wave % 2) * (kGlStage / 2));
  // one loop over adapters and their 32-deep steps, entered in any case (without an adapter nothing is
  // read and no row takes the result): a loop behind a branch doubled the accumulators' registers
  int a = next_adapter(row_id, -1), r0 = 0;
  do {
    const int r = a == kNoAdapter ? R : r0 + 8 * kg;
    const size_t base = a == kNoAdapter ? 0 : (size_t)a * R * N;
    bf16x8 ff[4];
    if constexpr (WT) {
      const __amdgpu_buffer_rsrc_t rf = raw_rsrc(f + base + (size_t)r0 * N + nw);
      const int rr = lane / 8, c = 8 * (lane % 8);
      uint4 v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)  // 32 rows of 64 columns: 8 of 16 bytes each
        v[i] = __builtin_bit_cast(uint4, buffer8(rf, a != kNoAdapter && r0 + 8 * i + rr < R && nw + c < N ? (rr * N + c) * 2 : kDropOffset, 16 * i * N));
      asm volatile("" ::: "memory");
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint2* d = (uint2*)(piece + (8 * i + rr) * kGlAdPitch + c);
        d[0] = make_uint2(v[i].x, v[i].y);
        d[1] = make_uint2(v[i].z, v[i].w);
      }
      asm volatile("" ::: "memory");
#pragma unroll
      for (int c = 0; c < 4; ++c) ff[c] = lds_col_frag(piece, kGlAdPitch, 0, 16 * c, lane);
    } else {
      const __amdgpu_buffer_rsrc_t rf = raw_rsrc(f + base + (size_t)nw * R);
#pragma unroll
      for (int c = 0; c < 4; ++c)
        ff[c] = buffer8(rf, r < R && nw + 16 * c + lr < N ? (lr * R + r) * 2 : kDropOffset, 32 * c * R);
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const bool mine = __shfl(row_id, 16 * t + lr) == a;
      const int off = r < R && mw + 16 * t + lr < rows.M ? (lr * R + r) * 2 : kDropOffset;
      const bf16x8 hi = buffer8(rhi, off, 32 * t * R), lo = buffer8(rlo, off, 32 * t * R);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        // (chosen, not multiplied by zero: an infinity in this adapter stays out of other rows)
        const f32x4 d = mfma16(ff[c], lo, mfma16(ff[c], hi, zero4()));
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[c][t][i] += mine ? d[i] : 0.f;
      }
      __builtin_amdgcn_sched_barrier(0);  // (all rows at once would spill registers)
    }
    r0 += kGlDepth;
    if (r0 >= R) {
      r0 = 0;
      a = next_adapter(row_id, a);
    }
  } while (a != kNoAdapter);
  // accumulator: column 16 c + 4 kg + i, row 16 t + lr of the wave's 64; through the wave's half stage
  // (128-byte rows, chunk q of row r in slot q ^ (r % 8)), so that eight lanes store a row's line
  char* out = reinterpret_cast<char*>(piece);
  asm volatile("" ::: "memory");
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      bf16x4 o;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = to_bf16(acc[c][t][i]);
      *(bf16x4*)(out + (16 * t + lr) * 128 + (((2 * c + kg / 2) ^ (lr & 7)) << 4) + 8 * (kg % 2)) = o;
    }
  asm volatile("" ::: "memory");
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = 8 * i + lane / 8, q = lane % 8, m = mw + r, n = nw + 8 * q;
    if (m < rows.M && n < N) *(bf16x8*)(y + (size_t)m * N + n) = *(const bf16x8*)(out + r * 128 + ((q ^ (r & 7)) << 4));
  }
}

}  // namespace kda

extern "C" int kda_lora_linear(int64_t M, int32_t N, int32_t K, int32_t R, int32_t n, const int32_t* ids,
                               int64_t rows_per_id, const void* x, int64_t ldx, const void* weight,
                               int32_t weight_rows, const void* u, const void* factor, void* y, hipStream_t stream) {
  using namespace kda;
  int rc = check_lora("lora_linear", M, K, R, n, ids, rows_per_id);
  if (rc != KDA_OK) return rc;
  KDA_REQUIRE(N > 0 && N % 8 == 0 && N <= (1 << 20) && K <= (1 << 20),
              "lora_linear: feature dimensions must be multiples of 8 and at most 2^20");
  if (M == 0) return KDA_OK;
  KDA_REQUIRE(x && weight && u && factor && y && aligned16(x, weight, u, factor, y), "lora_linear: null or unaligned pointer");
  KDA_REQUIRE(ldx >= K && ldx % 8 == 0 && ldx <= (1 << 20), "lora_linear: rows of x must be 16-byte aligned");
  const int64_t tiles_n = (N + kGlTile - 1) / kGlTile, items = tiles_n * ((M + kGlTile - 1) / kGlTile);
  KDA_REQUIRE(items <= (1 << 30), "lora_linear: too many tiles");
  const LoraRows rows{(int)M, n, ids, (int)rows_per_id};
  const unsigned grid = (unsigned)((items + kXcds - 1) / kXcds * kXcds);
  auto go = [&](auto kern) {
    hipLaunchKernelGGL(kern, dim3(grid), dim3(kGlThreads), 0, stream, rows, N, K, R, (const bf16*)x, (long)ldx,
                       (const bf16*)weight, (const bf16*)u, (const bf16*)factor, (bf16*)y, (int)tiles_n, (int)items);
  };
  weight_rows ? go(lora_linear_kernel<true>) : go(lora_linear_kernel<false>);
  KDA_LAUNCH_CHECK("lora_linear");
  return KDA_OK;
}
