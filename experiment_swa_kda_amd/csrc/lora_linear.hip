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
// Tiles of the same rows are neighbours on one XCD, whose L2 then holds x's rows and all of a small W, and
// of those two that follow each other share a CU, so that the second finds x's lines in the first level
// cache (8192 x 384 x 4096 57 -> 55 us, transposed 58 -> 52; calls of one round of tiles as before).
// A tile of several adapters adds each of them to its own rows.
//
// Bound by the operands' way from L2 to LDS: 8192 rows, 384 -> 1536, rank 16 take 21 us (the library's
// product without adapters 26), of them 9 for the tiles' set-up and the write of y, 3 for the adapters and
// 0.9 for every 32-deep step, 14 TB/s.  Long contractions gain less from the shared read and write of y
// than larger tiles would: 16384 x 2048 x 2048 165 us, 830 TFLOP/s.
#include "kda_device.hpp"
#include "kda_host.hpp"
#include "lora_rows.hpp"

namespace kda {

constexpr int kGlTile = 128, kGlDepth = 32, kGlStages = 4, kGlCompute = 4;
constexpr int kGlThreads = (kGlCompute + 2) * kWave;
constexpr int kGlPart = kGlTile * kGlDepth * 2;  // 8 KB: one operand's step
constexpr int kGlStage = 2 * kGlPart;
constexpr int kGlLoads = kGlPart / 1024;         // loads of a step and loader
constexpr int kGlPiecePitch = 32 + 8;            // a wave's 32 x 32 piece of F (WT)
static_assert(64 * 128 <= kGlStage / 2, "a wave's 64 x 64 results fit half a stage");
static_assert((kGlStages - 2) * kGlLoads < 64, "vmcnt range");

// A step of a row-major operand whose rows run along the contraction: 128 rows of 64 bytes.  The
// 16-byte chunk c of row r sits in slot c ^ (r / 4 % 4), so that sixteen neighbouring rows' reads of
// one chunk fall on different banks.
__device__ __forceinline__ bf16x8 gl_row_frag(const char* part, int r0, int lane) {
  const int r = r0 + lane % 16;
  return *reinterpret_cast<const bf16x8*>(part + r * 64 + (((lane / 16) ^ (r >> 2 & 3)) << 4));
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

// Adds the adapters of a wave's 64 rows from mw on, one after another, to its columns from nw on.
template <bool WT>
__device__ __forceinline__ void gl_add_adapters(LoraRows rows, int N, int R, const bf16* __restrict__ u,
                                                const bf16* __restrict__ f, int mw, int nw, int lane,
                                                bf16* piece, f32x4 (&acc)[4][4]) {
  const int lr = lane % 16, kg = lane / 16;
  const int row_id = rows.id(mw + lane);
  const size_t plane = (size_t)rows.M * R;
  // (buffers from the wave's first row or column: 32-bit offsets, and what is outside reads as zero)
  const __amdgpu_buffer_rsrc_t rhi = raw_rsrc(u + (size_t)mw * R), rlo = raw_rsrc(u + plane + (size_t)mw * R);
  int a = next_adapter(row_id, -1), r0 = 0;
  while (a != kNoAdapter) {
    const int r = r0 + 8 * kg;
    const size_t base = (size_t)a * R * N;
    bf16x8 ff[4];
    if constexpr (WT) {
      const __amdgpu_buffer_rsrc_t rf = raw_rsrc(f + base + (size_t)r0 * N + nw);
      const int rr = lane / 4, c = 8 * (lane % 4);
      bf16x8 v[2][2];
#pragma unroll
      for (int h = 0; h < 2; ++h)  // 32 rows of 32 columns
#pragma unroll
        for (int i = 0; i < 2; ++i)
          v[h][i] = buffer8(rf, r0 + 16 * i + rr < R && nw + 32 * h + c < N ? (rr * N + c) * 2 : kDropOffset, 32 * i * N + 64 * h);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        asm volatile("" ::: "memory");
#pragma unroll
        for (int i = 0; i < 2; ++i) *(bf16x8*)(piece + (16 * i + rr) * kGlPiecePitch + c) = v[h][i];
        asm volatile("" ::: "memory");
#pragma unroll
        for (int c2 = 0; c2 < 2; ++c2) ff[2 * h + c2] = lds_col_frag(piece, kGlPiecePitch, 0, 16 * c2, lane);
      }
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
  }
}

template <bool WT, bool FIRST>
__global__ __launch_bounds__(kGlThreads, 3) void lora_linear_kernel(LoraRows rows, int N, int K, int R,
                                                                    const bf16* __restrict__ x, long ldx,
                                                                    const bf16* __restrict__ w,
                                                                    const bf16* __restrict__ u,
                                                                    const bf16* __restrict__ f, bf16* __restrict__ y,
                                                                    int tiles_n, int items) {
  __shared__ __attribute__((aligned(16))) char smem[kGlStages * kGlStage];
  __shared__ __attribute__((aligned(16))) bf16 piece[WT ? kGlCompute : 1][WT ? 32 * kGlPiecePitch : 1];
  const int per_xcd = (items + kXcds - 1) / kXcds;
  // an XCD's 32 CUs take its workgroups in turn, twice over: at and at + 32 share one
  int at = blockIdx.x / kXcds;
  if (at < per_xcd / 64 * 64) at = at / 64 * 64 + 2 * (at % 32) + at % 64 / 32;
  const int item = (blockIdx.x % kXcds) * per_xcd + at;
  if (at >= per_xcd || item >= items) return;  // grid rounding (the whole workgroup)
  const int m0 = (item / tiles_n) * kGlTile, n0 = (item % tiles_n) * kGlTile;
  const int nsteps = (K + kGlDepth - 1) / kGlDepth;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave;
  constexpr int P = kGlStages - 1;

  if (wave >= kGlCompute) {
    // ---- loader waves: wave 4 moves rows of x, wave 5 W.  A step is kGlLoads loads whose offsets from the
    // step's base do not change (kDropOffset: outside the operand), so that issuing one keeps up with
    // the products; only the last step may have columns to drop ----
    const bool isx = wave == kGlCompute;
    const bool cols = WT && !isx;  // rows of the contraction
    const long ld = cols ? N : isx ? ldx : (long)K;
    int off[kGlLoads], k_of[kGlLoads];  // byte offset and place in the step's 32 of the contraction
#pragma unroll
    for (int i = 0; i < kGlLoads; ++i) {
      if (cols) {
        const int r = 4 * i + lane / 16, c = 8 * ((lane % 16) ^ (2 * (r & 3)));
        k_of[i] = r;
        off[i] = n0 + c < N ? (r * N + c) * 2 : kDropOffset;
      } else {
        const int r = 16 * i + lane / 4, k = 8 * ((lane % 4) ^ (r >> 2 & 3));
        k_of[i] = k;
        off[i] = (isx ? m0 + r < rows.M : n0 + r < N) ? (int)(r * ld + k) * 2 : kDropOffset;
      }
    }
    const bf16* base = cols ? w + n0 : (isx ? x + (size_t)m0 * ldx : w + (size_t)n0 * K);
    const size_t advance = cols ? (size_t)kGlDepth * N : kGlDepth;
    auto issue = [&](int q) {
      char* st = smem + (q % kGlStages) * kGlStage + (isx ? 0 : kGlPart);
      const __amdgpu_buffer_rsrc_t rs = raw_rsrc(base + q * advance);
      const int left = K - kGlDepth * q;
      if (left >= kGlDepth) {
#pragma unroll
        for (int i = 0; i < kGlLoads; ++i)
          __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)(st + i * 1024), 16, off[i],
                                                   0, 0, 0);
      } else {
#pragma unroll
        for (int i = 0; i < kGlLoads; ++i)
          __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)(st + i * 1024), 16,
                                                   k_of[i] < left ? off[i] : kDropOffset, 0, 0, 0);
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
      ring_barrier();  // A(q): step q + 1 visible; step q - 1's slot is read
      if (q + P < nsteps) issue(q + P);
    }
    return;
  }

  // ---- compute wave (wm, wn): rows m0 + 64 wm .., columns n0 + 64 wn .. ----
  const int wm = wave / 2, wn = wave % 2, lr = lane % 16, kg = lane / 16;
  const int mw = m0 + 64 * wm, nw = n0 + 64 * wn;
  f32x4 acc[4][4];  // [column tile][row tile]
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int t = 0; t < 4; ++t) acc[c][t] = zero4();

  // (while the loaders' first steps are on their way)
  if constexpr (FIRST) gl_add_adapters<WT>(rows, N, R, u, f, mw, nw, lane, piece[WT ? wave : 0], acc);
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
  if constexpr (!FIRST) {
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int t = 0; t < 4; ++t) asm volatile("" : "+v"(acc[c][t]));  // (one loop's results, the next one's start: no copies)
    gl_add_adapters<WT>(rows, N, R, u, f, mw, nw, lane, piece[WT ? wave : 0], acc);
  }

  // accumulator: column 16 c + 4 kg + i, row 16 t + lr of the wave's 64; through the wave's half stage
  // (128-byte rows, chunk q of row r in slot q ^ (r % 8); of stages that nobody reads any more: the last
  // step's is not among them), so that eight lanes store a row's line
  char* out = smem + ((nsteps + wave / 2) % kGlStages) * kGlStage + (wave % 2) * (kGlStage / 2);
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
  // One round of tiles (two workgroups a CU) adds the adapters while its first loads are on their way (8192 x
  // 1536 -> 384 20.9 us against 22.0); of several rounds one tile's adapters hide behind another's steps, and
  // come last, when the loads of the tile after are long under way (512 x 384 -> 32768 29.7 / 33.5, 8192 x 384
  // -> 4096 50 / 55).
  if (items <= 2 * 256)
    weight_rows ? go(lora_linear_kernel<true, true>) : go(lora_linear_kernel<false, true>);
  else
    weight_rows ? go(lora_linear_kernel<true, false>) : go(lora_linear_kernel<false, false>);
  KDA_LAUNCH_CHECK("lora_linear");
  return KDA_OK;
}

extern "C" int kda_lora_forward(int64_t M, int32_t N, int32_t K, int32_t R, int32_t n, const int32_t* ids,
                                int64_t rows_per_id, const void* x, int64_t ldx, const void* weight,
                                const void* lora_a, const void* lora_b, const float* scale, int32_t how, void* u,
                                void* y, hipStream_t stream) {
  KDA_REQUIRE(how >= KDA_LORA_ROWS && how <= KDA_LORA_PART, "lora_forward: unknown way");
  if (how == KDA_LORA_ROWS) {
    KDA_REQUIRE(M >= 0 && M <= 512, "lora_forward: at most 512 rows");
    return kda_lora_linear_rows((int32_t)M, N, K, R, n, ids, rows_per_id, x, ldx, weight, lora_a, lora_b, scale, u, y,
                                stream);
  }
  int rc = kda_lora_shrink(M, K, R, n, ids, rows_per_id, x, ldx, lora_a, 0, scale, u, stream);
  if (rc != KDA_OK) return rc;
  if (how == KDA_LORA_WHOLE)
    return kda_lora_linear(M, N, K, R, n, ids, rows_per_id, x, ldx, weight, 0, u, lora_b, y, stream);
  return kda_lora_expand(M, N, R, n, ids, rows_per_id, u, lora_b, 1, y, N, stream);
}

// t = s B^T dy in its three parts, then the factor gradients' partials (one gradient after the other)
static size_t lora_t_bytes(int64_t M, int32_t R) { return M > 0 && R > 0 ? kda::align256((size_t)3 * M * R * 2) : 0; }

extern "C" size_t kda_lora_backward_scratch_bytes(int64_t M, int32_t N, int32_t K, int32_t R, int32_t n) {
  const size_t a = kda_lora_grad_scratch_bytes(M, K, R, n), b = kda_lora_grad_scratch_bytes(M, N, R, n);
  return lora_t_bytes(M, R) + (a > b ? a : b);
}

extern "C" int kda_lora_backward(int64_t M, int32_t N, int32_t K, int32_t R, int32_t n, const int32_t* ids,
                                 int64_t rows_per_id, const void* x, int64_t ldx, const void* grad_output, int64_t ldg,
                                 const void* weight, const void* lora_a, const void* lora_b, const float* scale,
                                 const void* u, int32_t how, void* dx, float* da, float* db, void* scratch,
                                 hipStream_t stream) {
  KDA_REQUIRE(how == KDA_LORA_WHOLE || how == KDA_LORA_PART, "lora_backward: unknown way");
  KDA_REQUIRE(M <= 0 || scratch, "lora_backward: null scratch");
  void* t = scratch;
  void* part = scratch ? (char*)scratch + lora_t_bytes(M, R) : nullptr;
  int rc = KDA_OK;
  if (dx || da) rc = kda_lora_shrink(M, N, R, n, ids, rows_per_id, grad_output, ldg, lora_b, 1, scale, t, stream);
  if (rc == KDA_OK && dx)
    rc = how == KDA_LORA_WHOLE
             ? kda_lora_linear(M, K, N, R, n, ids, rows_per_id, grad_output, ldg, weight, 1, t, lora_a, dx, stream)
             : kda_lora_expand(M, K, R, n, ids, rows_per_id, t, lora_a, 0, dx, K, stream);
  if (rc == KDA_OK && da) rc = kda_lora_grad(M, K, R, n, ids, rows_per_id, x, ldx, t, 0, da, part, stream);
  if (rc == KDA_OK && db) rc = kda_lora_grad(M, N, R, n, ids, rows_per_id, grad_output, ldg, u, 1, db, part, stream);
  return rc;
}
