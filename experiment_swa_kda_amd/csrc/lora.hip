// Low-rank adapters of many requests beside a shared projection: row m of x belongs to adapter
// a = id(m) (none if outside [0, n)), and
//   y_m = W x_m + s_a B_a (A_a x_m)
// with A_a [R, K] and B_a [N, R] far smaller than W.  Three products with a factor F_a, each
// reading its long operand once:
//   shrink   u_m = s_a F_a x_m             (forward with A; the backward's t = s B^T dy with B)
//   expand   y_m = F_a^T u_m               (forward with B; the backward's A^T t with A)
//   grad     G_a = sum_{m of a} u_m x_m^T  (dB from s A x and dy; dA from t and x)
// F is read in either layout, [n, R, J] or [n, J, R] (J the long dimension), so neither direction
// needs a transposed copy.  u stays in f32 and meets the bf16 matrix cores as a sum of bf16 parts:
// two for expand (16 bits, its result is rounded to 8), three for grad (24 bits, f32 gradients).
//
// A tile of rows may hold several adapters: each product runs once per distinct adapter of the
// tile, in ascending order, with the other rows masked.  A row's id is ids[m / rows_per_id].
#include "kda_device.hpp"
#include "kda_host.hpp"

namespace kda {

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

// the smallest adapter above `prev` among the lanes' ids, 0x7fffffff if there is none
__device__ __forceinline__ int next_adapter(int id, int prev) {
  int v = id > prev ? id : 0x7fffffff;
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) v = min(v, __shfl_xor(v, o));
  return __builtin_amdgcn_readfirstlane(v);
}

constexpr int kNoAdapter = 0x7fffffff;

__device__ __forceinline__ bf16x8 keep8(bf16x8 v, bool ok) {
  const unsigned k = ok ? 0xffffffffu : 0u;
  uint4 u = __builtin_bit_cast(uint4, v);
  u.x &= k; u.y &= k; u.z &= k; u.w &= k;
  return __builtin_bit_cast(bf16x8, u);
}

// ---------------------------------------------------------------------------------------
// shrink: one workgroup per 16 MT rows; its waves split J and their partial tiles meet in LDS.
// RT = ceil(R / 16).  TRANSPOSED: F is [n, J, R], and 32 x R pieces of it pass through LDS for
// fragments that run down its columns.
// ---------------------------------------------------------------------------------------
constexpr int kShrinkWaves = 8;

template <int RT, int MT, bool TRANSPOSED>
__global__ __launch_bounds__(kShrinkWaves * kWave) void lora_shrink_kernel(LoraRows rows, int J, int R,
                                                                          const bf16* __restrict__ x, long ldx,
                                                                          const bf16* __restrict__ f,
                                                                          const float* __restrict__ scale,
                                                                          float* __restrict__ u) {
  constexpr int PITCH = 16 * RT + 4;  // elements; 8-byte aligned rows for the transposing reads
  constexpr int STAGE = TRANSPOSED ? kShrinkWaves * 32 * PITCH * 2 : 0;
  constexpr int PART = kShrinkWaves * RT * MT * kWave * 16;
  __shared__ __attribute__((aligned(16))) char smem[STAGE > PART ? STAGE : PART];
  f32x4(*part)[RT * MT][kWave] = reinterpret_cast<f32x4(*)[RT * MT][kWave]>(smem);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave;
  const int lr = lane % 16, kg = lane / 16;
  const int m0 = 16 * MT * blockIdx.x;
  const int my_id = rows.id(m0 + lane % (16 * MT));
  const bf16* xr[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) xr[t] = x + (size_t)min(m0 + 16 * t + lr, rows.M - 1) * ldx;
  for (int a = next_adapter(my_id, -1); a != kNoAdapter; a = next_adapter(my_id, a)) {
    const bf16* fa = f + (size_t)a * R * J;
    f32x4 acc[RT][MT];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int t = 0; t < MT; ++t) acc[r][t] = zero4();
    for (int j0 = 32 * wave; j0 < J; j0 += 32 * kShrinkWaves) {
      const int j = j0 + 8 * kg;
      const bool ok = j < J;  // J is a multiple of 8: a lane's eight columns are all in or all out
      const int jc = ok ? j : 0;
      bf16x8 fx[MT], ff[RT];
#pragma unroll
      for (int t = 0; t < MT; ++t) fx[t] = keep8(*(const bf16x8*)(xr[t] + jc), ok);
      if constexpr (TRANSPOSED) {
        bf16* st = reinterpret_cast<bf16*>(smem) + wave * 32 * PITCH;
        // 32 rows of R columns, 8 at a time (R is a multiple of 8); rows past J are zero
        for (int c = lane; c < 32 * (R / 8); c += kWave) {
          const int row = c / (R / 8), col = 8 * (c % (R / 8));
          const bool in = j0 + row < J;
          const bf16x8 v = keep8(*(const bf16x8*)(fa + (size_t)(in ? j0 + row : 0) * R + col), in);
          const uint4 w = __builtin_bit_cast(uint4, v);
          uint2* d = (uint2*)(st + row * PITCH + col);
          d[0] = make_uint2(w.x, w.y);
          d[1] = make_uint2(w.z, w.w);
        }
        asm volatile("" ::: "memory");
#pragma unroll
        for (int r = 0; r < RT; ++r) ff[r] = lds_col_frag(st, PITCH, 0, 16 * r, lane);
        asm volatile("" ::: "memory");
      } else {
#pragma unroll
        for (int r = 0; r < RT; ++r) ff[r] = keep8(*(const bf16x8*)(fa + (size_t)min(16 * r + lr, R - 1) * J + jc), ok);
      }
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[r][t] = mfma16(ff[r], fx[t], acc[r][t]);
    }
    __syncthreads();  // the stages (or the last adapter's partials) are read
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int t = 0; t < MT; ++t) part[wave][r * MT + t][lane] = acc[r][t];
    __syncthreads();
    const float s = scale ? scale[a] : 1.f;
    // accumulator: r 16 rt + 4 kg + i, row of x lr
    for (int q = wave; q < RT * MT; q += kShrinkWaves) {
      f32x4 v = part[0][q][lane];
#pragma unroll
      for (int w = 1; w < kShrinkWaves; ++w) v += part[w][q][lane];
      const int t = q % MT, r = 16 * (q / MT) + 4 * kg, m = m0 + 16 * t + lr;
      if (rows.id(m) == a && r < R) *(f32x4*)(u + (size_t)m * R + r) = v * s;
    }
    __syncthreads();  // the next adapter's stages overwrite the partials
  }
  // rows of no adapter
  for (int q = threadIdx.x; q < 16 * MT * (R / 4); q += kShrinkWaves * kWave) {
    const int m = m0 + q / (R / 4);
    if (m < rows.M && rows.id(m) < 0) *(f32x4*)(u + (size_t)m * R + 4 * (q % (R / 4))) = zero4();
  }
}

// ---------------------------------------------------------------------------------------
// expand: 64 rows x 256 columns per workgroup; wave w has rows 16 w .. and keeps their u in
// registers.  KS = ceil(R / 32) steps of the contraction.  TRANSPOSED: F is [n, R, J].
// ---------------------------------------------------------------------------------------
constexpr int kExpandCols = 256;

template <int KS, bool TRANSPOSED>
__global__ __launch_bounds__(256) void lora_expand_kernel(LoraRows rows, int J, int R, const float* __restrict__ u,
                                                          const bf16* __restrict__ f, bf16* __restrict__ y, long ldy) {
  constexpr int PITCH = 64 + 4;
  __shared__ __attribute__((aligned(16))) bf16 st[TRANSPOSED ? 32 * KS * PITCH : 1];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave;
  const int lr = lane % 16, kg = lane / 16;
  const int m0 = 64 * blockIdx.x, m = m0 + 16 * wave + lr;
  const int tile_id = rows.id(m0 + lane), my_id = rows.id(m);
  bf16x8 hi[KS], lo[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const int r = 32 * s + 8 * kg;
    float v[8];
    const bool ok = m < rows.M && r < R;
    load8f(u + (size_t)(ok ? m : 0) * R + (ok ? r : 0), v);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = ok ? v[e] : 0.f;
    split8(v, hi[s], lo[s]);
  }
  const int c_end = min(J, kExpandCols * ((int)blockIdx.y + 1));
  for (int c0 = kExpandCols * blockIdx.y; c0 < c_end; c0 += 64) {
    f32x4 acc[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) acc[t] = zero4();
    for (int a = next_adapter(tile_id, -1); a != kNoAdapter; a = next_adapter(tile_id, a)) {
      const bf16* fa = f + (size_t)a * R * J;
      const bool mine = my_id == a;
      if constexpr (TRANSPOSED) {
        __syncthreads();  // the previous piece is read
        for (int c = threadIdx.x; c < 32 * KS * 8; c += 256) {
          const int row = c / 8, col = 8 * (c % 8);
          const bool in = row < R && c0 + col < J;
          const uint4 w = __builtin_bit_cast(
              uint4, keep8(*(const bf16x8*)(fa + (in ? (size_t)row * J + c0 + col : (size_t)0)), in));
          uint2* d = (uint2*)(st + row * PITCH + col);
          d[0] = make_uint2(w.x, w.y);
          d[1] = make_uint2(w.z, w.w);
        }
        __syncthreads();
      }
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const bf16x8 h = keep8(hi[s], mine), l = keep8(lo[s], mine);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          bf16x8 ff;
          if constexpr (TRANSPOSED) {
            ff = lds_col_frag(st, PITCH, 32 * s, 16 * t, lane);
          } else {
            const int r = 32 * s + 8 * kg, j = min(c0 + 16 * t + lr, J - 1);
            ff = keep8(*(const bf16x8*)(fa + (size_t)j * R + (r < R ? r : 0)), r < R);
          }
          acc[t] = mfma16(ff, h, acc[t]);
          acc[t] = mfma16(ff, l, acc[t]);
        }
      }
    }
    // accumulator: column c0 + 16 t + 4 kg + i, row lr of the wave's 16
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int j = c0 + 16 * t + 4 * kg;
      if (m < rows.M && j < J) {
        bf16x4 o;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = to_bf16(acc[t][i]);
        *(bf16x4*)(y + (size_t)m * ldy + j) = o;
      }
    }
  }
}

// ---------------------------------------------------------------------------------------
// grad: workgroup (128 columns of J, adapter, range of rows) walks the 32-row steps of its range
// that hold a row of the adapter, with the other rows masked, and leaves an f32 partial and a
// flag; a second kernel sums the flagged partials in order.  A single range is the result itself
// (flag null).  COLS: the result is [n, J, R], else [n, R, J].
// ---------------------------------------------------------------------------------------
constexpr int kGradCols = 128;
constexpr int kGradWindow = 64;  // 32-row steps whose ids are looked at together

template <int RT, bool COLS>
__global__ __launch_bounds__(256) void lora_grad_kernel(LoraRows rows, int J, int R, const bf16* __restrict__ x,
                                                        long ldx, const float* __restrict__ u, int range,
                                                        float* __restrict__ part, int32_t* __restrict__ flag) {
  constexpr int XP = kGradCols + 4, UP = 16 * RT + 4;
  __shared__ __attribute__((aligned(16))) bf16 sx[32 * XP];
  __shared__ __attribute__((aligned(16))) bf16 su[3][32 * UP];
  __shared__ int s_any[kGradWindow];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid % kWave;
  const int lr = lane % 16, kg = lane / 16;
  const int j0 = kGradCols * blockIdx.x, a = blockIdx.y, split = blockIdx.z;
  const int mb = split * range, me = min(rows.M, mb + range), steps = (me - mb + 31) / 32;
  f32x4 acc[RT][2];
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int t = 0; t < 2; ++t) acc[r][t] = zero4();
  bool seen = false;
  for (int s = 0; s < steps; ++s) {
    const int q = s % kGradWindow;
    if (q == 0) {  // which of the next steps hold a row of the adapter
      __syncthreads();
      for (int w = wave; w < min(kGradWindow, steps - s); w += 4) {
        const int m = mb + 32 * (s + w) + lane;
        const bool any = __any(lane < 32 && m < me && rows.id(m) == a);
        if (lane == 0) s_any[w] = any;
      }
      __syncthreads();
    }
    if (!s_any[q]) continue;  // uniform
    seen = true;
    const int m1 = mb + 32 * s;
    __syncthreads();  // the previous step is read
    for (int c = tid; c < 32 * (kGradCols / 8); c += 256) {
      const int row = c / (kGradCols / 8), col = 8 * (c % (kGradCols / 8));
      // (rows of other adapters are zero too: whatever they hold stays out of the products)
      const bool in = m1 + row < me && j0 + col < J && rows.id(m1 + row) == a;
      const uint4 w = __builtin_bit_cast(
          uint4, keep8(*(const bf16x8*)(x + (in ? (size_t)(m1 + row) * ldx + j0 + col : (size_t)0)), in));
      uint2* d = (uint2*)(sx + row * XP + col);
      d[0] = make_uint2(w.x, w.y);
      d[1] = make_uint2(w.z, w.w);
    }
    for (int c = tid; c < 32 * 16 * RT; c += 256) {
      const int row = c / (16 * RT), r = c % (16 * RT);
      const bool in = m1 + row < me && r < R && rows.id(m1 + row) == a;
      float v = in ? u[(size_t)(m1 + row) * R + r] : 0.f;
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        const bf16 b = to_bf16(v);
        su[k][row * UP + r] = b;
        v -= (float)b;
      }
    }
    __syncthreads();
    bf16x8 fx[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) fx[t] = lds_col_frag(sx, XP, 0, 32 * wave + 16 * t, lane);
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        const bf16x8 fu = lds_col_frag(su[k], UP, 0, 16 * r, lane);
#pragma unroll
        for (int t = 0; t < 2; ++t) acc[r][t] = COLS ? mfma16(fx[t], fu, acc[r][t]) : mfma16(fu, fx[t], acc[r][t]);
      }
  }
  if (flag) {
    if (blockIdx.x == 0 && tid == 0) flag[split * rows.n + a] = seen;
    if (!seen) return;
  }
  float* out = part + ((size_t)split * rows.n + a) * R * J;
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int rr = 16 * r + (COLS ? lr : 4 * kg + i), j = j0 + 32 * wave + 16 * t + (COLS ? 4 * kg + i : lr);
        if (rr < R && j < J) out[COLS ? (size_t)j * R + rr : (size_t)rr * J + j] = acc[r][t][i];
      }
}

__global__ __launch_bounds__(256) void lora_grad_reduce_kernel(int splits, int n, long per,
                                                               const float* __restrict__ part,
                                                               const int32_t* __restrict__ flag,
                                                               float* __restrict__ out) {
  const int a = blockIdx.y;
  for (long i = ((long)blockIdx.x * 256 + threadIdx.x) * 4; i < per; i += (long)gridDim.x * 1024) {
    f32x4 v = zero4();
    for (int s = 0; s < splits; ++s)
      if (flag[s * n + a]) v += *(const f32x4*)(part + ((size_t)s * n + a) * per + i);
    *(f32x4*)(out + (size_t)a * per + i) = v;
  }
}

struct GradPlan {
  int range, splits;
};

// Ranges of rows: enough (column block, range) workgroups to fill the chip twice, and partials of
// at most 512 MB.
static GradPlan grad_plan(int64_t M, int32_t J, int32_t R, int32_t n) {
  const int64_t cols = (J + kGradCols - 1) / kGradCols;
  int64_t splits = (512 + cols - 1) / cols;
  const int64_t most = ((int64_t)512 << 20) / ((int64_t)n * R * J * 4);
  if (splits > most) splits = most;
  if (splits < 1) splits = 1;
  const int64_t range = ((M + splits - 1) / splits + 31) / 32 * 32;
  return {(int)range, (int)((M + range - 1) / range)};
}

}  // namespace kda

static int check_lora(const char* what, int64_t M, int32_t J, int32_t R, int32_t n, const void* ids,
                      int64_t rows_per_id) {
  KDA_REQUIRE(M >= 0 && M <= (1 << 30), "%s: invalid row count", what);
  KDA_REQUIRE(J > 0 && J % 8 == 0 && J <= (1 << 24), "%s: feature dimensions must be positive multiples of 8", what);
  KDA_REQUIRE(R > 0 && R % 8 == 0 && R <= 128, "%s: the rank must be a multiple of 8 and at most 128", what);
  KDA_REQUIRE(n > 0 && n <= 65535, "%s: the number of adapters must be in [1, 65535]", what);
  KDA_REQUIRE(M == 0 || ids, "%s: null ids", what);
  KDA_REQUIRE(rows_per_id > 0 && rows_per_id <= (1 << 30), "%s: invalid rows per id", what);
  return KDA_OK;
}

extern "C" int kda_lora_shrink(int64_t M, int32_t J, int32_t R, int32_t n, const int32_t* ids, int64_t rows_per_id,
                               const void* x, int64_t ldx, const void* factor, int32_t factor_cols, const float* scale,
                               float* u, hipStream_t stream) {
  using namespace kda;
  int rc = check_lora("lora_shrink", M, J, R, n, ids, rows_per_id);
  if (rc != KDA_OK) return rc;
  if (M == 0) return KDA_OK;
  KDA_REQUIRE(x && factor && u && aligned16(x, factor, u), "lora_shrink: null or unaligned pointer");
  KDA_REQUIRE(ldx >= J && ldx % 8 == 0, "lora_shrink: rows of x must be 16-byte aligned");
  const LoraRows rows{(int)M, n, ids, (int)rows_per_id};
  auto go = [&](auto kern, int mt) {
    hipLaunchKernelGGL(kern, dim3((unsigned)((M + 16 * mt - 1) / (16 * mt))), dim3(kShrinkWaves * kWave), 0, stream,
                       rows, J, R, (const bf16*)x, (long)ldx, (const bf16*)factor, scale, u);
  };
  // 32 rows share a read of the factor where that still leaves work for every CU
  auto pick = [&](auto k1, auto k2) { M >= 4096 ? go(k2, 2) : go(k1, 1); };
  if (factor_cols) {
    if (R <= 16) pick(lora_shrink_kernel<1, 1, true>, lora_shrink_kernel<1, 2, true>);
    else if (R <= 32) pick(lora_shrink_kernel<2, 1, true>, lora_shrink_kernel<2, 2, true>);
    else if (R <= 64) pick(lora_shrink_kernel<4, 1, true>, lora_shrink_kernel<4, 2, true>);
    else pick(lora_shrink_kernel<8, 1, true>, lora_shrink_kernel<8, 2, true>);
  } else {
    if (R <= 16) pick(lora_shrink_kernel<1, 1, false>, lora_shrink_kernel<1, 2, false>);
    else if (R <= 32) pick(lora_shrink_kernel<2, 1, false>, lora_shrink_kernel<2, 2, false>);
    else if (R <= 64) pick(lora_shrink_kernel<4, 1, false>, lora_shrink_kernel<4, 2, false>);
    else pick(lora_shrink_kernel<8, 1, false>, lora_shrink_kernel<8, 2, false>);
  }
  KDA_LAUNCH_CHECK("lora_shrink");
  return KDA_OK;
}

extern "C" int kda_lora_expand(int64_t M, int32_t J, int32_t R, int32_t n, const int32_t* ids, int64_t rows_per_id,
                               const float* u, const void* factor, int32_t factor_cols, void* y, int64_t ldy,
                               hipStream_t stream) {
  using namespace kda;
  int rc = check_lora("lora_expand", M, J, R, n, ids, rows_per_id);
  if (rc != KDA_OK) return rc;
  if (M == 0) return KDA_OK;
  KDA_REQUIRE(u && factor && y && aligned16(u, factor, y), "lora_expand: null or unaligned pointer");
  KDA_REQUIRE(ldy >= J && ldy % 8 == 0, "lora_expand: rows of y must be 16-byte aligned");
  const LoraRows rows{(int)M, n, ids, (int)rows_per_id};
  const dim3 grid((unsigned)((M + 63) / 64), (unsigned)((J + kExpandCols - 1) / kExpandCols));
  auto go = [&](auto kern) {
    hipLaunchKernelGGL(kern, grid, dim3(256), 0, stream, rows, J, R, u, (const bf16*)factor, (bf16*)y, (long)ldy);
  };
  if (factor_cols) {
    if (R <= 32) go(lora_expand_kernel<1, false>);
    else if (R <= 64) go(lora_expand_kernel<2, false>);
    else go(lora_expand_kernel<4, false>);
  } else {
    if (R <= 32) go(lora_expand_kernel<1, true>);
    else if (R <= 64) go(lora_expand_kernel<2, true>);
    else go(lora_expand_kernel<4, true>);
  }
  KDA_LAUNCH_CHECK("lora_expand");
  return KDA_OK;
}

extern "C" size_t kda_lora_grad_scratch_bytes(int64_t M, int32_t J, int32_t R, int32_t n) {
  if (M <= 0 || M > (1 << 30) || J <= 0 || R <= 0 || n <= 0) return 0;
  const kda::GradPlan p = kda::grad_plan(M, J, R, n);
  if (p.splits == 1) return 0;
  return kda::align256((size_t)p.splits * n * R * J * 4) + (size_t)p.splits * n * 4;
}

extern "C" int kda_lora_grad(int64_t M, int32_t J, int32_t R, int32_t n, const int32_t* ids, int64_t rows_per_id,
                             const void* x, int64_t ldx, const float* u, int32_t out_cols, float* grad, void* scratch,
                             hipStream_t stream) {
  using namespace kda;
  int rc = check_lora("lora_grad", M, J, R, n, ids, rows_per_id);
  if (rc != KDA_OK) return rc;
  KDA_REQUIRE(grad && aligned16(grad), "lora_grad: null or unaligned pointer");
  GradPlan p{32, 0};
  float* part = (float*)scratch;
  int32_t* flag = nullptr;
  if (M > 0) {
    KDA_REQUIRE(x && u && aligned16(x, u, scratch), "lora_grad: null or unaligned pointer");
    KDA_REQUIRE(ldx >= J && ldx % 8 == 0, "lora_grad: rows of x must be 16-byte aligned");
    p = grad_plan(M, J, R, n);
    if (p.splits == 1) {
      part = grad;
    } else {
      KDA_REQUIRE(scratch, "lora_grad: null scratch");
      flag = (int32_t*)((char*)scratch + align256((size_t)p.splits * n * R * J * 4));
    }
    const LoraRows rows{(int)M, n, ids, (int)rows_per_id};
    const dim3 grid((unsigned)((J + kGradCols - 1) / kGradCols), (unsigned)n, (unsigned)p.splits);
    auto go = [&](auto kern) {
      hipLaunchKernelGGL(kern, grid, dim3(256), 0, stream, rows, J, R, (const bf16*)x, (long)ldx, u, p.range, part,
                         flag);
    };
    if (out_cols) {
      if (R <= 16) go(lora_grad_kernel<1, true>);
      else if (R <= 32) go(lora_grad_kernel<2, true>);
      else if (R <= 64) go(lora_grad_kernel<4, true>);
      else go(lora_grad_kernel<8, true>);
    } else {
      if (R <= 16) go(lora_grad_kernel<1, false>);
      else if (R <= 32) go(lora_grad_kernel<2, false>);
      else if (R <= 64) go(lora_grad_kernel<4, false>);
      else go(lora_grad_kernel<8, false>);
    }
    KDA_LAUNCH_CHECK("lora_grad");
    if (p.splits == 1) return KDA_OK;
  }
  const long per = (long)R * J;
  const long blocks = (per / 4 + 255) / 256;
  hipLaunchKernelGGL(lora_grad_reduce_kernel, dim3((unsigned)(blocks < 1024 ? blocks : 1024), (unsigned)n), dim3(256), 0,
                     stream, p.splits, n, per, part, flag, grad);
  KDA_LAUNCH_CHECK("lora_grad reduce");
  return KDA_OK;
}
