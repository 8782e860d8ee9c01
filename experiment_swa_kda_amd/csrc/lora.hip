// Low-rank adapters of many requests beside a shared projection: row m of x belongs to adapter
// a = id(m) (none if outside [0, n)), and
//   y_m = W x_m + s_a B_a (A_a x_m)
// with A_a [R, K] and B_a [N, R] far smaller than W.  Three products with a factor F_a, each
// reading its long operand once:
//   shrink   u_m = s_a F_a x_m             (forward with A; the backward's t = s B^T dy with B)
//   expand   y_m = F_a^T u_m               (forward with B; the backward's A^T t with A)
//   grad     G_a = sum_{m of a} u_m x_m^T  (dB from s A x and dy; dA from t and x)
// F is read in either layout, [n, R, J] or [n, J, R] (J the long dimension), so neither direction
// needs a transposed copy.  u is f32, kept as three bf16 parts (lora_rows.hpp).
//
// A tile of rows may hold several adapters: each product runs once per distinct adapter of the
// tile, in ascending order, with the other rows masked.  A row's id is ids[m / rows_per_id].
#include "kda_device.hpp"
#include "kda_host.hpp"
#include "lora_rows.hpp"

namespace kda {

// ---------------------------------------------------------------------------------------
// shrink: one workgroup per 16 MT rows; its waves take 64 columns of J at a time each, and their
// partial tiles meet in LDS.  RT = ceil(R / 16).  Lanes load along rows (8 lanes to a 128-byte line:
// an MFMA fragment loaded directly has 16 rows in 16 neighbouring lanes, 64 cycles of address
// processing for its 1 KB instead of 16: 7777 x 4096 at rank 64 took 48 us, now 22, 2.9 TB/s) and pass the rows
// through an LDS stage of their own, so without a barrier; AHEAD groups of 64 columns are in flight.
// TRANSPOSED: F is [n, J, R], its fragments run down the stage's columns.
// ---------------------------------------------------------------------------------------
constexpr int kShrinkWaves = 8;

template <int RT, int MT, bool TRANSPOSED>
__global__ __launch_bounds__(kShrinkWaves * kWave) void lora_shrink_kernel(LoraRows rows, int seq_tiles, int J, int R,
                                                                          const bf16* __restrict__ x, long ldx,
                                                                          const bf16* __restrict__ f,
                                                                          const float* __restrict__ scale,
                                                                          bf16* __restrict__ u) {
  constexpr int AHEAD = RT >= 4 ? 1 : 2;
  constexpr int RG = RT < 4 ? RT : 4;    // rank tiles that pass through the stage together
  constexpr int PITCH = 16 * RT + 4;     // TRANSPOSED: elements; 8-byte aligned rows for the transposing reads
  constexpr int XB = 16 * MT * 128, FB = TRANSPOSED ? 32 * PITCH * 2 : 16 * RG * 128, STAGE = (XB + FB + 15) / 16 * 16;
  constexpr int PART = kShrinkWaves * RT * MT * kWave * 16;
  __shared__ __attribute__((aligned(16))) char smem[kShrinkWaves * STAGE > PART ? kShrinkWaves * STAGE : PART];
  f32x4(*part)[RT * MT][kWave] = reinterpret_cast<f32x4(*)[RT * MT][kWave]>(smem);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave;
  const int lr = lane % 16, kg = lane / 16;
  const size_t plane = (size_t)rows.M * R;
  int m0 = 16 * MT * blockIdx.x;
  if (seq_tiles) {  // tiles that end with their sequence, so that none has two adapters
    const int seq = blockIdx.x / seq_tiles;
    m0 = seq * rows.rows_per_id + 16 * MT * (blockIdx.x % seq_tiles);
    rows.M = (seq + 1) * rows.rows_per_id;
  }
  const int my_id = rows.id(m0 + lane % (16 * MT));
  char* sx = smem + wave * STAGE;
  char* sf = sx + XB;
  const int groups = (J + 63) / 64;
  const int row8 = lane / 8, chunk8 = lane % 8;  // a load covers eight rows of 64 columns
  for (int a = next_adapter(my_id, -1); a != kNoAdapter; a = next_adapter(my_id, a)) {
    const bf16* fa = f + (size_t)a * R * J;
    f32x4 acc[RT][MT];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int t = 0; t < MT; ++t) acc[r][t] = zero4();
    for (int s0 = wave; s0 < groups; s0 += AHEAD * kShrinkWaves) {
      bf16x8 vx[AHEAD][2 * MT], vf[AHEAD][2 * RT];
#pragma unroll
      for (int q = 0; q < AHEAD; ++q) {
        const int j0 = 64 * (s0 + q * kShrinkWaves), j = j0 + 8 * chunk8;
        const bool ok = j < J;  // J is a multiple of 8: eight columns are all in or all out
#pragma unroll
        for (int v = 0; v < 2 * MT; ++v)
          vx[q][v] = keep8(*(const bf16x8*)(x + (size_t)min(m0 + 8 * v + row8, rows.M - 1) * ldx + (ok ? j : 0)), ok);
#pragma unroll
        for (int v = 0; v < 2 * RT; ++v) {
          if constexpr (TRANSPOSED) {  // vector c of 64 rows of R columns, 8 to a vector
            const int c = v * kWave + lane, row = j0 + c / (2 * RT), col = 8 * (c % (2 * RT));
            const bool in = row < J && col < R;
            vf[q][v] = keep8(*(const bf16x8*)(fa + (in ? (size_t)row * R + col : (size_t)0)), in);
          } else {
            vf[q][v] = keep8(*(const bf16x8*)(fa + (size_t)min(8 * v + row8, R - 1) * J + (ok ? j : 0)), ok);
          }
        }
      }
#pragma unroll
      for (int q = 0; q < AHEAD; ++q) {
        asm volatile("" ::: "memory");
#pragma unroll
        for (int v = 0; v < 2 * MT; ++v) *(bf16x8*)(sx + row64_off(8 * v + row8, chunk8)) = vx[q][v];
        if constexpr (TRANSPOSED) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {  // 32 of the 64 rows at a time
            asm volatile("" ::: "memory");
#pragma unroll
            for (int v = 0; v < RT; ++v) {
              const int c = v * kWave + lane;
              const uint4 w = __builtin_bit_cast(uint4, vf[q][h * RT + v]);
              uint2* d = (uint2*)((bf16*)sf + c / (2 * RT) * PITCH + 8 * (c % (2 * RT)));
              d[0] = make_uint2(w.x, w.y);
              d[1] = make_uint2(w.z, w.w);
            }
            asm volatile("" ::: "memory");
            bf16x8 fx[MT];
#pragma unroll
            for (int t = 0; t < MT; ++t) fx[t] = *(const bf16x8*)(sx + row64_off(16 * t + lr, 4 * h + kg));
#pragma unroll
            for (int r = 0; r < RT; ++r) {
              const bf16x8 ff = lds_col_frag((const bf16*)sf, PITCH, 0, 16 * r, lane);
#pragma unroll
              for (int t = 0; t < MT; ++t) acc[r][t] = mfma16(ff, fx[t], acc[r][t]);
            }
          }
        } else {
#pragma unroll
          for (int g = 0; g < RT; g += RG) {
            asm volatile("" ::: "memory");
#pragma unroll
            for (int v = 0; v < 2 * RG; ++v) *(bf16x8*)(sf + row64_off(8 * v + row8, chunk8)) = vf[q][2 * g + v];
            asm volatile("" ::: "memory");
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              bf16x8 fx[MT];
#pragma unroll
              for (int t = 0; t < MT; ++t) fx[t] = *(const bf16x8*)(sx + row64_off(16 * t + lr, 4 * h + kg));
#pragma unroll
              for (int r = 0; r < RG; ++r) {
                const bf16x8 ff = *(const bf16x8*)(sf + row64_off(16 * r + lr, 4 * h + kg));
#pragma unroll
                for (int t = 0; t < MT; ++t) acc[g + r][t] = mfma16(ff, fx[t], acc[g + r][t]);
              }
            }
          }
        }
      }
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
      if (rows.id(m) == a && r < R) {
        bf16x4 p0, p1, p2;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          bf16 c0, c1, c2;
          split3(v[i] * s, c0, c1, c2);
          p0[i] = c0;
          p1[i] = c1;
          p2[i] = c2;
        }
        bf16* d = u + (size_t)m * R + r;
        *(bf16x4*)d = p0;
        *(bf16x4*)(d + plane) = p1;
        *(bf16x4*)(d + 2 * plane) = p2;
      }
    }
    __syncthreads();  // the next adapter's stages overwrite the partials
  }
  // rows of no adapter
  for (int q = threadIdx.x; q < 16 * MT * (R / 8); q += kShrinkWaves * kWave) {
    const int m = m0 + q / (R / 8);
    if (m < rows.M && rows.id(m) < 0)
#pragma unroll
      for (int k = 0; k < 3; ++k) *(uint4*)(u + k * plane + (size_t)m * R + 8 * (q % (R / 8))) = make_uint4(0, 0, 0, 0);
  }
}

// ---------------------------------------------------------------------------------------
// expand: 64 rows x 256 columns per workgroup; wave w has rows 16 w .. and keeps their u in
// registers.  KS = ceil(R / 32) steps of the contraction.  F passes through LDS in pieces of 64
// columns, the next piece on its way; so does the result, to be stored along rows.  TRANSPOSED: F is
// [n, R, J].  Bound by the write of y: 7777 x 2048 and x 4096 at rank 64 take 15 and 23 us (2.1 and 2.8
// TB/s), 8192 x 32768 at rank 16 159 us (3.4).
// ---------------------------------------------------------------------------------------
constexpr int kExpandCols = 256;

template <int KS, bool TRANSPOSED>
__global__ __launch_bounds__(256) void lora_expand_kernel(LoraRows rows, int J, int R, const bf16* __restrict__ u,
                                                          const bf16* __restrict__ f, bf16* __restrict__ y, long ldy) {
  constexpr int PITCH = TRANSPOSED ? 64 + 8 : 32 * KS + 8;  // elements of a row of the piece: [rank][column], [column][rank]
  __shared__ __attribute__((aligned(16))) bf16 st[(TRANSPOSED ? 32 * KS : 64) * PITCH];
  __shared__ __attribute__((aligned(16))) char s_out[4][16 * 128];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid % kWave;
  const int lr = lane % 16, kg = lane / 16;
  const int m0 = 64 * blockIdx.x, m = m0 + 16 * wave + lr;
  const int tile_id = rows.id(m0 + lane), my_id = rows.id(m);
  char* out = s_out[wave];
  bf16x8 hi[KS], lo[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const int r = 32 * s + 8 * kg;
    const bool ok = m < rows.M && r < R;
    const bf16* pu = u + (ok ? (size_t)m * R + r : (size_t)0);
    hi[s] = keep8(*(const bf16x8*)pu, ok);
    lo[s] = keep8(*(const bf16x8*)(pu + (size_t)rows.M * R), ok);
  }
  const int c_end = min(J, kExpandCols * ((int)blockIdx.y + 1)), first = next_adapter(tile_id, -1);
  bf16x8 piece[KS];
  auto load = [&](int c0, int a) {
    const bf16* fa = f + (size_t)a * R * J;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int c = s * 256 + tid;
      if constexpr (TRANSPOSED) {
        const int r = c / 8, j = c0 + 8 * (c % 8);
        const bool in = r < R && j < J;
        piece[s] = keep8(*(const bf16x8*)(fa + (in ? (size_t)r * J + j : (size_t)0)), in);
      } else {
        const int j = c0 + c / (4 * KS), r = 8 * (c % (4 * KS));
        const bool in = r < R && j < J;
        piece[s] = keep8(*(const bf16x8*)(fa + (in ? (size_t)j * R + r : (size_t)0)), in);
      }
    }
  };
  int c0 = kExpandCols * blockIdx.y, a = first;
  if (first != kNoAdapter) load(c0, a);
  f32x4 acc[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) acc[t] = zero4();
  while (c0 < c_end) {  // pieces in order: the adapters of a block of columns, then the next block
    const int now = a;
    bool last = true;
    if (first != kNoAdapter) {
      __syncthreads();  // the previous piece is read
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int c = s * 256 + tid, per = TRANSPOSED ? 8 : 4 * KS;
        *(bf16x8*)(st + c / per * PITCH + 8 * (c % per)) = piece[s];
      }
      a = next_adapter(tile_id, now);
      last = a == kNoAdapter;
      if (last) a = first;
      if (!last || c0 + 64 < c_end) load(last ? c0 + 64 : c0, a);  // in flight over this piece's products
      wait_lgkm0();
      ring_barrier();
      f32x4 d[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) d[t] = zero4();
#pragma unroll
      for (int s = 0; s < KS; ++s) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          bf16x8 ff;
          if constexpr (TRANSPOSED)
            ff = lds_col_frag(st, PITCH, 32 * s, 16 * t, lane);
          else
            ff = *(const bf16x8*)(st + (16 * t + lr) * PITCH + 32 * s + 8 * kg);
          d[t] = mfma16(ff, hi[s], d[t]);
          d[t] = mfma16(ff, lo[s], d[t]);
        }
      }
      // (chosen, not multiplied by zero: an infinity in this adapter stays out of other rows)
      const bool mine = my_id == now;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[t][i] = mine ? d[t][i] : acc[t][i];
      if (!last) continue;
    }
    // accumulator: column c0 + 16 t + 4 kg + i, row lr of the wave's 16; stored along rows (as loads: a
    // store of 16 rows from 16 neighbouring lanes takes four times as long)
    asm volatile("" ::: "memory");
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      bf16x4 o;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = to_bf16(acc[t][i]);
      *(bf16x4*)(out + row64_off(lr, 2 * t + kg / 2) + 8 * (kg % 2)) = o;
      acc[t] = zero4();
    }
    asm volatile("" ::: "memory");
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int row = 8 * p + lane / 8, mr = m0 + 16 * wave + row, j = c0 + 8 * (lane % 8);
      if (mr < rows.M && j < J) *(bf16x8*)(y + (size_t)mr * ldy + j) = *(const bf16x8*)(out + row64_off(row, lane % 8));
    }
    c0 += 64;
  }
}

// Rows that each have an id of their own (a token of every request): tiles would hold as many
// adapters as rows, so every row takes its own products with vector FMAs (lora_shrink_rows_kernel,
// and here a thread per column of y, whose R factors lie together).  Rank 16, 384 -> 1536, shrink + expand
// + the library's product, ids drawn from 8 and from M adapters, against tiles: M 256 12 and 12 us (36
// and 149), M 1024 23 and 24 (39 and 195); beyond, neighbours mostly share an adapter (M 2048, four runs: 36
// us against 21).
constexpr int kLoraRowsMost = 1024;
__global__ __launch_bounds__(256) void lora_expand_rows_kernel(LoraRows rows, int J, int R, const bf16* __restrict__ u,
                                                               const bf16* __restrict__ f, bf16* __restrict__ y,
                                                               long ldy) {
  const int m = blockIdx.x, j = 256 * blockIdx.y + threadIdx.x, a = rows.id(m);
  if (j >= J) return;
  float s = 0.f;
  if (a >= 0) {
    const bf16* pf = f + ((size_t)a * J + j) * R;
    const bf16* pu = u + (size_t)m * R;
    const size_t plane = (size_t)rows.M * R;
#pragma unroll 2
    for (int r = 0; r < R; r += 8) {
      const bf16x8 v = *(const bf16x8*)(pf + r), u0 = *(const bf16x8*)(pu + r), u1 = *(const bf16x8*)(pu + plane + r);
#pragma unroll
      for (int e = 0; e < 8; ++e) s = fmaf((float)u0[e] + (float)u1[e], (float)v[e], s);
    }
  }
  y[(size_t)m * ldy + j] = to_bf16(s);
}

// ---------------------------------------------------------------------------------------
// grad: workgroup (128 columns of J, adapter, range of rows) walks the 64-row steps of its range
// that hold a row of the adapter, with the other rows masked and the next step's loads in flight, and
// leaves an f32 partial and a flag; a second kernel sums the flagged partials in order.  A single
// range is the result itself (flag null).  COLS: the result is [n, J, R], else [n, R, J].
// Bound by reading x once and u's three parts for every 128 columns: 8192 x 32768 at rank 16 takes 128 us
// with the sum (4.2 TB/s of x), 7777 x 4096 at rank 64 45 us (1.4: there u's parts are more than x, and the
// ranges' partials 22 MB).
// ---------------------------------------------------------------------------------------
constexpr int kGradCols = 128;
constexpr int kGradRows = 64;
constexpr int kGradWindow = 32;  // steps whose ids are looked at together

template <int RT, bool COLS>
__global__ __launch_bounds__(256) void lora_grad_kernel(LoraRows rows, int J, int R, const bf16* __restrict__ x,
                                                        long ldx, const bf16* __restrict__ u, int range,
                                                        float* __restrict__ part, int32_t* __restrict__ flag) {
  constexpr int XP = kGradCols + 8, UP = 16 * RT + 8;  // pitches: 16-byte rows, 4 banks apart
  constexpr int XV = kGradRows * kGradCols / 8 / 256;  // vectors of a step and thread
  constexpr int UN = 3 * kGradRows * 2 * RT, UV = (UN + 255) / 256;
  __shared__ __attribute__((aligned(16))) bf16 sx[kGradRows * XP];
  __shared__ __attribute__((aligned(16))) bf16 su[3][kGradRows * UP];
  __shared__ int s_any[kGradWindow];
  __shared__ int s_id[kGradRows * kGradWindow];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid % kWave;
  const int j0 = kGradCols * blockIdx.x, a = blockIdx.y, split = blockIdx.z;
  const int mb = split * range, me = min(rows.M, mb + range), steps = (me - mb + kGradRows - 1) / kGradRows;
  f32x4 acc[RT][2];
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int t = 0; t < 2; ++t) acc[r][t] = zero4();
  bool seen = false;
  for (int w0 = 0; w0 < steps; w0 += kGradWindow) {  // which of the next steps hold a row of the adapter
    const int wn = min(kGradWindow, steps - w0);
    __syncthreads();
    for (int s = wave; s < wn; s += 4) {
      const int i = kGradRows * s + lane, m = mb + kGradRows * w0 + i, id = m < me ? rows.id(m) : -1;
      s_id[i] = id;
      const bool any = __any(id == a);
      if (lane == 0) s_any[s] = any;
    }
    __syncthreads();
    auto next = [&](int s) {
      while (s < wn && !s_any[s]) ++s;
      return __builtin_amdgcn_readfirstlane(s);
    };
    bf16x8 vx[XV], vu[UV];
    auto load = [&](int s) {
      const int m1 = mb + kGradRows * (w0 + s);
#pragma unroll
      for (int q = 0; q < XV; ++q) {
        const int c = q * 256 + tid, row = c / (kGradCols / 8), col = 8 * (c % (kGradCols / 8));
        // (rows of other adapters are zero: whatever they hold stays out of the products)
        const bool in = j0 + col < J && s_id[kGradRows * s + row] == a;
        vx[q] = keep8(*(const bf16x8*)(x + (in ? (size_t)(m1 + row) * ldx + j0 + col : (size_t)0)), in);
      }
#pragma unroll
      for (int q = 0; q < UV; ++q) {
        const int c = q * 256 + tid, k = c / (UN / 3), row = c / (2 * RT) % kGradRows, r = 8 * (c % (2 * RT));
        const bool in = c < UN && r < R && s_id[kGradRows * s + row] == a;
        vu[q] = keep8(*(const bf16x8*)(u + (in ? ((size_t)k * rows.M + m1 + row) * R + r : (size_t)0)), in);
      }
    };
    int s = next(0);
    if (s < wn) load(s);
    while (s < wn) {
      seen = true;
      __syncthreads();  // the previous step is read
#pragma unroll
      for (int q = 0; q < XV; ++q) {
        const int c = q * 256 + tid;
        *(bf16x8*)(sx + c / (kGradCols / 8) * XP + 8 * (c % (kGradCols / 8))) = vx[q];
      }
#pragma unroll
      for (int q = 0; q < UV; ++q) {
        const int c = q * 256 + tid;
        if (c < UN) *(bf16x8*)(su[c / (UN / 3)] + c / (2 * RT) % kGradRows * UP + 8 * (c % (2 * RT))) = vu[q];
      }
      s = next(s + 1);
      if (s < wn) load(s);  // in flight over this step's products
      wait_lgkm0();
      ring_barrier();
#pragma unroll
      for (int h = 0; h < kGradRows / 32; ++h) {
        bf16x8 fx[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) fx[t] = lds_col_frag(sx, XP, 32 * h, 32 * wave + 16 * t, lane);
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int k = 0; k < 3; ++k) {
            const bf16x8 fu = lds_col_frag(su[k], UP, 32 * h, 16 * r, lane);
#pragma unroll
            for (int t = 0; t < 2; ++t) acc[r][t] = COLS ? mfma16(fx[t], fu, acc[r][t]) : mfma16(fu, fx[t], acc[r][t]);
          }
      }
    }
  }
  if (flag) {
    if (blockIdx.x == 0 && tid == 0) flag[split * rows.n + a] = seen;
    if (!seen) return;
  }
  const int lr = lane % 16, kg = lane / 16;
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

// The flagged partials of every element, in order: a workgroup lists them, its four waves take every
// fourth one, eight loads in flight, and their sums meet in LDS.
constexpr int kGradSplits = 512;
__global__ __launch_bounds__(256) void lora_grad_reduce_kernel(int splits, int n, long per,
                                                               const float* __restrict__ part,
                                                               const int32_t* __restrict__ flag,
                                                               float* __restrict__ out) {
  __shared__ int list[kGradSplits], s_count;
  __shared__ f32x4 red[4][kWave];
  const int a = blockIdx.y, g = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const long i = ((long)blockIdx.x * kWave + lane) * 4, ic = i < per ? i : 0;
  if (g == 0) {
    int count = 0;
    for (int s0 = 0; s0 < splits; s0 += kWave) {
      const int s = s0 + lane;
      const bool on = s < splits && flag[s * n + a];
      const unsigned long long m = __ballot(on);
      if (on) list[count + __popcll(m & ((1ull << lane) - 1))] = s;
      count += __popcll(m);
    }
    if (lane == 0) s_count = count;
  }
  __syncthreads();
  const int count = s_count;
  f32x4 v = zero4();
  for (int k0 = g; k0 < count; k0 += 32) {
    f32x4 p[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const int k = k0 + 4 * q;
      p[q] = *(const f32x4*)(part + ((size_t)list[k < count ? k : g] * n + a) * per + ic);
      if (k >= count) p[q] = zero4();
    }
#pragma unroll
    for (int q = 0; q < 8; ++q) v += p[q];
  }
  red[g][lane] = v;
  __syncthreads();
  if (g == 0 && i < per) *(f32x4*)(out + (size_t)a * per + i) = ((red[0][lane] + red[1][lane]) + red[2][lane]) + red[3][lane];
}

struct GradPlan {
  int range, splits;
};

// Ranges of rows: enough (column block, range) workgroups to fill the chip twice, and partials of
// at most 512 MB.
// Ranges for 512 workgroups of one adapter; more of them shorten a range but add partials (8192 x 4096 at
// rank 32: 32 / 27 / 29 / 32 us for 512 / 768 / 1024 / 1536, 7777 x 4096 at rank 64 39 / 41 / 36 / 44,
// 8192 x 1536 at rank 16 18 / 18 / 21 / 26).  Partials stay under 512 MB.
static GradPlan grad_plan(int64_t M, int32_t J, int32_t R, int32_t n) {
  const int64_t cols = (J + kGradCols - 1) / kGradCols;
  int64_t splits = (kGradSplits + cols - 1) / cols;
  const int64_t most = ((int64_t)512 << 20) / ((int64_t)n * R * J * 4);
  if (splits > most) splits = most;
  if (splits < 1) splits = 1;
  const int64_t range = ((M + splits - 1) / splits + kGradRows - 1) / kGradRows * kGradRows;
  return {(int)range, (int)((M + range - 1) / range)};
}

}  // namespace kda

extern "C" int kda_lora_shrink(int64_t M, int32_t J, int32_t R, int32_t n, const int32_t* ids, int64_t rows_per_id,
                               const void* x, int64_t ldx, const void* factor, int32_t factor_cols, const float* scale,
                               void* u, hipStream_t stream) {
  using namespace kda;
  int rc = kda::check_lora("lora_shrink", M, J, R, n, ids, rows_per_id);
  if (rc != KDA_OK) return rc;
  if (M == 0) return KDA_OK;
  KDA_REQUIRE(x && factor && u && aligned16(x, factor, u), "lora_shrink: null or unaligned pointer");
  KDA_REQUIRE(ldx >= J && ldx % 8 == 0, "lora_shrink: rows of x must be 16-byte aligned");
  const LoraRows rows{(int)M, n, ids, (int)rows_per_id};
  if (rows_per_id == 1 && M <= kLoraRowsMost && !factor_cols) {
    hipLaunchKernelGGL(lora_shrink_rows_kernel<4>, dim3((unsigned)M, (unsigned)((R + 3) / 4)), dim3(256), 0, stream, rows,
                       J, R, (const bf16*)x, (long)ldx, (const bf16*)factor, scale, (bf16*)u);
    KDA_LAUNCH_CHECK("lora_shrink");
    return KDA_OK;
  }
  auto go = [&](auto kern, int mt) {
    // a tile of two adapters takes two passes, twice the time of the only round of tiles that M 7777 is
    // (28 us against 18); tiles of their own per sequence are at most a quarter more of them
    const int tile = 16 * mt;
    const bool own = rows_per_id >= 4 * tile && M % rows_per_id == 0;
    const int seq_tiles = own ? (int)((rows_per_id + tile - 1) / tile) : 0;
    const int64_t grid = own ? M / rows_per_id * seq_tiles : (M + tile - 1) / tile;
    hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(kShrinkWaves * kWave), 0, stream, rows, seq_tiles, J, R,
                       (const bf16*)x, (long)ldx, (const bf16*)factor, scale, (bf16*)u);
  };
  // 32 rows share a read of the factor where there are more than 16 for every CU (x from memory, us, tiles of
  // 32 / 16: 6144 x 4096 at rank 64 20 / 26, 8192 x 4096 at rank 128 31 / 44, 8192 x 1536 at rank 16 8.3 / 8.6, but
  // 4096 x 4096 at rank 64 19 / 15)
  auto pick = [&](auto k1, auto k2) { M > 4096 ? go(k2, 2) : go(k1, 1); };
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
                               const void* u, const void* factor, int32_t factor_cols, void* y, int64_t ldy,
                               hipStream_t stream) {
  using namespace kda;
  int rc = kda::check_lora("lora_expand", M, J, R, n, ids, rows_per_id);
  if (rc != KDA_OK) return rc;
  if (M == 0) return KDA_OK;
  KDA_REQUIRE(u && factor && y && aligned16(u, factor, y), "lora_expand: null or unaligned pointer");
  KDA_REQUIRE(ldy >= J && ldy % 8 == 0, "lora_expand: rows of y must be 16-byte aligned");
  const LoraRows rows{(int)M, n, ids, (int)rows_per_id};
  if (rows_per_id == 1 && M <= kLoraRowsMost && factor_cols) {
    hipLaunchKernelGGL(lora_expand_rows_kernel, dim3((unsigned)M, (unsigned)((J + 255) / 256)), dim3(256), 0, stream,
                       rows, J, R, (const bf16*)u, (const bf16*)factor, (bf16*)y, (long)ldy);
    KDA_LAUNCH_CHECK("lora_expand");
    return KDA_OK;
  }
  const dim3 grid((unsigned)((M + 63) / 64), (unsigned)((J + kExpandCols - 1) / kExpandCols));
  auto go = [&](auto kern) {
    hipLaunchKernelGGL(kern, grid, dim3(256), 0, stream, rows, J, R, (const bf16*)u, (const bf16*)factor, (bf16*)y, (long)ldy);
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
                             const void* x, int64_t ldx, const void* u, int32_t out_cols, float* grad, void* scratch,
                             hipStream_t stream) {
  using namespace kda;
  int rc = kda::check_lora("lora_grad", M, J, R, n, ids, rows_per_id);
  if (rc != KDA_OK) return rc;
  KDA_REQUIRE(grad && aligned16(grad), "lora_grad: null or unaligned pointer");
  GradPlan p{kGradRows, 0};
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
      hipLaunchKernelGGL(kern, grid, dim3(256), 0, stream, rows, J, R, (const bf16*)x, (long)ldx, (const bf16*)u, p.range, part,
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
  hipLaunchKernelGGL(lora_grad_reduce_kernel, dim3((unsigned)((per / 4 + kWave - 1) / kWave), (unsigned)n), dim3(256), 0,
                     stream, p.splits, n, per, part, flag, grad);
  KDA_LAUNCH_CHECK("lora_grad reduce");
  return KDA_OK;
}
