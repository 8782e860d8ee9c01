// Losses on the log-probabilities of given tokens under soft-capped bf16 logits: what a
// pretrained decoder is trained on next.  With z = cap tanh(l / cap) over the vocabulary columns
// of a row, lse = log sum_j e^z_j and p = e^(z - lse),
//   logp = z_y - lse,   H = lse - sum_j p_j z_j          (target y, entropy)
//   dl_j = (1 - (z_j / cap)^2) [ g ([j = y] - p_j) - h p_j (z_j - lse + H) ]
// for the row's upstream gradients g of logp and h of H.  The losses only differ in what they make
// of logp and in the g they come back with (one thread's work per row):
//   policy      w (-min(rho A, clip(rho, lo, hi) A) + c (e^d - d - 1)),  rho = e^(logp - old), d = ref - logp
//   preference  mean over pairs of -(1 - s) log sigmoid(m) - s log sigmoid(-m), m = beta times the
//               difference of the two sequences' summed (or mean) log-probabilities, each less its reference
// Rows without a target (or without weight) are not read: whatever their logits hold, their
// outputs and gradients are zero.
#include "kda_device.hpp"
#include "kda_host.hpp"
#include "softcap_table.hpp"

namespace kda {

constexpr int kTokThreads = 256;
constexpr int kTokBatch = 8;                          // 16-byte vectors in flight per lane
constexpr int kTokChunk = kWave * 8 * kTokBatch;      // columns of one item
constexpr int kTokFwdPerCu = 4, kTokPairPerCu = 2;    // workgroups per CU: 33 KB and 66 KB tables

// One 4096-column chunk of a row per wave; columns from `last` on re-read the vector at `last`.
__device__ __forceinline__ void tok_load(const bf16* __restrict__ row, long c0, long last, bf16x8* x) {
  const long c = c0 + (threadIdx.x % kWave) * 8;
#pragma unroll
  for (int b = 0; b < kTokBatch; ++b) {
    const long cb = c + b * kWave * 8;
    x[b] = *reinterpret_cast<const bf16x8*>(row + (cb < last ? cb : last));
  }
}

// logp, lse and entropy of a row from its sums se = sum e^z, sz = sum z e^z, in 64 bits: the
// sums over a sequence that the losses take, and their differences, keep what f32 rows would lose.
__device__ __forceinline__ void tok_finish(float se, float sz, float raw, float cap, bool in_range, bool entropy,
                                           double& logp, double& lse, double& ent) {
  lse = log((double)se);
  logp = in_range ? (double)cap * tanh((double)raw / (double)cap) - lse : (double)__builtin_nanf("");
  ent = entropy ? lse - (double)sz / (double)se : 0.0;
}

// Forward: one wave per row, the next item's loads in flight while one is summed.  TabT: float
// (e^z) or float2 (e^z, z e^z) with the entropy.
template <bool ENT>
__global__ __launch_bounds__(kTokThreads) void token_fwd_kernel(long rows, int vocab, long stride, float cap,
                                                                const bf16* __restrict__ logits,
                                                                const int64_t* __restrict__ targets,
                                                                int64_t ignore_index, float* __restrict__ logp_row,
                                                                double* __restrict__ logp64_row,
                                                                float* __restrict__ lse_row,
                                                                float* __restrict__ ent_row) {
  using TabT = typename std::conditional<ENT, float2, float>::type;
  __shared__ TabT tab[kTabSize];
  for (int i = threadIdx.x; i < kTabSize; i += kTokThreads) {
    const float z = cap * tanhf(tab_pattern_value(i) / cap), e = expf(z);
    if constexpr (ENT)
      tab[i] = make_float2(e, z * e);
    else
      tab[i] = e;
  }
  __syncthreads();
  const TabT* tabz = tab - (kTabELo << 7);
  const int lane = threadIdx.x % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const long last = ((vocab - 1) / 8) * 8;  // last vector start that holds a vocabulary column
  const int nch = (vocab + kTokChunk - 1) / kTokChunk;
  for (long k = (long)blockIdx.x * (kTokThreads / kWave) + wave; k < rows; k += (long)gridDim.x * (kTokThreads / kWave)) {
    const long r = rows - 1 - k;  // last to first: the rows written last are still cached
    const int64_t y = targets[r];
    if (y == ignore_index) {
      if (lane == 0) {
        if (logp_row) logp_row[r] = 0.f;
        if (logp64_row) logp64_row[r] = 0.0;
        if (lse_row) lse_row[r] = 0.f;
        if (ENT) ent_row[r] = 0.f;
      }
      continue;
    }
    const bf16* row = logits + r * stride;
    float se = 0.f, sz = 0.f;
    u16x2 mag = (u16x2)0;  // running maximum of the magnitude bits (NaN detection)
    auto consume = [&](int ch, const bf16x8* x) {
      const int c0 = ch * kTokChunk + lane * 8;
#pragma unroll
      for (int b = 0; b < kTokBatch; ++b) {
        const int c = c0 + b * kWave * 8;
        const uint4 w = __builtin_bit_cast(uint4, x[b]);
        const unsigned ws[4] = {w.x, w.y, w.z, w.w};
        float be = 0.f, bz = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          int i0, i1;
          tab_index2_biased(ws[e], i0, i1);
          const bool k0 = c + 2 * e < vocab, k1 = c + 2 * e + 1 < vocab;
          const unsigned m = ws[e] & ((k0 ? 0x7fffu : 0u) | (k1 ? 0x7fff0000u : 0u));
          mag = __builtin_elementwise_max(mag, __builtin_bit_cast(u16x2, m));
          const TabT v0 = tabz[i0], v1 = tabz[i1];
          if constexpr (ENT) {
            be += (k0 ? v0.x : 0.f) + (k1 ? v1.x : 0.f);
            bz += (k0 ? v0.y : 0.f) + (k1 ? v1.y : 0.f);
          } else {
            be += (k0 ? v0 : 0.f) + (k1 ? v1 : 0.f);
          }
        }
        se += be;
        sz += bz;
      }
    };
    bf16x8 xa[kTokBatch], xb[kTokBatch];
    tok_load(row, 0, last, xa);
    for (int ch = 0; ch < nch; ch += 2) {
      if (ch + 1 < nch) tok_load(row, (long)(ch + 1) * kTokChunk, last, xb);
      consume(ch, xa);
      if (ch + 1 >= nch) break;
      if (ch + 2 < nch) tok_load(row, (long)(ch + 2) * kTokChunk, last, xa);
      consume(ch + 1, xb);
    }
    const bool nan_here = mag.x > 0x7f80 || mag.y > 0x7f80;
    se = wave_sum(nan_here ? __builtin_nanf("") : se);
    if (ENT) sz = wave_sum(sz);
    if (lane == 0) {
      const bool in_range = y >= 0 && y < vocab;
      double lp, lse, ent;
      tok_finish(se, sz, in_range ? (float)row[y] : 0.f, cap, in_range, ENT, lp, lse, ent);
      if (logp_row) logp_row[r] = (float)lp;
      if (logp64_row) logp64_row[r] = lp;
      if (lse_row) lse_row[r] = (float)lse;
      if (ENT) ent_row[r] = (float)ent;
    }
  }
}

// Backward for given row gradients: g of logp (times *scale if given) and, with ENT, h of the
// entropy.  Nothing is reduced, so (row, chunk) items go to the waves in order.
template <bool ENT>
__global__ __launch_bounds__(kTokThreads) void token_bwd_kernel(
    long rows, int vocab, long stride, float cap, const bf16* __restrict__ logits, const int64_t* __restrict__ targets,
    int64_t ignore_index, const float* __restrict__ lse_row, const float* __restrict__ ent_row,
    const float* __restrict__ g_row, const float* __restrict__ h_row, const float* __restrict__ scale,
    bf16* __restrict__ grad) {
  __shared__ float2 tab[kTabSize];  // (e^z, 1 - tanh^2), with the entropy (e^z, tanh)
  for (int i = threadIdx.x; i < kTabSize; i += kTokThreads) {
    const float th = tanhf(tab_pattern_value(i) / cap);
    tab[i] = make_float2(expf(cap * th), ENT ? th : 1.0f - th * th);
  }
  __syncthreads();
  const int lane = threadIdx.x % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int nch = (int)((stride + kTokChunk - 1) / kTokChunk);
  const long items = rows * nch;
  const float up = scale ? *scale : 1.f;
  for (long j = (long)blockIdx.x * (kTokThreads / kWave) + wave; j < items; j += (long)gridDim.x * (kTokThreads / kWave)) {
    const long r = j / nch;
    const int c0 = (int)(j - r * nch) * kTokChunk + lane * 8;
    const int64_t y = targets[r];
    const bool on = y != ignore_index;
    float g = on && g_row ? g_row[r] * up : 0.f, h = ENT && on && h_row ? h_row[r] * up : 0.f;
    bf16* q = grad + r * stride;
    if (g == 0.f && h == 0.f) {
#pragma unroll
      for (int b = 0; b < kTokBatch; ++b) {
        const int c = c0 + b * kWave * 8;
        if (c < stride) *reinterpret_cast<uint4*>(q + c) = make_uint4(0, 0, 0, 0);
      }
      continue;
    }
    bf16x8 x[kTokBatch];
    tok_load(logits + r * stride, c0 - lane * 8, stride - 8, x);
    const float lse = lse_row[r], einv = expf(-lse);
    const float ent = ENT ? ent_row[r] : 0.f;
    const int tc = y >= 0 && y < vocab ? (int)y : -1;
    if (tc < 0) g = __builtin_nanf("");  // out-of-range target: its log-probability is NaN
#pragma unroll
    for (int b = 0; b < kTokBatch; ++b) {
      const int c = c0 + b * kWave * 8;
      bf16x8 o;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float2 v = tab[tab_index(bf16_bits(x[b][e]))];
        const float p = v.x * einv;
        float d = g * ((c + e == tc ? 1.f : 0.f) - p);
        float s2 = v.y;
        if constexpr (ENT) {
          d -= h * p * (cap * v.y - lse + ent);
          s2 = 1.f - v.y * v.y;
        }
        o[e] = to_bf16(c + e < vocab ? d * s2 : 0.f);
      }
      if (c < stride) *reinterpret_cast<bf16x8*>(q + c) = o;
    }
  }
}

// ---------------------------------------------------------------------------------------
// The policy loss of a row, and its derivative by logp.
// ---------------------------------------------------------------------------------------
struct PolicyArgs {
  const float* old_logp;
  const float* adv;
  const float* ref_logp;  // null: no KL term
  const float* weights;   // null: 1 / (number of rows with a target)
  float lo, hi, kl_coef;
};

struct PolicyTerm {
  float loss, kl, slope;
  bool clipped;
};

__device__ __forceinline__ PolicyTerm policy_term(const PolicyArgs& a, long r, float logp) {
  const float adv = a.adv[r], ratio = expf(logp - a.old_logp[r]);
  const float free_ = adv == 0.f ? 0.f : ratio * adv;  // an infinite ratio of no advantage counts nothing
  const float held = fminf(fmaxf(ratio, a.lo), a.hi) * adv;
  PolicyTerm t;
  t.clipped = held < free_;
  t.loss = -(t.clipped ? held : free_);
  t.slope = t.clipped ? 0.f : -free_;
  t.kl = 0.f;
  if (a.ref_logp) {
    const float d = a.ref_logp[r] - logp, em = expm1f(d);
    t.kl = em - d;
    if (a.kl_coef != 0.f) {
      t.loss += a.kl_coef * t.kl;
      t.slope -= a.kl_coef * em;
    }
  }
  return t;
}

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) v += __shfl_xor(v, o);
  return v;
}

// Sums over the rows in one workgroup and a fixed order: loss and stats = (KL, share of clipped
// rows), all weighted as the loss is; slope_row (optional): the rows' gradients of the loss by logp.
constexpr int kRowsThreads = 1024;
__global__ __launch_bounds__(kRowsThreads) void policy_rows_kernel(long rows, const int64_t* __restrict__ targets,
                                                                   int64_t ignore_index,
                                                                   const float* __restrict__ logp_row, PolicyArgs a,
                                                                   float* __restrict__ loss, float* __restrict__ stats,
                                                                   float* __restrict__ slope_row) {
  __shared__ double red[3][kRowsThreads / kWave];
  __shared__ double s_count[kRowsThreads / kWave];
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  double w1 = 1.0;
  if (!a.weights) {
    double n = 0.0;  // exact: at most 2^31 rows
    for (long r = threadIdx.x; r < rows; r += kRowsThreads) n += targets[r] != ignore_index ? 1.0 : 0.0;
    n = wave_sum64(n);
    if (lane == 0) s_count[wave] = n;
    __syncthreads();
    n = 0.0;
    for (int v = 0; v < kRowsThreads / kWave; ++v) n += s_count[v];
    w1 = 1.0 / n;  // no row: the sums below are 0 times infinity, NaN as the mean of nothing
  }
  double sl = 0.0, sk = 0.0, sc = 0.0;
  for (long r = threadIdx.x; r < rows; r += kRowsThreads) {
    const float w = a.weights ? a.weights[r] : 1.f;
    const bool on = targets[r] != ignore_index && w != 0.f;
    float slope = 0.f;
    if (on) {
      const PolicyTerm t = policy_term(a, r, logp_row[r]);
      sl += (double)w * t.loss;
      sk += (double)w * t.kl;
      sc += t.clipped ? (double)w : 0.0;
      slope = (float)(w1 * w) * t.slope;
    }
    if (slope_row) slope_row[r] = slope;
  }
  sl = wave_sum64(sl);
  sk = wave_sum64(sk);
  sc = wave_sum64(sc);
  if (lane == 0) {
    red[0][wave] = sl;
    red[1][wave] = sk;
    red[2][wave] = sc;
  }
  __syncthreads();
  if (threadIdx.x < 3) {
    double s = 0.0;
    for (int v = 0; v < kRowsThreads / kWave; ++v) s += red[threadIdx.x][v];
    *(threadIdx.x == 0 ? loss : stats + threadIdx.x - 1) = (float)(s * w1);
  }
}

// ---------------------------------------------------------------------------------------
// The preference loss of P pairs: sequences 0 .. P - 1 are the chosen ones, P + i is the rejected
// partner of i.  Sequence s holds rows T s .. T s + T - 1, or cu[s] .. cu[s + 1] - 1.  One workgroup;
// a wave sums a sequence, in 64 bits and a fixed order.  Sequence bounds that are no
// non-decreasing walk inside the rows make every output NaN (nothing is read outside the rows).
// ---------------------------------------------------------------------------------------
__global__ __launch_bounds__(kRowsThreads) void preference_pairs_kernel(
    long rows, long T, int P, const int32_t* __restrict__ cu, const int64_t* __restrict__ targets,
    int64_t ignore_index, const double* __restrict__ logp_row, const float* __restrict__ ref, float beta,
    float smoothing, int average, float* __restrict__ loss, float* __restrict__ seq_logp, float* __restrict__ margins,
    float* __restrict__ slope_row, double* __restrict__ scratch) {
  __shared__ double red[kRowsThreads / kWave];
  __shared__ int s_bad;
  const int tid = threadIdx.x, wave = tid / kWave, lane = tid % kWave, S = 2 * P;
  double* gain = scratch;          // [S] log-probability less the reference
  double* per = scratch + S;       // [S] 1, or 1 / counted rows
  if (tid == 0) s_bad = 0;
  __syncthreads();
  if (cu) {
    bool bad = false;
    for (int s = tid; s <= S; s += kRowsThreads)
      bad |= cu[s] < 0 || cu[s] > rows || (s > 0 && cu[s] < cu[s - 1]);
    if (bad) s_bad = 1;  // every writer writes the same value
  }
  __syncthreads();
  const bool bad = s_bad != 0;
  const float nan = __builtin_nanf("");
  auto first = [&](int s) { return cu ? (long)cu[s] : T * s; };
  for (int s = wave; s < S; s += kRowsThreads / kWave) {
    double sum = 0.0, n = 0.0;
    if (!bad) {
      const long r1 = first(s + 1);
      for (long r = first(s) + lane; r < r1; r += kWave) {
        sum += logp_row[r];  // 0 without a target
        n += targets[r] != ignore_index ? 1.0 : 0.0;
      }
    }
    sum = wave_sum64(sum);
    n = wave_sum64(n);
    const double w = average ? 1.0 / (n > 0.0 ? n : 1.0) : 1.0;
    if (lane == 0) {
      seq_logp[s] = bad ? nan : (float)(sum * w);
      gain[s] = sum * w - (ref ? (double)ref[s] : 0.0);
      per[s] = w;
    }
  }
  __syncthreads();
  double sl = 0.0;
  for (int i = tid; i < P; i += kRowsThreads) {
    const double m = (double)beta * (gain[i] - gain[P + i]);
    // log sigmoid(m) = min(m, 0) - log(1 + e^-|m|), and the sigmoids from the same e^-|m|
    const double e = exp(-fabs(m)), l = log1p(e);
    const double up = fmin(m, 0.0) - l, down = fmin(-m, 0.0) - l;
    const double sig_up = (m >= 0.0 ? 1.0 : e) / (1.0 + e), sig_down = (m >= 0.0 ? e : 1.0) / (1.0 + e);
    sl -= (1.0 - smoothing) * up + smoothing * down;
    margins[i] = bad ? nan : (float)m;
    const double slope = (double)beta / P * (smoothing * sig_up - (1.0 - smoothing) * sig_down);
    gain[i] = slope;
    gain[P + i] = -slope;
  }
  sl = wave_sum64(sl);
  if (lane == 0) red[wave] = sl;
  __syncthreads();
  if (tid == 0) {
    double s = 0.0;
    for (int v = 0; v < kRowsThreads / kWave; ++v) s += red[v];
    *loss = bad ? nan : (float)(s / P);
  }
  if (!slope_row) return;
  if (bad || cu)  // rows of no sequence
    for (long r = tid; r < rows; r += kRowsThreads)
      if (bad || r < cu[0] || r >= cu[S]) slope_row[r] = bad ? nan : 0.f;
  if (bad) return;
  for (int s = wave; s < S; s += kRowsThreads / kWave) {
    const float v = (float)(gain[s] * per[s]);
    const long r1 = first(s + 1);
    for (long r = first(s) + lane; r < r1; r += kWave) slope_row[r] = v;
  }
}

static unsigned tok_grid(int64_t units, int per_cu) {
  int dev = 0, cus = 256;
  if (hipGetDevice(&dev) == hipSuccess)
    (void)hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev);
  const long g = (long)cus * per_cu;
  const long need = (units + kTokThreads / kWave - 1) / (kTokThreads / kWave);
  return (unsigned)(need < g ? need : g);
}

}  // namespace kda

static int check_tok_args(int64_t rows, int32_t vocab, int64_t stride, float softcap, const void* logits,
                          const void* targets) {
  KDA_REQUIRE(rows >= 0 && rows <= 0x7fffffff, "softcap_log_probs: invalid row count");
  KDA_REQUIRE(vocab > 0 && vocab <= (1 << 24), "softcap_log_probs: vocab must be in [1, 2^24]");
  KDA_REQUIRE(stride >= vocab && stride % 8 == 0 && stride <= (1 << 30),
              "softcap_log_probs: row stride must be >= vocab, a multiple of 8 and <= 2^30");
  KDA_REQUIRE(softcap > 0.f && softcap <= 60.f, "softcap_log_probs: softcap must be in (0, 60]");
  KDA_REQUIRE(rows == 0 || (logits && targets), "softcap_log_probs: null pointer");
  KDA_REQUIRE(kda::aligned16(logits), "softcap_log_probs: logits must be 16-byte aligned");
  return KDA_OK;
}

extern "C" int kda_softcap_log_probs_forward(int64_t rows, int32_t vocab, int64_t stride, float softcap,
                                             const void* logits, const int64_t* targets, int64_t ignore_index,
                                             float* log_probs, double* log_probs64, float* lse_rows,
                                             float* entropy_rows, hipStream_t stream) {
  using namespace kda;
  int rc = check_tok_args(rows, vocab, stride, softcap, logits, targets);
  if (rc != KDA_OK) return rc;
  KDA_REQUIRE(rows == 0 || log_probs || log_probs64, "softcap_log_probs_forward: null output");
  if (rows == 0) return KDA_OK;
  auto go = [&](auto kern, int per_cu) {
    hipLaunchKernelGGL(kern, dim3(tok_grid(rows, per_cu)), dim3(kTokThreads), 0, stream, (long)rows, vocab,
                       (long)stride, softcap, (const bf16*)logits, targets, ignore_index, log_probs, log_probs64,
                       lse_rows, entropy_rows);
  };
  entropy_rows ? go(token_fwd_kernel<true>, kTokPairPerCu) : go(token_fwd_kernel<false>, kTokFwdPerCu);
  KDA_LAUNCH_CHECK("softcap_log_probs_forward");
  return KDA_OK;
}

extern "C" int kda_softcap_log_probs_backward(int64_t rows, int32_t vocab, int64_t stride, float softcap,
                                              const void* logits, const int64_t* targets, int64_t ignore_index,
                                              const float* lse_rows, const float* entropy_rows, const float* g_rows,
                                              const float* h_rows, const float* scale, void* grad_logits,
                                              hipStream_t stream) {
  using namespace kda;
  int rc = check_tok_args(rows, vocab, stride, softcap, logits, targets);
  if (rc != KDA_OK) return rc;
  KDA_REQUIRE(rows == 0 || (lse_rows && grad_logits && (g_rows || h_rows)), "softcap_log_probs_backward: null pointer");
  KDA_REQUIRE(!h_rows || entropy_rows, "softcap_log_probs_backward: an entropy gradient needs the entropies");
  KDA_REQUIRE(aligned16(grad_logits), "softcap_log_probs_backward: grad must be 16-byte aligned");
  if (rows == 0) return KDA_OK;
  const int64_t items = rows * ((stride + kTokChunk - 1) / kTokChunk);
  auto go = [&](auto kern) {
    hipLaunchKernelGGL(kern, dim3(tok_grid(items, kTokPairPerCu)), dim3(kTokThreads), 0, stream, (long)rows, vocab,
                       (long)stride, softcap, (const bf16*)logits, targets, ignore_index, lse_rows, entropy_rows,
                       g_rows, h_rows, scale, (bf16*)grad_logits);
  };
  h_rows ? go(token_bwd_kernel<true>) : go(token_bwd_kernel<false>);
  KDA_LAUNCH_CHECK("softcap_log_probs_backward");
  return KDA_OK;
}

extern "C" int kda_policy_rows(int64_t rows, const int64_t* targets, int64_t ignore_index, const float* log_probs,
                               const float* old_log_probs, const float* advantages, const float* ref_log_probs,
                               const float* weights, float clip_lo, float clip_hi, float kl_coef, float* loss,
                               float* stats, float* slope_rows, hipStream_t stream) {
  using namespace kda;
  KDA_REQUIRE(rows >= 0 && rows <= 0x7fffffff, "policy_rows: invalid row count");
  KDA_REQUIRE(loss && stats && (rows == 0 || (targets && log_probs && old_log_probs && advantages)), "policy_rows: null pointer");
  KDA_REQUIRE(clip_lo <= 1.f && clip_hi >= 1.f, "policy_rows: the clipping range must hold 1");
  const PolicyArgs a{old_log_probs, advantages, ref_log_probs, weights, clip_lo, clip_hi, kl_coef};
  hipLaunchKernelGGL(policy_rows_kernel, dim3(1), dim3(kRowsThreads), 0, stream, (long)rows, targets, ignore_index,
                     log_probs, a, loss, stats, slope_rows);
  KDA_LAUNCH_CHECK("policy_rows");
  return KDA_OK;
}

extern "C" size_t kda_preference_pairs_scratch_bytes(int32_t pairs) {
  return pairs > 0 ? (size_t)pairs * 4 * sizeof(double) : 0;
}

extern "C" int kda_preference_pairs(int64_t rows, int64_t seq_len, int32_t pairs, const int32_t* cu_seqlens,
                                    const int64_t* targets, int64_t ignore_index, const double* log_probs64,
                                    const float* ref_log_probs, float beta, float label_smoothing, int32_t average,
                                    float* loss, float* seq_log_probs, float* margins, float* slope_rows,
                                    void* scratch, hipStream_t stream) {
  using namespace kda;
  KDA_REQUIRE(rows >= 0 && rows <= 0x7fffffff, "preference_pairs: invalid row count");
  KDA_REQUIRE(pairs > 0 && pairs <= (1 << 24), "preference_pairs: pairs must be in [1, 2^24]");
  KDA_REQUIRE(cu_seqlens || (seq_len >= 0 && seq_len * 2 * (int64_t)pairs == rows),
              "preference_pairs: rows must be 2 * pairs * seq_len");
  KDA_REQUIRE(label_smoothing >= 0.f && label_smoothing <= 1.f, "preference_pairs: label_smoothing must be in [0, 1]");
  KDA_REQUIRE(loss && seq_log_probs && margins && scratch && (rows == 0 || (targets && log_probs64)),
              "preference_pairs: null pointer");
  KDA_REQUIRE(aligned16(scratch), "preference_pairs: scratch must be 16-byte aligned");
  hipLaunchKernelGGL(preference_pairs_kernel, dim3(1), dim3(kRowsThreads), 0, stream, (long)rows, (long)seq_len, pairs,
                     cu_seqlens, targets, ignore_index, log_probs64, ref_log_probs, beta, label_smoothing, average,
                     loss, seq_log_probs, margins, slope_rows, (double*)scratch);
  KDA_LAUNCH_CHECK("preference_pairs");
  return KDA_OK;
}
