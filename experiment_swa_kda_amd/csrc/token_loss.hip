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

// tanh(x / cap) and exp(cap tanh(x / cap)), each to about 1.5 ulp, in some 30 instructions from the
// hardware's 2^x and 1 / x (a table has 8448 entries: with library functions its fill took 5 us of
// a CU, more than the row of a short call).  x / cap is rounded once; below 0.3 the odd series up
// to the 11th power (next term 2e-9 of the value), above it 1 - 2 q / (1 + q), q = e^(-2 |a|); the
// exponential's argument is split so that its rounding error is put back to first order.
__device__ __forceinline__ float tok_tanh(float x, float cap, float inv_cap) {
  float a = x * inv_cap;
  a = fmaf(fmaf(-a, cap, x), inv_cap, a);
  const float b = a * a;
  float p = fmaf(b, -1382.f / 155925.f, 62.f / 2835.f);
  p = fmaf(b, p, -17.f / 315.f);
  p = fmaf(b, p, 2.f / 15.f);
  p = fmaf(b, p, -1.f / 3.f);
  p = fmaf(a * b, p, a);
  const float q = __builtin_amdgcn_exp2f(-2.8853900817779268f * fabsf(a));
  const float t = copysignf(1.f - 2.f * q * __builtin_amdgcn_rcpf(1.f + q), a);
  return fabsf(a) < 0.3f ? p : t;
}
__device__ __forceinline__ float tok_exp(float z) {
  const float hi = z * 1.4426950408889634f;
  const float lo = fmaf(z, 1.4426950408889634f, -hi) + z * 1.9259629911e-8f;  // log2 e less its f32 value
  const float e = __builtin_amdgcn_exp2f(hi);
  return fmaf(e, lo * 0.6931471805599453f, e);
}

// One 4096-column chunk of a row per wave; columns from `last` on re-read the vector at `last`.
__device__ __forceinline__ void tok_load(const bf16* __restrict__ row, long c0, long last, bf16x8* x) {
  const long c = c0 + (threadIdx.x % kWave) * 8;
#pragma unroll
  for (int b = 0; b < kTokBatch; ++b) {
    const long cb = c + b * kWave * 8;
    x[b] = *reinterpret_cast<const bf16x8*>(row + (cb < last ? cb : last));
  }
}

// The forward's table: e^z per pattern, with the entropy (e^z, z e^z), and the sums over it.
template <bool ENT>
struct TokSum {
  using Tab = typename std::conditional<ENT, float2, float>::type;
  float se = 0.f, sz = 0.f;
  u16x2 mag = (u16x2)0;  // running maximum of the magnitude bits (NaN detection)

  static __device__ __forceinline__ void fill(Tab* tab, float cap, int threads) {
    const float inv = 1.f / cap;
    for (int i = threadIdx.x; i < kTabSize; i += threads) {
      const float z = cap * tok_tanh(tab_pattern_value(i), cap, inv), e = tok_exp(z);
      if constexpr (ENT)
        tab[i] = make_float2(e, z * e);
      else
        tab[i] = e;
    }
  }
  // adds the eight columns c .. c + 7; FULL: all of them are vocabulary
  template <bool FULL>
  __device__ __forceinline__ void add(const Tab* tabz, bf16x8 x, int c, int vocab) {
    const uint4 w = __builtin_bit_cast(uint4, x);
    const unsigned ws[4] = {w.x, w.y, w.z, w.w};
    float be = 0.f, bz = 0.f;  // a partial per vector: short chains of dependent adds
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      int i0, i1;
      tab_index2_biased(ws[e], i0, i1);
      const bool k0 = FULL || c + 2 * e < vocab, k1 = FULL || c + 2 * e + 1 < vocab;
      const unsigned m = FULL ? 0x7fff7fffu : (k0 ? 0x7fffu : 0u) | (k1 ? 0x7fff0000u : 0u);
      mag = __builtin_elementwise_max(mag, __builtin_bit_cast(u16x2, ws[e] & m));
      const Tab v0 = tabz[i0], v1 = tabz[i1];
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
  __device__ __forceinline__ void wave_total() {
    se = wave_sum(mag.x > 0x7f80 || mag.y > 0x7f80 ? __builtin_nanf("") : se);
    if (ENT) sz = wave_sum(sz);
  }
};

// logp, lse and entropy of a row from its sums se = sum e^z, sz = sum z e^z, and its target's logit.
// Formed in 64 bits from f32 pieces that are small, so that none loses what an f32 lse of 10 would:
// lse = k log 2 + log m with se = m 2^k, m around 1; z_y = cap (1 - d), d = 2 / (1 + e^(2|a|)), for |a| of 4
// and more.  Sequence sums and their differences then keep 1e-7 of a row.
__device__ __forceinline__ double tok_lse(float se) {
  int k;
  float m = frexpf(se, &k);  // [0.5, 1)
  if (m < 0.70710678f) {
    m *= 2.f;
    k -= 1;
  }
  return (double)k * 0.69314718055994530942 + (double)logf(m);
}
// (f32's tanh would leave a z of 5 up to 2^-21 off, most of a row's error; Lambert's continued fraction
// tanh a = a / (1 + a^2 / (3 + a^2 / (5 + ...))), ten levels of it by its recurrence, is within 1e-9 for
// |a| < 4, and beyond that d is small)
__device__ __forceinline__ double tok_z(float raw, float cap) {
  const double a = (double)raw / (double)cap, b = a * a;
  double p0 = 1.0, p1 = 1.0, q0 = 0.0, q1 = 1.0;
#pragma unroll 1
  for (int k = 3; k <= 21; k += 2) {
    const double p = fma(b, p0, k * p1), q = fma(b, q0, k * q1);
    p0 = p1;
    p1 = p;
    q0 = q1;
    q1 = q;
  }
  const float m = fabsf(raw) / cap;
  const double far = (double)cap * (1.0 - (double)(2.f / (1.f + expf(2.f * m))));
  const double z = m < 4.f ? (double)cap * fabs(a) * q1 / p1 : far;
  return raw < 0.f ? -z : raw != raw ? (double)raw : z;
}

struct TokOut {
  float* logp;
  double* logp64;
  float* lse;
  float* ent;
  __device__ __forceinline__ void none(long r) const {
    if (logp) logp[r] = 0.f;
    if (logp64) logp64[r] = 0.0;
    if (lse) lse[r] = 0.f;
    if (ent) ent[r] = 0.f;
  }
  __device__ __forceinline__ void row(long r, float se, float sz, float raw, float cap, bool in_range) const {
    const double l = tok_lse(se), lp = in_range ? tok_z(raw, cap) - l : (double)__builtin_nanf("");
    if (logp) logp[r] = (float)lp;
    if (logp64) logp64[r] = lp;
    if (lse) lse[r] = (float)l;
    if (ent) ent[r] = (float)(l - (double)(sz / se));
  }
};

// Forward of many rows: one wave per row, so that a row's sums are a wave's and no barrier stalls
// the loads; the next chunk's loads, also the next row's, are in flight while one is summed.  Rows
// go last to first: the ones the projection before wrote last are still in the memory-side cache.
// Bound by that read: 8192 x 32768 takes 99 us, 5.4 TB/s, with the entropy 3001 x 50000 90 us, 3.3 (two
// table values an element).
template <bool ENT>
__global__ __launch_bounds__(kTokThreads) void token_fwd_kernel(long rows, int vocab, long stride, float cap,
                                                                const bf16* __restrict__ logits,
                                                                const int64_t* __restrict__ targets,
                                                                int64_t ignore_index, TokOut out) {
  __shared__ typename TokSum<ENT>::Tab tab[kTabSize];
  const int lane = threadIdx.x % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const long last = ((vocab - 1) / 8) * 8;  // last vector start that holds a vocabulary column
  const int nch = (vocab + kTokChunk - 1) / kTokChunk;
  const long step = (long)gridDim.x * (kTokThreads / kWave);
  // the next row with a target from k on (as a distance from the last row); `rows` if there is none
  auto next_row = [&](long k, int64_t& y) {
    for (; k < rows; k += step) {
      y = targets[rows - 1 - k];
      if (y != ignore_index) break;
      if (lane == 0) out.none(rows - 1 - k);
    }
    return k < rows ? k : rows;
  };
  int64_t y = 0, yn = 0;
  long k = next_row((long)blockIdx.x * (kTokThreads / kWave) + wave, y), kn = 0;
  bf16x8 xa[kTokBatch], xb[kTokBatch];
  if (k < rows) tok_load(logits + (rows - 1 - k) * stride, 0, last, xa);
  TokSum<ENT>::fill(tab, cap, kTokThreads);
  __syncthreads();
  const auto* tabz = tab - (kTabELo << 7);
  TokSum<ENT> sum;
  int ch = 0;
  // sums the chunk in x, with the item after it on its way into xn; false after the last
  auto item = [&](const bf16x8* x, bf16x8* xn) {
    const bool ends = ch == nch - 1;
    if (ends) kn = next_row(k + step, yn);
    if (!ends || kn < rows)
      tok_load(logits + (rows - 1 - (ends ? kn : k)) * stride, ends ? 0 : (long)(ch + 1) * kTokChunk, last, xn);
    const int c0 = ch * kTokChunk + lane * 8;
    if ((ch + 1) * kTokChunk <= vocab) {  // uniform
#pragma unroll
      for (int b = 0; b < kTokBatch; ++b) sum.template add<true>(tabz, x[b], 0, 0);
    } else {
#pragma unroll
      for (int b = 0; b < kTokBatch; ++b) sum.template add<false>(tabz, x[b], c0 + b * kWave * 8, vocab);
    }
    if (!ends) {
      ++ch;
      return true;
    }
    sum.wave_total();
    if (lane == 0) {
      const long r = rows - 1 - k;
      const bool in_range = y >= 0 && y < vocab;
      out.row(r, sum.se, sum.sz, in_range ? (float)logits[r * stride + y] : 0.f, cap, in_range);
    }
    sum = TokSum<ENT>();
    ch = 0;
    k = kn;
    y = yn;
    return k < rows;
  };
  if (k >= rows) return;
  while (item(xa, xb) && item(xb, xa)) {
  }
}

// Forward of few rows: a workgroup per row, the row's first loads in flight while the table fills.
constexpr int kTokWide = 1024;
constexpr int kTokWideBatch = 4;
constexpr int kTokWideRows = 256, kTokWideVocab = 8192;
template <bool ENT>
__global__ __launch_bounds__(kTokWide) void token_fwd_wide_kernel(long rows, int vocab, long stride, float cap,
                                                                  const bf16* __restrict__ logits,
                                                                  const int64_t* __restrict__ targets,
                                                                  int64_t ignore_index, TokOut out) {
  __shared__ typename TokSum<ENT>::Tab tab[kTabSize];
  __shared__ float s_e[kTokWide / kWave], s_z[kTokWide / kWave];
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const int last = ((vocab - 1) / 8) * 8;
  constexpr int CHUNK = kTokWide * 8 * kTokWideBatch;
  bool filled = false;
  for (long r = blockIdx.x; r < rows; r += gridDim.x) {
    const int64_t y = targets[r];
    if (y == ignore_index) {
      if (tid == 0) out.none(r);
      continue;
    }
    const bf16* row = logits + r * stride;
    const bool in_range = y >= 0 && y < vocab;
    const float raw = in_range ? (float)row[y] : 0.f;
    TokSum<ENT> sum;
    for (int c0 = 0; c0 < vocab; c0 += CHUNK) {
      bf16x8 x[kTokWideBatch];
#pragma unroll
      for (int b = 0; b < kTokWideBatch; ++b) {
        const int c = c0 + (b * kTokWide + tid) * 8;
        x[b] = *reinterpret_cast<const bf16x8*>(row + (c < last ? c : last));
      }
      if (!filled) {
        TokSum<ENT>::fill(tab, cap, kTokWide);
        __syncthreads();
        filled = true;
      }
      const auto* tabz = tab - (kTabELo << 7);
#pragma unroll
      for (int b = 0; b < kTokWideBatch; ++b)
        sum.template add<false>(tabz, x[b], c0 + (b * kTokWide + tid) * 8, vocab);
    }
    sum.wave_total();
    __syncthreads();  // the last row's partials are read
    if (lane == 0) {
      s_e[wave] = sum.se;
      s_z[wave] = sum.sz;
    }
    __syncthreads();
    if (tid == 0) {
      float se = 0.f, sz = 0.f;
      for (int w = 0; w < kTokWide / kWave; ++w) {
        se += s_e[w];
        sz += s_z[w];
      }
      out.row(r, se, sz, raw, cap, in_range);
    }
  }
}

// Backward for given row gradients: g of logp (times *scale if given) and, with ENT, h of the
// entropy.  Nothing is reduced, so (row, chunk) items go to the waves in order.
// Bound by one read and one write: 8192 x 32768 takes 179 us behind the forward (last-level cache) and 204
// alone, 5.3 TB/s; with the entropy 3001 x 50000 107 us, 5.6.
template <bool ENT>
__global__ __launch_bounds__(kTokThreads) void token_bwd_kernel(
    long rows, int vocab, long stride, float cap, const bf16* __restrict__ logits, const int64_t* __restrict__ targets,
    int64_t ignore_index, const float* __restrict__ lse_row, const float* __restrict__ ent_row,
    const float* __restrict__ g_row, const float* __restrict__ h_row, const float* __restrict__ scale,
    bf16* __restrict__ grad) {
  __shared__ float2 tab[kTabSize];  // (e^z, 1 - tanh^2), with the entropy (e^z, tanh)
  const int lane = threadIdx.x % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int nch = (int)((stride + kTokChunk - 1) / kTokChunk);
  const long items = rows * nch, step = (long)gridDim.x * (kTokThreads / kWave);
  const float up = scale ? *scale : 1.f;
  struct Item {
    long r;
    int c0;  // first column of the chunk
    int64_t y;
    float g, h, lse, ent;
  };
  // an item and, unless its row's gradient is zero, its loads
  auto fetch = [&](long j, Item& it, bf16x8* x) {
    it.r = j / nch;
    it.c0 = (int)(j - it.r * nch) * kTokChunk;
    it.y = targets[it.r];
    const bool on = it.y != ignore_index;
    it.g = on && g_row ? g_row[it.r] * up : 0.f;
    it.h = ENT && on && h_row ? h_row[it.r] * up : 0.f;
    if (it.g == 0.f && it.h == 0.f) return;
    tok_load(logits + it.r * stride, it.c0, stride - 8, x);
    it.lse = lse_row[it.r];
    it.ent = ENT ? ent_row[it.r] : 0.f;
  };
  auto finish = [&](const Item& it, const bf16x8* x) {
    bf16* q = grad + it.r * stride;
    const int c1 = it.c0 + lane * 8;
    if (it.g == 0.f && it.h == 0.f) {
#pragma unroll
      for (int b = 0; b < kTokBatch; ++b) {
        const int c = c1 + b * kWave * 8;
        if (c < stride) *reinterpret_cast<uint4*>(q + c) = make_uint4(0, 0, 0, 0);
      }
      return;
    }
    const int tc = it.y >= 0 && it.y < vocab ? (int)it.y : -1;
    // (a target outside the vocabulary has no log-probability, though the row has an entropy)
    const float g = tc < 0 && it.g != 0.f ? __builtin_nanf("") : it.g;
    const float einv = tok_exp(-it.lse), ge = -g * einv, he = it.h * einv, off = it.ent - it.lse;
    const float2* tabz = tab - (kTabELo << 7);
    auto value = [&](float2 v) {  // the gradient of a column that is not the target
      if constexpr (ENT) return v.x * (ge - he * fmaf(cap, v.y, off)) * fmaf(-v.y, v.y, 1.f);
      return v.x * ge * v.y;
    };
    const bool full = it.c0 + kTokChunk <= vocab;  // uniform
#pragma unroll
    for (int b = 0; b < kTokBatch; ++b) {
      const int c = c1 + b * kWave * 8;
      const uint4 w = __builtin_bit_cast(uint4, x[b]);
      const unsigned ws[4] = {w.x, w.y, w.z, w.w};
      bf16x8 o;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        int i0, i1;
        tab_index2_biased(ws[e], i0, i1);
        o[2 * e] = to_bf16(value(tabz[i0]));
        o[2 * e + 1] = to_bf16(value(tabz[i1]));
      }
      if (!full) {
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = c + e < vocab ? o[e] : to_bf16(0.f);
      }
      if (c < stride) *reinterpret_cast<bf16x8*>(q + c) = o;
    }
    // the target's column again, with its own term: the lane that has just written it
    const int ct = tc - it.c0;
    if (tc >= 0 && ct >= 0 && ct < kTokChunk && (ct / 8) % kWave == lane) {
      const float2 v = tab[tab_index(bf16_bits(logits[it.r * stride + tc]))];
      const float s2 = ENT ? fmaf(-v.y, v.y, 1.f) : v.y;
      q[tc] = to_bf16(fmaf(g, s2, value(v)));
    }
  };
  Item ia, ib;
  bf16x8 xa[kTokBatch], xb[kTokBatch];
  long j = (long)blockIdx.x * (kTokThreads / kWave) + wave;
  if (j < items) fetch(j, ia, xa);
  {
    const float inv = 1.f / cap;
    for (int i = threadIdx.x; i < kTabSize; i += kTokThreads) {
      const float th = tok_tanh(tab_pattern_value(i), cap, inv);
      tab[i] = make_float2(tok_exp(cap * th), ENT ? th : fmaf(-th, th, 1.f));
    }
  }
  __syncthreads();
  for (; j < items; j += 2 * step) {
    if (j + step < items) fetch(j + step, ib, xb);
    finish(ia, xa);
    if (j + step >= items) break;
    if (j + 2 * step < items) fetch(j + 2 * step, ia, xa);
    finish(ib, xb);
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

// (the log-probability in 64 bits: rounded first, a value of 10 would leave its difference 2^-21 off)
__device__ __forceinline__ PolicyTerm policy_term(const PolicyArgs& a, double logp, float old, float adv, float ref) {
  const float ratio = expf((float)(logp - old));
  const float free_ = adv == 0.f ? 0.f : ratio * adv;  // an infinite ratio of no advantage counts nothing
  const float held = fminf(fmaxf(ratio, a.lo), a.hi) * adv;
  PolicyTerm t;
  t.clipped = held < free_;
  t.loss = -(t.clipped ? held : free_);
  t.slope = t.clipped ? 0.f : -free_;
  t.kl = 0.f;
  if (a.ref_logp) {
    const float d = (float)(ref - logp), em = expm1f(d);
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

// Loss and logit gradient in one read of the logits, for rows of at most NV passes of a workgroup:
// a row (NV vectors a thread, the next row's already in flight) is summed from the table (waves,
// then their partials through LDS in a fixed order); the row's slope, which depends on nothing
// outside the row but the number of rows with a target (counted by every workgroup at the start),
// then gives the gradient for the upstream gradient `expected` from the indices kept in registers.
// All that is one value per row is done for 64 rows at once by the first
// wave's lanes: targets, weights and z of the targets before them (two log-ratio offsets wait in
// LDS), log-probabilities and loss terms after them; in between every thread only adds the
// partials and forms the slope from two hardware exponentials.  part[workgroup] = f64 sums of its
// rows' (loss, KL, clipped weight), for policy_sum_kernel.
// Bound by one read and one write: 8192 x 32768 takes 198 us, 5.4 TB/s (the two passes 303; with workgroups
// of 512 threads and eight vectors each 266), 500 x 8003 15 us.
constexpr int kFusedMaxVec = 4;
constexpr int kFusedMost = 1024;                       // threads of the widest workgroup
constexpr int kFusedMaxCols = kFusedMost * 8 * kFusedMaxVec;
constexpr int kFusedBatch = kWave;  // rows whose scalars are formed together
typedef int i32x4 __attribute__((ext_vector_type(4)));
constexpr unsigned kNullIndex2 = 0x00010001u * (kTabSize + (kTabELo << 7));  // two (biased) padding entries
constexpr int kRowOff = -2, kRowBad = -1;  // a row that does not count; a target outside the vocabulary

template <int NV, int THREADS>
__global__ __launch_bounds__(THREADS, 4) void policy_fused_kernel(
    long rows, int vocab, int stride, float cap, const bf16* __restrict__ logits, const int64_t* __restrict__ targets,
    int64_t ignore_index, PolicyArgs pa, float expected, float* __restrict__ logp_row, double* __restrict__ part,
    bf16* __restrict__ grad) {
  constexpr int WAVES = THREADS / kWave;
  __shared__ float2 tab[kTabSize + 1];  // and the entry of a padding column, (0, 0)
  __shared__ f32x4 s_part[2][WAVES / 4];
  __shared__ int s_count[WAVES];
  __shared__ int s_col[kFusedBatch];     // the target's column, kRowOff or kRowBad
  __shared__ float4 s_row[kFusedBatch];  // z - old, ref - z, advantage, weight
  __shared__ float s_sum[kFusedBatch];   // sum of e^z
  __shared__ double s_z[kFusedBatch];    // z of the target
  __shared__ double s_acc[3][kFusedBatch];  // the lanes' loss sums (registers are for the row)
  const int tid = threadIdx.x, lane = tid % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const long G = gridDim.x;
  const long mine = (rows - 1 - blockIdx.x) / G + 1;  // rows blockIdx.x, + G, ...: at least one
  // a row as a buffer of its own: vectors past its end read as zero, stores to them are dropped
  auto buffer = [&](const bf16* base, long r) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<bf16*>(base) + r * stride, (short)0, 2 * stride, 0x00020000);
  };
  auto load = [&](long r, int col, bf16x8* x) {
    if (col == kRowOff) return;
    const auto rs = buffer(logits, r);
#pragma unroll
    for (int v = 0; v < NV; ++v)
      x[v] = __builtin_bit_cast(bf16x8, __builtin_amdgcn_raw_buffer_load_b128(rs, (v * THREADS + tid) * 16, 0, 0));
  };
  // the first wave: scalars of rows k0 .. of the workgroup, one a lane
  auto scalars = [&](long k0) {
    const long r = blockIdx.x + (k0 + lane) * G;
    if (k0 + lane >= mine) return;
    const int64_t y = targets[r];
    const float w = pa.weights ? pa.weights[r] : 1.f;
    int col = kRowOff;
    if (y != ignore_index && w != 0.f) {
      col = y >= 0 && y < vocab ? (int)y : kRowBad;
      const float old = pa.old_logp[r], adv = pa.adv[r], ref = pa.ref_logp ? pa.ref_logp[r] : 0.f;
      const double zt = col >= 0 ? tok_z((float)logits[r * stride + col], cap) : (double)__builtin_nanf("");
      s_row[lane] = make_float4((float)(zt - old), (float)(ref - zt), adv, w);
      s_z[lane] = zt;
    }
    s_col[lane] = col;
  };
  // Before the first row: its loads, the count of targets, and the table from all waves but the
  // first, which forms its rows' scalars (three dependent loads) in the meantime.
  bf16x8 xa[NV], xb[NV];
  {
    const bool on = targets[blockIdx.x] != ignore_index && (!pa.weights || pa.weights[blockIdx.x] != 0.f);
    load(blockIdx.x, on ? 0 : kRowOff, xa);
  }
  int count = 0;
  if (!pa.weights) {
    for (long i0 = 0; i0 < rows; i0 += 8 * THREADS) {
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const long i = i0 + q * THREADS + tid;
        count += targets[i < rows ? i : rows - 1] != ignore_index && i < rows ? 1 : 0;
      }
    }
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) count += __shfl_xor(count, o);
    if (lane == 0) s_count[wave] = count;
  }
  if (wave == 0) {
    scalars(0);
#pragma unroll
    for (int k = 0; k < 3; ++k) s_acc[k][lane] = 0.0;
    if (lane == 0) tab[kTabSize] = make_float2(0.f, 0.f);
  } else {
    const float inv = 1.f / cap;
    for (int i = tid - kWave; i < kTabSize; i += THREADS - kWave) {
      const float th = tok_tanh(tab_pattern_value(i), cap, inv);
      tab[i] = make_float2(tok_exp(cap * th), fmaf(-th, th, 1.f));
    }
  }
  wait_lgkm0();
  ring_barrier();
  const float2* tabz = tab - (kTabELo << 7);
  double w1 = 1.0;
  if (!pa.weights) {
    count = 0;
    for (int w = 0; w < WAVES; ++w) count += s_count[w];
    w1 = 1.0 / (double)count;
  }
  const float w1f = (float)w1 * expected;
  int slot = 0;  // alternates over the rows that pass the barrier, so that one barrier a row suffices
  auto process = [&](long r, int i, int col, const bf16x8* x) {
    const auto rs = buffer(grad, r);
    if (col == kRowOff) {
#pragma unroll
      for (int v = 0; v < NV; ++v)
        __builtin_amdgcn_raw_buffer_store_b128(i32x4{0, 0, 0, 0}, rs, (v * THREADS + tid) * 16, 0, 0);
      return;
    }
    float sum = 0.f;
    unsigned idx[NV][4];  // table indices, two in a word
    u16x2 mag = (u16x2)0;
    int cols = vocab;  // (opaque: hoisted out of the rows, the column tests would fill the scalar registers)
    asm volatile("" : "+s"(cols));
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * THREADS + tid) * 8;
      const uint4 w = __builtin_bit_cast(uint4, x[v]);
      unsigned m[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) idx[v][e] = tab_index2_packed(m[e]);
      if ((v * THREADS + (wave + 1) * kWave) * 8 > cols) {  // uniform: some of the wave's columns are padding
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const unsigned keep = (cols - c > 2 * e ? 0xffffu : 0u) | (cols - c > 2 * e + 1 ? 0xffff0000u : 0u);
          m[e] &= keep;
          idx[v][e] = (idx[v][e] & keep) | (kNullIndex2 & ~keep);
        }
      }
      float sb = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        mag = __builtin_elementwise_max(mag, __builtin_bit_cast(u16x2, m[e] & 0x7fff7fffu));
        sb += tabz[idx[v][e] & 0xffffu].x + tabz[idx[v][e] >> 16].x;
      }
      sum += sb;
    }
    sum = wave_sum(mag.x > 0x7f80 || mag.y > 0x7f80 ? __builtin_nanf("") : sum);
    if (lane == 0) reinterpret_cast<float*>(s_part[slot])[wave] = sum;
    wait_lgkm0();
    ring_barrier();  // LDS alone: the next row's loads stay in flight
    f32x4 se4 = s_part[slot][0];
#pragma unroll
    for (int w = 1; w < WAVES / 4; ++w) se4 += s_part[slot][w];
    slot ^= 1;
    const float se = (se4[0] + se4[1]) + (se4[2] + se4[3]);
    if (tid == 0) s_sum[i] = se;
    const float4 row = s_row[i];
    const float l2 = __builtin_amdgcn_logf(se);  // log2
    const float ratio = __builtin_amdgcn_exp2f(fmaf(row.x, 1.4426950408889634f, -l2));
    const float free_ = row.z == 0.f ? 0.f : ratio * row.z;
    float g = fminf(fmaxf(ratio, pa.lo), pa.hi) * row.z < free_ ? 0.f : -free_;
    if (pa.ref_logp && pa.kl_coef != 0.f)
      g -= pa.kl_coef * (__builtin_amdgcn_exp2f(fmaf(row.y, 1.4426950408889634f, l2)) - 1.f);
    g *= row.w * w1f;
    // (p = e^z / sum; an out-of-range target has no log-probability, so no finite slope)
    g = col == kRowBad ? __builtin_nanf("") : g;
    const float ge = -g * (1.f / se);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * THREADS + tid) * 8;
      bf16x8 o;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        asm volatile("" : "+v"(idx[v][e]));  // (looked up again: kept from the sum, the values would spill)
        const float2 v0 = tabz[idx[v][e] & 0xffffu], v1 = tabz[idx[v][e] >> 16];
        o[2 * e] = to_bf16(v0.x * ge * v0.y);
        o[2 * e + 1] = to_bf16(v1.x * ge * v1.y);
      }
      if ((v * THREADS + (wave + 1) * kWave) * 8 > cols) {  // padding is zero beside a NaN slope too
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = cols - c > e ? o[e] : to_bf16(0.f);
      }
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(i32x4, o), rs, c * 2, 0, 0);
    }
    // the target's column again, with its own term: the thread that has just written it
    if (col >= 0 && (col / 8) % THREADS == tid) {
      const float2 v = tab[tab_index(bf16_bits(logits[r * stride + col]))];
      grad[r * stride + col] = to_bf16(fmaf(g, v.y, v.x * ge * v.y));
    }
  };
  for (long k0 = 0; k0 < mine; k0 += kFusedBatch) {
    const int n = (int)(mine - k0 < kFusedBatch ? mine - k0 : kFusedBatch);
    if (k0 > 0) {
      if (wave == 0) scalars(k0);
      wait_lgkm0();
      ring_barrier();
    }
    auto at = [&](int i) { return blockIdx.x + (k0 + i) * G; };
    auto col = [&](int i) { return __builtin_amdgcn_readfirstlane(s_col[i]); };
    int ca = col(0), cb = kRowOff;
    if (k0 > 0) load(at(0), ca, xa);
    for (int i = 0; i < n; i += 2) {
      if (i + 1 < n) load(at(i + 1), cb = col(i + 1), xb);
      process(at(i), i, ca, xa);
      if (i + 1 >= n) break;
      if (i + 2 < n) load(at(i + 2), ca = col(i + 2), xa);
      process(at(i + 1), i + 1, cb, xb);
    }
    wait_lgkm0();
    ring_barrier();  // the rows' sums are in LDS, and their scalars are read
    if (wave == 0 && lane < n) {
      const long rl = at(lane);
      float logp = 0.f;
      if (s_col[lane] != kRowOff) {
        const double lp = s_z[lane] - tok_lse(s_sum[lane]);
        logp = (float)lp;
        const double w = pa.weights ? pa.weights[rl] : 1.f;
        const PolicyTerm t = policy_term(pa, lp, pa.old_logp[rl], pa.adv[rl], pa.ref_logp ? pa.ref_logp[rl] : 0.f);
        s_acc[0][lane] += w * t.loss;
        s_acc[1][lane] += w * t.kl;
        s_acc[2][lane] += t.clipped ? w : 0.0;
      }
      logp_row[rl] = logp;
    }
  }
  if (wave == 0)
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      const double v = wave_sum64(s_acc[k][lane]);
      if (lane == 0) part[3 * blockIdx.x + k] = v * w1;
    }
}

// the workgroups' sums, in order
__global__ __launch_bounds__(kWave) void policy_sum_kernel(int parts, const double* __restrict__ part,
                                                           float* __restrict__ loss, float* __restrict__ stats) {
  double s[3] = {0.0, 0.0, 0.0};
  for (int i = threadIdx.x; i < parts; i += kWave)
#pragma unroll
    for (int k = 0; k < 3; ++k) s[k] += part[3 * i + k];
#pragma unroll
  for (int k = 0; k < 3; ++k) s[k] = wave_sum64(s[k]);
  if (threadIdx.x == 0) {
    *loss = (float)s[0];
    stats[0] = (float)s[1];
    stats[1] = (float)s[2];
  }
}

// Sums over the rows in one workgroup and a fixed order: loss and stats = (KL, share of clipped
// rows), all weighted as the loss is; slope_row (optional): the rows' gradients of the loss by logp.
constexpr int kRowsThreads = 1024;
constexpr int kRowsAhead = 4;  // rows of a thread whose loads are in flight together
__global__ __launch_bounds__(kRowsThreads) void policy_rows_kernel(long rows, const int64_t* __restrict__ targets,
                                                                   int64_t ignore_index,
                                                                   const double* __restrict__ logp_row, PolicyArgs a,
                                                                   float* __restrict__ loss, float* __restrict__ stats,
                                                                   float* __restrict__ slope_row) {
  __shared__ double red[3][kRowsThreads / kWave];
  __shared__ double s_count[kRowsThreads / kWave];
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  double w1 = 1.0;
  if (!a.weights) {
    int n = 0;
    for (long r0 = threadIdx.x; r0 < rows; r0 += kRowsAhead * kRowsThreads) {
#pragma unroll
      for (int q = 0; q < kRowsAhead; ++q) {
        const long r = r0 + q * kRowsThreads;
        n += targets[r < rows ? r : rows - 1] != ignore_index && r < rows ? 1 : 0;
      }
    }
    const double total = wave_sum64((double)n);  // exact: at most 2^31 rows
    if (lane == 0) s_count[wave] = total;
    __syncthreads();
    double all = 0.0;
    for (int v = 0; v < kRowsThreads / kWave; ++v) all += s_count[v];
    w1 = 1.0 / all;  // no row: the sums below are 0 times infinity, NaN as the mean of nothing
  }
  double sl = 0.0, sk = 0.0, sc = 0.0;
  for (long r0 = threadIdx.x; r0 < rows; r0 += kRowsAhead * kRowsThreads) {
    float w[kRowsAhead], old[kRowsAhead], adv[kRowsAhead], ref[kRowsAhead];
    double lp[kRowsAhead];
    bool on[kRowsAhead];
#pragma unroll
    for (int q = 0; q < kRowsAhead; ++q) {  // all loads before any is used
      const long r = r0 + q * kRowsThreads, i = r < rows ? r : rows - 1;
      w[q] = a.weights ? a.weights[i] : 1.f;
      on[q] = targets[i] != ignore_index && r < rows;
      lp[q] = logp_row[i];
      old[q] = a.old_logp[i];
      adv[q] = a.adv[i];
      ref[q] = a.ref_logp ? a.ref_logp[i] : 0.f;
    }
#pragma unroll
    for (int q = 0; q < kRowsAhead; ++q) {
      const long r = r0 + q * kRowsThreads;
      float slope = 0.f;
      if (on[q] && w[q] != 0.f) {
        const PolicyTerm t = policy_term(a, lp[q], old[q], adv[q], ref[q]);
        sl += (double)w[q] * t.loss;
        sk += (double)w[q] * t.kl;
        sc += t.clipped ? (double)w[q] : 0.0;
        slope = (float)(w1 * w[q]) * t.slope;
      }
      if (slope_row && r < rows) slope_row[r] = slope;
    }
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
// Bound by the latency of its few dependent steps: 5.4 us for 4 pairs of 764 rows in all, 6.7 for 8192.
// ---------------------------------------------------------------------------------------
constexpr int kPairAhead = 8;
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
      for (long r0 = first(s) + lane; r0 < r1; r0 += kPairAhead * kWave) {
        double v[kPairAhead];
        int64_t y[kPairAhead];
#pragma unroll
        for (int q = 0; q < kPairAhead; ++q) {
          const long r = r0 + q * kWave, i = r < r1 ? r : r0;
          v[q] = logp_row[i];  // 0 without a target
          y[q] = average ? targets[i] : 0;
        }
#pragma unroll
        for (int q = 0; q < kPairAhead; ++q) {
          const bool in = r0 + q * kWave < r1;
          sum += in ? v[q] : 0.0;
          n += in && y[q] != ignore_index ? 1.0 : 0.0;
        }
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
  const TokOut out{log_probs, log_probs64, lse_rows, entropy_rows};
  auto go = [&](auto kern, unsigned grid, int threads) {
    hipLaunchKernelGGL(kern, dim3(grid), dim3(threads), 0, stream, (long)rows, vocab, (long)stride, softcap,
                       (const bf16*)logits, targets, ignore_index, out);
  };
  // a workgroup per row where there are no more rows than CUs and a wave would walk a row for long:
  // 200 x 32768 takes 8.1 us (a wave per row 19), but 500 x 8003 11.7 (9.2), 300 x 1000 11.3 (7.5)
  if (rows <= kTokWideRows && vocab > kTokWideVocab)
    entropy_rows ? go(token_fwd_wide_kernel<true>, rows, kTokWide) : go(token_fwd_wide_kernel<false>, rows, kTokWide);
  else
    entropy_rows ? go(token_fwd_kernel<true>, tok_grid(rows, kTokPairPerCu), kTokThreads)
                 : go(token_fwd_kernel<false>, tok_grid(rows, kTokFwdPerCu), kTokThreads);
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

extern "C" int kda_policy_rows(int64_t rows, const int64_t* targets, int64_t ignore_index, const double* log_probs64,
                               const float* old_log_probs, const float* advantages, const float* ref_log_probs,
                               const float* weights, float clip_lo, float clip_hi, float kl_coef, float* loss,
                               float* stats, float* slope_rows, hipStream_t stream) {
  using namespace kda;
  KDA_REQUIRE(rows >= 0 && rows <= 0x7fffffff, "policy_rows: invalid row count");
  KDA_REQUIRE(loss && stats && (rows == 0 || (targets && log_probs64 && old_log_probs && advantages)), "policy_rows: null pointer");
  KDA_REQUIRE(clip_lo <= 1.f && clip_hi >= 1.f, "policy_rows: the clipping range must hold 1");
  const PolicyArgs a{old_log_probs, advantages, ref_log_probs, weights, clip_lo, clip_hi, kl_coef};
  hipLaunchKernelGGL(policy_rows_kernel, dim3(1), dim3(kRowsThreads), 0, stream, (long)rows, targets, ignore_index,
                     log_probs64, a, loss, stats, slope_rows);
  KDA_LAUNCH_CHECK("policy_rows");
  return KDA_OK;
}

extern "C" int kda_policy_fused_supported(int64_t stride) { return stride > 0 && stride <= kda::kFusedMaxCols; }

// Waves enough for every SIMD's four: one workgroup of sixteen per CU for long rows, two of eight
// otherwise, so that the barrier of a row hides behind the other one's loads (8192 x 8192: 85 us
// with one of sixteen).
static int fused_per_cu(int64_t stride) { return stride > kda::kFusedMaxCols / 2 ? 1 : 2; }

static unsigned fused_grid(int64_t rows, int64_t stride) {
  int dev = 0, cus = 256;
  if (hipGetDevice(&dev) == hipSuccess) (void)hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev);
  cus *= fused_per_cu(stride);
  return (unsigned)(rows < cus ? rows : cus);
}

extern "C" size_t kda_policy_fused_scratch_bytes(int64_t rows, int64_t stride) {
  return rows > 0 && kda_policy_fused_supported(stride) ? (size_t)fused_grid(rows, stride) * 3 * sizeof(double) : 0;
}

extern "C" int kda_policy_fused(int64_t rows, int32_t vocab, int64_t stride, float softcap, const void* logits,
                                const int64_t* targets, int64_t ignore_index, const float* old_log_probs,
                                const float* advantages, const float* ref_log_probs, const float* weights,
                                float clip_lo, float clip_hi, float kl_coef, float expected_grad, float* loss,
                                float* stats, float* log_probs, void* grad_logits, void* scratch, hipStream_t stream) {
  using namespace kda;
  int rc = check_tok_args(rows, vocab, stride, softcap, logits, targets);
  if (rc != KDA_OK) return rc;
  KDA_REQUIRE(kda_policy_fused_supported(stride), "policy_fused: rows of at most %d columns", kFusedMaxCols);
  KDA_REQUIRE(rows > 0, "policy_fused: no rows");
  KDA_REQUIRE(old_log_probs && advantages && loss && stats && log_probs && grad_logits && scratch,
              "policy_fused: null pointer");
  KDA_REQUIRE(aligned16(grad_logits, scratch), "policy_fused: grad and scratch must be 16-byte aligned");
  KDA_REQUIRE(clip_lo <= 1.f && clip_hi >= 1.f, "policy_fused: the clipping range must hold 1");
  const PolicyArgs a{old_log_probs, advantages, ref_log_probs, weights, clip_lo, clip_hi, kl_coef};
  const unsigned grid = fused_grid(rows, stride);
  const int threads = kFusedMost / fused_per_cu(stride);
  auto go = [&](auto kern) {
    hipLaunchKernelGGL(kern, dim3(grid), dim3(threads), 0, stream, (long)rows, vocab, (int)stride, softcap,
                       (const bf16*)logits, targets, ignore_index, a, expected_grad, log_probs, (double*)scratch,
                       (bf16*)grad_logits);
  };
  const int nv = (int)((stride + threads * 8 - 1) / (threads * 8));
  if (threads == kFusedMost) {  // 16384 columns at least
    nv == 3 ? go(policy_fused_kernel<3, kFusedMost>) : go(policy_fused_kernel<4, kFusedMost>);
  } else {
    switch (nv) {
      case 1: go(policy_fused_kernel<1, kFusedMost / 2>); break;
      case 2: go(policy_fused_kernel<2, kFusedMost / 2>); break;
      case 3: go(policy_fused_kernel<3, kFusedMost / 2>); break;
      default: go(policy_fused_kernel<4, kFusedMost / 2>); break;
    }
  }
  KDA_LAUNCH_CHECK("policy_fused");
  hipLaunchKernelGGL(policy_sum_kernel, dim3(1), dim3(kWave), 0, stream, (int)grid, (const double*)scratch, loss, stats);
  KDA_LAUNCH_CHECK("policy_sum");
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
