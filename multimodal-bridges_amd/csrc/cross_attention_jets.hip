// Cross attention of small clouds in floats, heads up to 32 wide: 16 x 16 tiles.
//
// The resident scheme of cross_attention_resident.hip (one key head of one cloud a workgroup, rows in LDS, one barrier) on
// v_mfma_f32_16x16x4: a jet's heads are 16 or 32 features wide and some 50 slots long, and 32 x 32 tiles of them are half
// padding -- a 16-wide head fills half the feature rows of its second product, 75 slots fill 96.  The rate of the two
// instructions is the same, the wave's registers shrink to a third (acc 4, not 16, a feature tile), and six or more waves a
// SIMD hide the chain mask -> slots -> rows that each workgroup's time consists of.
// Lane (c = lane & 15, g = lane >> 4) holds column c and rows 4g .. 4g+3 of a tile, which again is the B operand of the next
// product: step i contracts over rows {i, 4 + i, 8 + i, 12 + i}.
#include "cross_attention.h"

namespace mmb {
namespace xattn {

struct JetArgs {
  Shape sh;
  const float *q, *k, *v, *out, *dout;
  int64_t q_ld, k_ld, v_ld, out_ld, dout_ld, dq_ld, dk_ld, dv_ld;
  const float *mq, *mk;
  float* lse;
  float scale;
  float *o, *dq, *dk, *dv;
  int parts, nkp, nqp;                            // (as in the resident kernels; slots padded to 32)
  GridMap map;
};

__device__ __forceinline__ f32x4 zero4() { return f32x4{0.0f, 0.0f, 0.0f, 0.0f}; }
template <int FT> constexpr int jet_pitch() { return 16 * FT + 4; }

// a row as an operand: features 16t + 4g .. + 3
template <int FT, bool VEC>
__device__ __forceinline__ void jet_row(f32x4* r, const float* __restrict__ p, int D, bool ok) {
  const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int t = 0; t < FT; ++t) r[t] = __builtin_bit_cast(f32x4, load_chunk<float, VEC>(p, 16 * t + 4 * g, D, ok));
}
// 16 rows from LDS . b
template <int FT>
__device__ __forceinline__ f32x4 jet_dot(const float* rows, const f32x4* b) {
  const int lane = threadIdx.x & 63;
  const float* p = rows + (lane & 15) * jet_pitch<FT>() + (lane >> 4) * 4;
  f32x4 s = zero4();
#pragma unroll
  for (int t = 0; t < FT; ++t) {
    const f32x4 a = *reinterpret_cast<const f32x4*>(p + 16 * t);
#pragma unroll
    for (int i = 0; i < 4; ++i) s = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[t][i], s, 0, 0, 0);
  }
  return s;
}
// acc[t] (features x columns) += rows^T . w
template <int FT>
__device__ __forceinline__ void jet_cols(const float* rows, f32x4 w, f32x4* acc) {
  const int lane = threadIdx.x & 63;
  const float* p = rows + (lane >> 4) * 4 * jet_pitch<FT>() + (lane & 15);
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int t = 0; t < FT; ++t) acc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(p[i * jet_pitch<FT>() + 16 * t], w[i], acc[t], 0, 0, 0);
}
template <int FT, bool VEC>
__device__ __forceinline__ void jet_store(float* __restrict__ p, const f32x4* acc, float mul, int D) {
  const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int t = 0; t < FT; ++t) {
    const int d = 16 * t + 4 * g;
    if constexpr (VEC) {
      if (d < D) *reinterpret_cast<f32x4*>(p + d) = acc[t] * mul;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (d + i < D) p[d + i] = acc[t][i] * mul;
    }
  }
}
__device__ __forceinline__ float over_rows_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float over_rows_sum(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

// rows of one head of two matrices into LDS, padded to 32 with zeros; four chunks of each are in flight a thread
template <int FT, int NT, bool VEC>
__device__ __forceinline__ void jet_fill(float* __restrict__ d0, float* __restrict__ d1, const float* __restrict__ s0, int64_t ld0,
                                         const float* __restrict__ s1, int64_t ld1, const int* list, int n, int D) {
  constexpr int CH = 4 * FT;
  const int work = ((n + 31) & ~31) * CH;
  for (int it0 = threadIdx.x; it0 < work; it0 += 4 * NT) {
    u32x4 c0[4], c1[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int it = it0 + j * NT, row = it / CH, ch = it % CH;
      const bool ok = row < n;
      const int64_t slot = ok ? list[row] : 0;
      c0[j] = load_chunk<float, VEC>(s0 + slot * ld0, ch * 4, D, ok);
      c1[j] = load_chunk<float, VEC>(s1 + slot * ld1, ch * 4, D, ok);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int it = it0 + j * NT, at = (it / CH) * jet_pitch<FT>() + (it % CH) * 4;
      if (it < work) {
        *reinterpret_cast<u32x4*>(d0 + at) = c0[j];
        *reinterpret_cast<u32x4*>(d1 + at) = c1[j];
      }
    }
  }
}

// lists of kept keys and queries by two waves; counts[0], counts[1]
template <int NW>
__device__ __forceinline__ void jet_lists(const float* mk, int Nk, int* klist, const float* mq, int Nq, int* qlist, int* counts) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  if (wave == 0) {
    const int c = keep_list(mk, Nk, klist);
    if (lane == 0) counts[0] = c;
  }
  if (wave == NW - 1) {
    const int c = keep_list(mq, Nq, qlist);
    if (lane == 0) counts[1] = c;
  }
}

template <int FT, int NW, bool VEC>
__global__ void __launch_bounds__(64 * NW, 4) jet_fwd_kernel(JetArgs a) {
  constexpr int P = jet_pitch<FT>();
  extern __shared__ __attribute__((aligned(16))) float jsm[];
  const Shape& sh = a.sh;
  int b, item;
  if (!a.map.decode(blockIdx.x, b, item)) return;
  const int hk = item / a.parts, part = item - hk * a.parts;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  float *Ks = jsm, *Vs = Ks + a.nkp * P;
  int* klist = reinterpret_cast<int*>(Vs + a.nkp * P);
  int* qlist = klist + a.nkp;
  int* counts = qlist + a.nqp;
  const int64_t qrow = (int64_t)b * sh.Nq, krow = (int64_t)b * sh.Nk;
  const float* mq = a.mq ? a.mq + qrow : nullptr;
  jet_lists<NW>(a.mk ? a.mk + krow : nullptr, sh.Nk, klist, mq, sh.Nq, qlist, counts);
  const int heads = sh.g, h0 = hk * sh.g;
  if (mq && part == 0) {
    zero_masked_rows<64 * NW, VEC>(a.o + qrow * a.out_ld + (int64_t)h0 * sh.D, a.out_ld, mq, 0, sh.Nq, 1, heads * sh.D);
    if (a.lse)
      for (int n = threadIdx.x; n < sh.Nq; n += 64 * NW)
        if (mq[n] == 0.0f)
          for (int hd = 0; hd < heads; ++hd) a.lse[((int64_t)b * sh.nh + h0 + hd) * sh.Nq + n] = -INFINITY;
  }
  __syncthreads();
  const int nk = counts[0], nq = counts[1];
  const int qt = (nq + 15) >> 4, items = heads * qt, step = NW * a.parts;
  const float* qb = a.q + qrow * a.q_ld + (int64_t)h0 * sh.D;
  f32x4 nf[FT];
  auto fetch = [&](int it) {                      // the next item's query rows
    const int hd = it / qt, r = (it - hd * qt) * 16 + col;
    const bool ok = it < items && r < nq;
    jet_row<FT, VEC>(nf, ok ? qb + (int64_t)qlist[r] * a.q_ld + (int64_t)hd * sh.D : nullptr, sh.D, ok);
  };
  int it = part * NW + wave;
  if (qt) fetch(it);
  jet_fill<FT, 64 * NW, VEC>(Ks, Vs, a.k + krow * a.k_ld + (int64_t)hk * sh.D, a.k_ld, a.v + krow * a.v_ld + (int64_t)hk * sh.D, a.v_ld, klist, nk, sh.D);
  __syncthreads();
  const float c = a.scale * kLog2e;
  for (; it < items; it += step) {
    const int hd = it / qt, r = (it - hd * qt) * 16 + col;
    f32x4 qf[FT], acc[FT];
#pragma unroll
    for (int t = 0; t < FT; ++t) {
      qf[t] = nf[t];
      acc[t] = zero4();
    }
    fetch(it + step);
    float m = -INFINITY, l = 0.0f;
    for (int kt = 0; kt < nk; kt += 64) {
      const float *kh = Ks + kt * P, *vh = Vs + kt * P;
      const int left = nk - kt, subs = min(4, (left + 15) >> 4);
      f32x4 s[4];
      float top = -INFINITY;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (u < subs) s[u] = jet_dot<FT>(kh + u * 16 * P, qf);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (16 * u + 4 * g + i >= left) s[u][i] = -INFINITY;
          top = fmaxf(top, s[u][i]);
        }
      }
      const float mn = fmaxf(m, over_rows_max(top)), ms = mn == -INFINITY ? 0.0f : mn;
      const float alpha = __builtin_amdgcn_exp2f((m - ms) * c);
      l *= alpha;
#pragma unroll
      for (int t = 0; t < FT; ++t) acc[t] *= alpha;
      m = mn;
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (u < subs) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            s[u][i] = __builtin_amdgcn_exp2f((s[u][i] - ms) * c);
            l += s[u][i];
          }
          jet_cols<FT>(vh + u * 16 * P, s[u], acc);
        }
    }
    l = over_rows_sum(l);
    if (r < nq) {
      const int n = qlist[r];
      jet_store<FT, VEC>(a.o + (qrow + n) * a.out_ld + (int64_t)(h0 + hd) * sh.D, acc, l == 0.0f ? 0.0f : 1.0f / l, sh.D);
      if (a.lse && g == 0) a.lse[((int64_t)b * sh.nh + h0 + hd) * sh.Nq + n] = l == 0.0f ? -INFINITY : m * a.scale + logf(l);
    }
  }
}

template <int FT, int NW, bool VEC>
__global__ void __launch_bounds__(64 * NW, 4) jet_bwd_kernel(JetArgs a) {
  constexpr int P = jet_pitch<FT>();
  extern __shared__ __attribute__((aligned(16))) float jsm[];
  const Shape& sh = a.sh;
  int b, hk;
  if (!a.map.decode(blockIdx.x, b, hk)) return;
  const int heads = sh.g, h0 = hk * sh.g;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int qs = a.nqp * P, big = max(a.nkp * P, heads * qs);
  float *A0 = jsm, *A1 = A0 + big, *sl = A1 + big, *sd = sl + heads * a.nqp;          // K / q, V / dout, log-sums, deltas
  int* klist = reinterpret_cast<int*>(sd + heads * a.nqp);
  int* qlist = klist + a.nkp;
  int* counts = qlist + a.nqp;
  const int64_t qrow = (int64_t)b * sh.Nq, krow = (int64_t)b * sh.Nk;
  const float *mq = a.mq ? a.mq + qrow : nullptr, *mk = a.mk ? a.mk + krow : nullptr;
  jet_lists<NW>(mk, sh.Nk, klist, mq, sh.Nq, qlist, counts);
  if (mq) zero_masked_rows<64 * NW, VEC>(a.dq + qrow * a.dq_ld + (int64_t)h0 * sh.D, a.dq_ld, mq, 0, sh.Nq, 1, heads * sh.D);
  if (mk) {
    zero_masked_rows<64 * NW, VEC>(a.dk + krow * a.dk_ld + (int64_t)hk * sh.D, a.dk_ld, mk, 0, sh.Nk, 1, sh.D);
    zero_masked_rows<64 * NW, VEC>(a.dv + krow * a.dv_ld + (int64_t)hk * sh.D, a.dv_ld, mk, 0, sh.Nk, 1, sh.D);
  }
  __syncthreads();
  const int nk = counts[0], nq = counts[1];
  const float* qb = a.q + qrow * a.q_ld + (int64_t)h0 * sh.D;
  const float* gb = a.dout + qrow * a.dout_ld + (int64_t)h0 * sh.D;
  const float* ob = a.out + qrow * a.out_ld + (int64_t)h0 * sh.D;
  const float* kb = a.k + krow * a.k_ld + (int64_t)hk * sh.D;
  const float* vb = a.v + krow * a.v_ld + (int64_t)hk * sh.D;
  const int qt = (nq + 15) >> 4, kt = (nk + 15) >> 4;

  // ---- dq: keys resident
  f32x4 nqf[FT], ngf[FT];
  float nl = INFINITY, nd = 0.0f;
  auto fetch_q = [&](int it) {
    const int hd = it / qt, r = (it - hd * qt) * 16 + col;
    const bool ok = it < heads * qt && r < nq;
    const int64_t n = ok ? qlist[r] : 0;
    f32x4 of[FT];
    jet_row<FT, VEC>(nqf, qb + n * a.q_ld + (int64_t)hd * sh.D, sh.D, ok);
    jet_row<FT, VEC>(ngf, gb + n * a.dout_ld + (int64_t)hd * sh.D, sh.D, ok);
    jet_row<FT, VEC>(of, ob + n * a.out_ld + (int64_t)hd * sh.D, sh.D, ok);
    nl = ok ? row_stat<float>(a.lse[((int64_t)b * sh.nh + h0 + hd) * sh.Nq + n]) : INFINITY;
    nd = 0.0f;
#pragma unroll
    for (int t = 0; t < FT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) nd = fmaf(of[t][i], ngf[t][i], nd);
  };
  jet_fill<FT, 64 * NW, VEC>(A0, A1, kb, a.k_ld, vb, a.v_ld, klist, nk, sh.D);
  if (qt) fetch_q(wave);
  __syncthreads();
  for (int it = wave; it < heads * qt; it += NW) {
    const int hd = it / qt, r0 = (it - hd * qt) * 16;
    f32x4 qf[FT], gf[FT], acc[FT];
    const float lse = nl;
    float delta = over_rows_sum(nd);
#pragma unroll
    for (int t = 0; t < FT; ++t) {
      qf[t] = nqf[t];
      gf[t] = ngf[t];
      acc[t] = zero4();
    }
    if (it + NW < heads * qt) fetch_q(it + NW);
    for (int k0 = 0; k0 < nk; k0 += 32) {         // two tiles at a time: their chains of products interleave
      const float *kh = A0 + k0 * P, *vh = A1 + k0 * P;
      f32x4 s[2], dp[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        s[u] = jet_dot<FT>(kh + u * 16 * P, qf);
        dp[u] = jet_dot<FT>(vh + u * 16 * P, gf);
      }
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[u][i] = k0 + 16 * u + 4 * g + i < nk ? prob<float>(s[u][i], a.scale, 0.0f, lse) : 0.0f;
      if (nk <= 32) {                             // the whole row at once: delta from p and dp, p normalised by its own sum
        float sum = 0.0f;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) sum += s[u][i];
        sum = over_rows_sum(sum);
        delta = 0.0f;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) delta = fmaf(sum == 0.0f ? 0.0f : s[u][i] / sum, dp[u][i], delta);
        delta = over_rows_sum(delta);
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int i = 0; i < 4; ++i) s[u][i] *= dp[u][i] - delta;
        jet_cols<FT>(kh + u * 16 * P, s[u], acc);
      }
    }
    if (g == 0) {
      sl[hd * a.nqp + r0 + col] = lse;
      sd[hd * a.nqp + r0 + col] = lse == INFINITY ? 0.0f : delta;
    }
    if (r0 + col < nq) jet_store<FT, VEC>(a.dq + (qrow + qlist[r0 + col]) * a.dq_ld + (int64_t)(h0 + hd) * sh.D, acc, a.scale, sh.D);
  }
  if (qt & 1)                                     // (dk and dv walk two tiles at a time: no weight in the odd one)
    for (int i = threadIdx.x; i < heads * 16; i += 64 * NW) {
      sl[(i >> 4) * a.nqp + qt * 16 + (i & 15)] = INFINITY;
      sd[(i >> 4) * a.nqp + qt * 16 + (i & 15)] = 0.0f;
    }
  // ---- dk, dv: queries resident
  f32x4 kf[FT], vf[FT];
  auto fetch_k = [&](int it) {
    const int r = it * 16 + col;
    const bool ok = r < nk;
    const int64_t n = ok ? klist[r] : 0;
    jet_row<FT, VEC>(kf, kb + n * a.k_ld, sh.D, ok);
    jet_row<FT, VEC>(vf, vb + n * a.v_ld, sh.D, ok);
  };
  fetch_k(wave);
  __syncthreads();                                // K and V have been read
  for (int gi = 0; gi < heads; ++gi)
    jet_fill<FT, 64 * NW, VEC>(A0 + gi * qs, A1 + gi * qs, qb + (int64_t)gi * sh.D, a.q_ld, gb + (int64_t)gi * sh.D, a.dout_ld, qlist, nq, sh.D);
  __syncthreads();
  for (int it = wave; it < kt; it += NW) {
    const int r = it * 16 + col;
    if (it != wave) fetch_k(it);
    f32x4 dk[FT], dv[FT];
#pragma unroll
    for (int t = 0; t < FT; ++t) {
      dk[t] = zero4();
      dv[t] = zero4();
    }
    for (int gi = 0; gi < heads; ++gi)
      for (int q0 = 0; q0 < nq; q0 += 32) {
        const float *qh = A0 + gi * qs + q0 * P, *gh = A1 + gi * qs + q0 * P;
        f32x4 s[2], dp[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          s[u] = jet_dot<FT>(qh + u * 16 * P, kf);
          dp[u] = jet_dot<FT>(gh + u * 16 * P, vf);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const f32x4 ls = *reinterpret_cast<const f32x4*>(sl + gi * a.nqp + q0 + 16 * u + 4 * g);
          const f32x4 dl = *reinterpret_cast<const f32x4*>(sd + gi * a.nqp + q0 + 16 * u + 4 * g);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            s[u][i] = prob<float>(s[u][i], a.scale, 0.0f, ls[i]);
            dp[u][i] = s[u][i] * (dp[u][i] - dl[i]);
          }
          jet_cols<FT>(gh + u * 16 * P, s[u], dv);
          jet_cols<FT>(qh + u * 16 * P, dp[u], dk);
        }
      }
    if (r < nk) {
      const int64_t n = krow + klist[r];
      jet_store<FT, VEC>(a.dk + n * a.dk_ld + (int64_t)hk * sh.D, dk, a.scale, sh.D);
      jet_store<FT, VEC>(a.dv + n * a.dv_ld + (int64_t)hk * sh.D, dv, 1.0f, sh.D);
    }
  }
}

// ---- host --------------------------------------------------------------------------------------------------------
constexpr int kJetBudget = 53 * 1024;             // three workgroups on a CU

static int64_t jet_bytes(const Shape& s, bool bwd) {
  const int64_t pitch = s.D <= 16 ? 20 : 36, nkp = (s.Nk + 31) / 32 * 32, nqp = (s.Nq + 31) / 32 * 32;
  int64_t rows = nkp;
  if (bwd && s.g * nqp > rows) rows = s.g * nqp;
  return (2 * rows * pitch + (bwd ? 2 * s.g * nqp : 0) + nkp + nqp + 4) * 4;
}
bool jets_fit(const Shape& s, int dtype, bool bwd) {
  return dtype == MMB_DT_F32 && s.D <= 32 && s.Nk <= 1024 && s.Nq <= 1024 && s.Nq >= 8 && (int64_t)s.B * s.nkv >= 256 && jet_bytes(s, bwd) <= kJetBudget;
}

template <bool BWD, int FT, bool VEC>
static int launch_jets(JetArgs& a, hipStream_t st) {
  constexpr int NW = 4;                           // (eight waves: 1.05 the time forward, 1.2 in training)
  const Shape& s = a.sh;
  a.nkp = (s.Nk + 31) / 32 * 32;
  a.nqp = (s.Nq + 31) / 32 * 32;
  a.parts = 1;                                    // forward: a head's query tiles over several workgroups while the chip is not full
  if (!BWD)
    while ((int64_t)s.B * s.nkv * a.parts < 1024 && a.parts * NW < s.g * (a.nqp / 16)) a.parts *= 2;
  a.map = {s.B, s.nkv * a.parts, s.B % 8 == 0 || s.B >= 64 ? 1 : 0};
  MMB_REQUIRE(grid_fits(a.map.blocks(), 64 * NW), "mmb_cross_attention: %lld workgroups are more than a launch takes", (long long)a.map.blocks());
  void (*kern)(JetArgs);
  if constexpr (BWD) kern = jet_bwd_kernel<FT, NW, VEC>;
  else kern = jet_fwd_kernel<FT, NW, VEC>;
  kern<<<dim3((unsigned)a.map.blocks()), dim3(64 * NW), (size_t)jet_bytes(s, BWD), st>>>(a);
  return check_launch(BWD ? "mmb_cross_attention_bwd (jets)" : "mmb_cross_attention_fwd (jets)");
}

int jets_fwd(const Shape& s, bool vec, const float* q, int64_t q_ld, const float* k, int64_t k_ld, const float* v, int64_t v_ld,
             const float* mq, const float* mk, float scale, float* out, int64_t out_ld, float* lse, hipStream_t st) {
  JetArgs a = {};
  a.sh = s; a.q = q; a.q_ld = q_ld; a.k = k; a.k_ld = k_ld; a.v = v; a.v_ld = v_ld; a.mq = mq; a.mk = mk; a.scale = scale;
  a.o = out; a.out_ld = out_ld; a.lse = lse;
  if (s.D <= 16) return vec ? launch_jets<false, 1, true>(a, st) : launch_jets<false, 1, false>(a, st);
  return vec ? launch_jets<false, 2, true>(a, st) : launch_jets<false, 2, false>(a, st);
}
int jets_bwd(const Shape& s, bool vec, const float* q, int64_t q_ld, const float* k, int64_t k_ld, const float* v, int64_t v_ld,
             const float* mq, const float* mk, float scale, const float* out, int64_t out_ld, const float* dout, int64_t dout_ld,
             const float* lse, float* dq, int64_t dq_ld, float* dk, int64_t dk_ld, float* dv, int64_t dv_ld, hipStream_t st) {
  JetArgs a = {};
  a.sh = s; a.q = q; a.q_ld = q_ld; a.k = k; a.k_ld = k_ld; a.v = v; a.v_ld = v_ld; a.mq = mq; a.mk = mk; a.scale = scale;
  a.out = out; a.out_ld = out_ld; a.dout = dout; a.dout_ld = dout_ld; a.lse = const_cast<float*>(lse);
  a.dq = dq; a.dq_ld = dq_ld; a.dk = dk; a.dk_ld = dk_ld; a.dv = dv; a.dv_ld = dv_ld;
  if (s.D <= 16) return vec ? launch_jets<true, 1, true>(a, st) : launch_jets<true, 1, false>(a, st);
  return vec ? launch_jets<true, 2, true>(a, st) : launch_jets<true, 2, false>(a, st);
}

}  // namespace xattn
}  // namespace mmb
