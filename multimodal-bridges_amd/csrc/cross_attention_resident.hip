// Cross attention of small clouds (jets): the keys of a head fit into LDS whole.
//
// With some hundred slots a cloud is a few 32 x 32 tiles a head, and what a call costs is not its products but the chain
// mask -> kept slots -> rows -> products of every workgroup.  Here a workgroup owns one key head of one cloud: the masks are
// read and compacted once, and after ONE barrier every wave walks its own (query head, 32 rows) items without meeting the
// others.  The reverse does this twice, with K and V resident for dq and with q and dout resident for dk and dv; delta stays in
// LDS between the two.  What counts is how many workgroups a CU holds at once (their chains hide each other): two or four
// heads a workgroup, which would share the masks and read longer row segments, need as much more LDS and measured 1.04 to
// 1.4 times the time; eight waves instead of four 1.1 to 1.3 times.
#include "cross_attention.h"

namespace mmb {
namespace xattn {

template <typename T, int DP>
struct ResTile {
  static constexpr int E = Traits<T>::EPC, CH = DP / E, PITCH = row_pitch<T, DP>(), FT = DP / 32;
};

struct ResArgs {
  Shape sh;
  const void *q, *k, *v, *out, *dout;
  int64_t q_ld, k_ld, v_ld, out_ld, dout_ld, dq_ld, dk_ld, dv_ld;
  const float *mq, *mk;
  float* lse;
  float scale;
  void *o, *dq, *dk, *dv;
  int parts;                                      // workgroups that share a head's query tiles (forward)
  int nkp, nqp;                                   // slots padded to 32
  GridMap map;                                    // units = clouds, items = key heads * parts
};

// rows of one head of two matrices into LDS, padded to 32 with zeros; four chunks of each are in flight a thread
template <typename T, int DP, int NT, bool VEC>
__device__ __forceinline__ void fill2(T* __restrict__ d0, T* __restrict__ d1, const T* __restrict__ s0, int64_t ld0, const T* __restrict__ s1,
                                      int64_t ld1, const int* list, int n, int D) {
  using R = ResTile<T, DP>;
  const int work = ((n + 31) & ~31) * R::CH;
  for (int it0 = threadIdx.x; it0 < work; it0 += 4 * NT) {
    u32x4 c0[4], c1[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int it = it0 + j * NT, row = it / R::CH, ch = it % R::CH;
      const bool ok = row < n;
      const int64_t slot = ok ? list[row] : 0;
      c0[j] = load_chunk<T, VEC>(s0 + slot * ld0, ch * R::E, D, ok);
      c1[j] = load_chunk<T, VEC>(s1 + slot * ld1, ch * R::E, D, ok);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int it = it0 + j * NT;
      if (it < work) {
        *reinterpret_cast<u32x4*>(d0 + chunk_at<T, DP>(it / R::CH, it % R::CH)) = c0[j];
        *reinterpret_cast<u32x4*>(d1 + chunk_at<T, DP>(it / R::CH, it % R::CH)) = c1[j];
      }
    }
  }
}

// (no instance here may spill registers: cross_attention_bwd.hip says why)
template <typename T, int DP, int NW, bool VEC>
__global__ void __launch_bounds__(64 * NW, DP < 128 ? 3 : sizeof(T) == 4 && !VEC ? 1 : 2) res_fwd_kernel(ResArgs a) {
  using R = ResTile<T, DP>;
  constexpr int S = DP / (2 * R::E);
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const Shape& sh = a.sh;
  int b, item;
  if (!a.map.decode(blockIdx.x, b, item)) return;
  const int hk = item / a.parts, part = item - hk * a.parts;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, col = lane & 31, h = lane >> 5;
  T* Ks = reinterpret_cast<T*>(lds);
  T* Vs = Ks + a.nkp * R::PITCH;
  int* klist = reinterpret_cast<int*>(Vs + a.nkp * R::PITCH);
  int* qlist = klist + a.nkp;
  int* counts = qlist + a.nqp;
  const float* mq = a.mq ? a.mq + (int64_t)b * sh.Nq : nullptr;
  const float* mk = a.mk ? a.mk + (int64_t)b * sh.Nk : nullptr;
  if (wave == 0) {
    const int c = keep_list(mk, sh.Nk, klist);
    if (lane == 0) counts[0] = c;
  }
  if (wave == NW - 1) {
    const int c = keep_list(mq, sh.Nq, qlist);
    if (lane == 0) counts[1] = c;
  }
  const int heads = sh.g, h0 = hk * sh.g;
  if (mq && part == 0) {                          // masked queries: zero rows over all heads of the workgroup, no log-sum
    zero_masked_rows<64 * NW, VEC>((T*)a.o + (int64_t)b * sh.Nq * a.out_ld + (int64_t)h0 * sh.D, a.out_ld, mq, 0, sh.Nq, 1, heads * sh.D);
    if (a.lse)
      for (int i = threadIdx.x; i < heads * sh.Nq; i += 64 * NW) {
        const int hd = i / sh.Nq, n = i - hd * sh.Nq;
        if (mq[n] == 0.0f) a.lse[((int64_t)b * sh.nh + h0 + hd) * sh.Nq + n] = -INFINITY;
      }
  }
  __syncthreads();
  const int nk = counts[0], nq = counts[1];
  const int64_t krow = (int64_t)b * sh.Nk;
  const float c = a.scale * kLog2e;
  const int qt = (nq + 31) >> 5, items = heads * qt, step = NW * a.parts;
  const T* qb = (const T*)a.q + (int64_t)b * sh.Nq * a.q_ld + (int64_t)h0 * sh.D;
  u32x4 nf[S];                                    // the next item's query rows
  auto fetch = [&](int it) {
    const int hd = it / qt, r = (it - hd * qt) * 32 + col;
    const bool ok = it < items && r < nq;
    load_row<T, DP, VEC>(nf, ok ? qb + (int64_t)qlist[r] * a.q_ld + (int64_t)hd * sh.D : nullptr, sh.D, ok);
  };
  int it = part * NW + wave;
  if (qt) fetch(it);
  fill2<T, DP, 64 * NW, VEC>(Ks, Vs, (const T*)a.k + krow * a.k_ld + (int64_t)hk * sh.D, a.k_ld,
                             (const T*)a.v + krow * a.v_ld + (int64_t)hk * sh.D, a.v_ld, klist, nk, sh.D);
  __syncthreads();
  for (; it < items; it += step) {
    const int hd = it / qt, r = (it - hd * qt) * 32 + col;
    u32x4 qf[S];
#pragma unroll
    for (int s = 0; s < S; ++s) qf[s] = nf[s];
    fetch(it + step);
    f32x16 acc[R::FT];
#pragma unroll
    for (int t = 0; t < R::FT; ++t) acc[t] = zero16();
    float m = -INFINITY, l = 0.0f;
    for (int kt = 0; kt < nk; kt += 32) attend<T, DP, 32>(Ks + kt * R::PITCH, Vs + kt * R::PITCH, nk - kt, qf, c, m, l, acc);
    l += __shfl_xor(l, 32);
    if (r < nq) {
      const int n = qlist[r];
      store_col<T, DP, VEC>((T*)a.o + ((int64_t)b * sh.Nq + n) * a.out_ld + (int64_t)(h0 + hd) * sh.D, acc, l == 0.0f ? 0.0f : 1.0f / l, sh.D, again(threadIdx.x));
      if (a.lse && h == 0) a.lse[((int64_t)b * sh.nh + h0 + hd) * sh.Nq + n] = row_lse<T>(m, l, a.scale);
    }
  }
}

template <typename T, int DP, int NW, bool VEC>
__global__ void __launch_bounds__(64 * NW, DP == 128 || (DP == 64 && sizeof(T) == 4 && !VEC) ? 1 : 2) res_bwd_kernel(ResArgs a) {
  using R = ResTile<T, DP>;
  constexpr int S = DP / (2 * R::E), E = R::E;
  constexpr bool HALF = __is_same(T, _Float16);
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const Shape& sh = a.sh;
  int b, item;
  if (!a.map.decode(blockIdx.x, b, item)) return;
  const int hk = item, heads = sh.g, h0 = hk * sh.g;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, col = lane & 31, h = lane >> 5;
  const int qs = a.nqp * R::PITCH, big = max(a.nkp * R::PITCH, heads * qs);
  T* A0 = reinterpret_cast<T*>(lds);              // K, then q
  T* A1 = A0 + big;                               // V, then dout
  float* sl = reinterpret_cast<float*>(A1 + big);                      // [head][nqp] log-sums, then deltas
  float* sd = sl + heads * a.nqp;
  int* klist = reinterpret_cast<int*>(sd + heads * a.nqp);
  int* qlist = klist + a.nkp;
  int* counts = qlist + a.nqp;
  const float* mq = a.mq ? a.mq + (int64_t)b * sh.Nq : nullptr;
  const float* mk = a.mk ? a.mk + (int64_t)b * sh.Nk : nullptr;
  if (wave == 0) {
    const int c = keep_list(mk, sh.Nk, klist);
    if (lane == 0) counts[0] = c;
  }
  if (wave == NW - 1) {
    const int c = keep_list(mq, sh.Nq, qlist);
    if (lane == 0) counts[1] = c;
  }
  const int64_t krow = (int64_t)b * sh.Nk, qrow = (int64_t)b * sh.Nq;
  if (mq) zero_masked_rows<64 * NW, VEC>((T*)a.dq + qrow * a.dq_ld + (int64_t)h0 * sh.D, a.dq_ld, mq, 0, sh.Nq, 1, heads * sh.D);
  if (mk) {
    zero_masked_rows<64 * NW, VEC>((T*)a.dk + krow * a.dk_ld + (int64_t)hk * sh.D, a.dk_ld, mk, 0, sh.Nk, 1, sh.D);
    zero_masked_rows<64 * NW, VEC>((T*)a.dv + krow * a.dv_ld + (int64_t)hk * sh.D, a.dv_ld, mk, 0, sh.Nk, 1, sh.D);
  }
  __syncthreads();
  const int nk = counts[0], nq = counts[1];
  const float c = a.scale * kLog2e;
  const T* qb = (const T*)a.q + qrow * a.q_ld + (int64_t)h0 * sh.D;
  const T* gb = (const T*)a.dout + qrow * a.dout_ld + (int64_t)h0 * sh.D;
  const T* ob = (const T*)a.out + qrow * a.out_ld + (int64_t)h0 * sh.D;
  const T* kb = (const T*)a.k + krow * a.k_ld + (int64_t)hk * sh.D;
  const T* vb = (const T*)a.v + krow * a.v_ld + (int64_t)hk * sh.D;

  // ---- dq: keys resident
  const int qt = (nq + 31) >> 5, kt = (nk + 31) >> 5;
  u32x4 nqf[S], ngf[S], nof[S];
  float nl = INFINITY;
  auto fetch_q = [&](int it) {
    const int hd = it / qt, r = (it - hd * qt) * 32 + col;
    const bool ok = it < heads * qt && r < nq;
    const int64_t n = ok ? qlist[r] : 0;
    load_row<T, DP, VEC>(nqf, qb + n * a.q_ld + (int64_t)hd * sh.D, sh.D, ok);
    load_row<T, DP, VEC>(ngf, gb + n * a.dout_ld + (int64_t)hd * sh.D, sh.D, ok);
    load_row<T, DP, VEC>(nof, ob + n * a.out_ld + (int64_t)hd * sh.D, sh.D, ok);
    nl = ok ? row_stat<T>(a.lse[((int64_t)b * sh.nh + h0 + hd) * sh.Nq + n]) : INFINITY;
  };
  if (qt) fetch_q(wave);
  fill2<T, DP, 64 * NW, VEC>(A0, A1, kb, a.k_ld, vb, a.v_ld, klist, nk, sh.D);
  __syncthreads();
  for (int it = wave; it < heads * qt; it += NW) {
    const int hd = it / qt, r0 = (it - hd * qt) * 32;
    u32x4 qf[S], gf[S];
    float delta = 0.0f;
    const float lse = nl;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      qf[s] = nqf[s];
      gf[s] = ngf[s];
      T x[E], y[E];
      __builtin_memcpy(x, &nof[s], 16);
      __builtin_memcpy(y, &gf[s], 16);
#pragma unroll
      for (int i = 0; i < E; ++i) delta = fmaf((float)x[i], (float)y[i], delta);
    }
    delta += __shfl_xor(delta, 32);
    fetch_q(it + NW);
    const T *kh = A0, *vh = A1;
    f32x16 acc[R::FT];
#pragma unroll
    for (int t = 0; t < R::FT; ++t) acc[t] = zero16();
    if (nk <= 32) {                               // the whole row at once: delta from p and dp (as few_keys elsewhere)
      f32x16 s = dot_rows<T, DP>(kh, 0, qf, zero16());
      const f32x16 dp = dot_rows<T, DP>(vh, 0, gf, zero16());
      float sum = 0.0f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[r] = crow(r, h) < nk ? prob<T>(s[r], a.scale, c, lse) : 0.0f;
        sum += s[r];
      }
      sum += __shfl_xor(sum, 32);
      delta = 0.0f;
#pragma unroll
      for (int r = 0; r < 16; ++r) delta = fmaf(sum == 0.0f ? 0.0f : s[r] / sum, dp[r], delta);
      delta += __shfl_xor(delta, 32);
    }
    if (h == 0) {
      sl[hd * a.nqp + r0 + col] = HALF ? lse - kHalfLog : lse;
      sd[hd * a.nqp + r0 + col] = lse == INFINITY ? 0.0f : delta;
    }
    ColScale cs;
    float st = HALF ? lse - log2_pow2(cs.sc) : lse;
    for (int kt0 = 0; kt0 < nk; kt0 += 32) {
      f32x16 s = dot_rows<T, DP>(kh, kt0, qf, zero16());
      const f32x16 dp = dot_rows<T, DP>(vh, kt0, gf, zero16());
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = prob<T>(s[r], a.scale, c, st) * (dp[r] - delta);
      if (kt0 + 32 > nk) {
        rarely();
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (kt0 + crow(r, h) >= nk) s[r] = 0.0f;
      }
      if constexpr (HALF) {
        if (cs.fit<1>(&s, acc, R::FT)) st = lse - log2_pow2(cs.sc);
      }
      dot_cols<T, DP>(kh, kt0, s, acc);
    }
    if (r0 + col < nq)
      store_col<T, DP, VEC>((T*)a.dq + (qrow + qlist[r0 + col]) * a.dq_ld + (int64_t)(h0 + hd) * sh.D, acc, HALF ? a.scale / cs.sc : a.scale, sh.D, again(threadIdx.x));
  }
  // ---- dk, dv: queries resident
  u32x4 kf[S], vf[S];
  auto fetch_k = [&](int it) {
    const int r = it * 32 + col;
    const bool ok = r < nk;
    const int64_t n = ok ? klist[r] : 0;
    load_row<T, DP, VEC>(kf, kb + n * a.k_ld, sh.D, ok);
    load_row<T, DP, VEC>(vf, vb + n * a.v_ld, sh.D, ok);
  };
  fetch_k(wave);
  __syncthreads();                                // K and V have been read
  for (int gi = 0; gi < heads; ++gi)
    fill2<T, DP, 64 * NW, VEC>(A0 + gi * qs, A1 + gi * qs, qb + (int64_t)gi * sh.D, a.q_ld, gb + (int64_t)gi * sh.D, a.dout_ld, qlist, nq, sh.D);
  __syncthreads();
  const int h2 = (again(threadIdx.x) & 63) >> 5;
  for (int it = wave; it < kt; it += NW) {
    const int r = it * 32 + col;
    if (it != wave) fetch_k(it);
    f32x16 dk[R::FT], dv[R::FT];
#pragma unroll
    for (int t = 0; t < R::FT; ++t) {
      dk[t] = zero16();
      dv[t] = zero16();
    }
    ColScale cs;
    for (int gi = 0; gi < sh.g; ++gi) {
      const T* qh = A0 + gi * qs;
      const T* gh = A1 + gi * qs;
      const float* lh = sl + gi * a.nqp;
      const float* dh = sd + gi * a.nqp;
      for (int q0 = 0; q0 < nq; q0 += 32) {
        f32x16 s = dot_rows<T, DP>(qh, q0, kf, zero16());
        f32x16 dp = dot_rows<T, DP>(gh, q0, vf, zero16());
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4) {
          const f32x4 ls = *reinterpret_cast<const f32x4*>(lh + q0 + 8 * g4 + 4 * h2);
          const f32x4 dl = *reinterpret_cast<const f32x4*>(dh + q0 + 8 * g4 + 4 * h2);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r2 = 4 * g4 + i;
            s[r2] = prob<T>(s[r2], a.scale, c, ls[i]);      // (rows past the end: log-sum +inf, p = 0)
            dp[r2] = s[r2] * (dp[r2] - dl[i]);
          }
        }
        if constexpr (HALF) {
#pragma unroll
          for (int r2 = 0; r2 < 16; ++r2) dp[r2] *= cs.sc;
          cs.fit<1>(&dp, dk, R::FT);
        }
        dot_cols<T, DP>(gh, q0, s, dv);
        dot_cols<T, DP>(qh, q0, dp, dk);
      }
    }
    if (r < nk) {
      const int64_t n = krow + klist[r];
      const int t = again(threadIdx.x);           // (feature places found again: no register to spare for them)
      store_col<T, DP, VEC>((T*)a.dk + n * a.dk_ld + (int64_t)hk * sh.D, dk, HALF ? a.scale / kHalfP / cs.sc : a.scale, sh.D, t);
      store_col<T, DP, VEC>((T*)a.dv + n * a.dv_ld + (int64_t)hk * sh.D, dv, HALF ? 1.0f / kHalfP : 1.0f, sh.D, t);
    }
  }
}

// ---- host --------------------------------------------------------------------------------------------------------
constexpr int kResBudget = 53 * 1024;             // three workgroups on a CU
constexpr int kResWaves = 4;

static int64_t res_bytes(const Shape& s, int dtype, bool bwd) {
  const int es = dtype == MMB_DT_F32 ? 4 : 2, dp = pad_width(s.D), pitch = es == 2 ? dp : dp + 4;
  const int64_t nkp = (s.Nk + 31) / 32 * 32, nqp = (s.Nq + 31) / 32 * 32;
  int64_t rows = nkp;
  if (bwd && s.g * nqp > rows) rows = s.g * nqp;
  return 2 * rows * pitch * es + (bwd ? 2 * s.g * nqp * 4 : 0) + (nkp + nqp + 4) * 4;
}
// Whether a cloud is small: its workgroups leave room for two others on a CU (1024 clouds of 150 x 128 slots, 4 heads of 16 floats in
// 32-wide tiles: 225 us a training step against 524 in the streaming kernels; at one workgroup a CU the two are level), there are clouds for every CU -- fewer
// are spread better by the streaming kernels --, and a query tile is at least half full.
bool resident_fits(const Shape& s, int dtype, bool bwd) {
  return s.Nk <= 1024 && s.Nq <= 1024 && s.Nq >= 16 && (int64_t)s.B * s.nkv >= 256 && res_bytes(s, dtype, bwd) <= kResBudget;
}

template <bool BWD, typename T, int DP, bool VEC>
static int launch_res(ResArgs& a, int64_t bytes, hipStream_t st) {
  constexpr int NW = kResWaves;
  void (*kern)(ResArgs);
  if constexpr (BWD) kern = res_bwd_kernel<T, DP, NW, VEC>;
  else kern = res_fwd_kernel<T, DP, NW, VEC>;
  kern<<<dim3((unsigned)a.map.blocks()), dim3(64 * NW), (size_t)bytes, st>>>(a);
  return check_launch(BWD ? "mmb_cross_attention_bwd (resident)" : "mmb_cross_attention_fwd (resident)");
}
template <bool BWD, typename T, bool VEC>
static int pick_res(ResArgs& a, int dtype, int64_t bytes, hipStream_t st) {
  switch (pad_width(a.sh.D)) {
    case 32: return launch_res<BWD, T, 32, VEC>(a, bytes, st);
    case 64: return launch_res<BWD, T, 64, VEC>(a, bytes, st);
    default: return launch_res<BWD, T, 128, VEC>(a, bytes, st);
  }
}
template <bool BWD>
static int run_res(ResArgs& a, int dtype, bool vec, hipStream_t st) {
  const Shape& s = a.sh;
  a.nkp = (s.Nk + 31) / 32 * 32;
  a.nqp = (s.Nq + 31) / 32 * 32;
  // forward: a head's query tiles over several workgroups while the chip is not full
  a.parts = 1;
  if (!BWD)
    while ((int64_t)s.B * s.nkv * a.parts < 1024 && a.parts * kResWaves < s.g * (a.nqp / 32)) a.parts *= 2;
  a.map = {s.B, s.nkv * a.parts, s.B % 8 == 0 || s.B >= 64 ? 1 : 0};
  MMB_REQUIRE(grid_fits(a.map.blocks(), 64 * kResWaves), "mmb_cross_attention: %lld workgroups are more than a launch takes", (long long)a.map.blocks());
  const int64_t bytes = res_bytes(s, dtype, BWD);
  if (dtype == MMB_DT_F32) return vec ? pick_res<BWD, float, true>(a, dtype, bytes, st) : pick_res<BWD, float, false>(a, dtype, bytes, st);
  if (dtype == MMB_DT_BF16) return vec ? pick_res<BWD, __bf16, true>(a, dtype, bytes, st) : pick_res<BWD, __bf16, false>(a, dtype, bytes, st);
  return vec ? pick_res<BWD, _Float16, true>(a, dtype, bytes, st) : pick_res<BWD, _Float16, false>(a, dtype, bytes, st);
}

int resident_fwd(const Shape& s, int dtype, bool vec, const void* q, int64_t q_ld, const void* k, int64_t k_ld, const void* v,
                 int64_t v_ld, const float* mq, const float* mk, float scale, void* out, int64_t out_ld, float* lse, hipStream_t st) {
  ResArgs a = {};
  a.sh = s; a.q = q; a.q_ld = q_ld; a.k = k; a.k_ld = k_ld; a.v = v; a.v_ld = v_ld; a.mq = mq; a.mk = mk; a.scale = scale;
  a.o = out; a.out_ld = out_ld; a.lse = lse;
  return run_res<false>(a, dtype, vec, st);
}
int resident_bwd(const Shape& s, int dtype, bool vec, const void* q, int64_t q_ld, const void* k, int64_t k_ld, const void* v,
                 int64_t v_ld, const float* mq, const float* mk, float scale, const void* out, int64_t out_ld, const void* dout,
                 int64_t dout_ld, const float* lse, void* dq, int64_t dq_ld, void* dk, int64_t dk_ld, void* dv, int64_t dv_ld, hipStream_t st) {
  ResArgs a = {};
  a.sh = s; a.q = q; a.q_ld = q_ld; a.k = k; a.k_ld = k_ld; a.v = v; a.v_ld = v_ld; a.mq = mq; a.mk = mk; a.scale = scale;
  a.out = out; a.out_ld = out_ld; a.dout = dout; a.dout_ld = dout_ld; a.lse = const_cast<float*>(lse);
  a.dq = dq; a.dq_ld = dq_ld; a.dk = dk; a.dk_ld = dk_ld; a.dv = dv; a.dv_ld = dv_ld;
  return run_res<true>(a, dtype, vec, st);
}

}  // namespace xattn
}  // namespace mmb
