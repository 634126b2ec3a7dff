// Cross attention of the slots of one cloud to the slots of another, reverse.
//
//   p_ij  = exp(s_ij - lse_i)                     recomputed from q, k and the forward's log-sum
//   dp_ij = do_i . v_j      delta_i = sum_j p_ij dp_ij = do_i . o_i      ds_ij = p_ij (dp_ij - delta_i)
//   dv_j  = sum_i p_ij do_i      dq_i = scale sum_j ds_ij k_j      dk_j = scale sum_i ds_ij q_i
//
// Two launches, each owning its outputs, so that every sum runs in a fixed order and nothing is accumulated with atomics:
// dq (a wave owns 32 query rows and walks the keys; it also writes delta), then dk and dv (a wave owns 32 keys and walks
// the queries of every head that shares them).  That recomputes s and dp once: 7 products instead of the 5 that one launch
// with atomically summed dq would need.
#include "cross_attention.h"

namespace mmb {
namespace xattn {

struct BwdArgs {
  Shape sh;
  const void *q, *k, *v, *out, *dout;
  int64_t q_ld, k_ld, v_ld, out_ld, dout_ld, dq_ld, dk_ld, dv_ld;
  const float *mq, *mk, *lse;
  float scale;
  void *dq, *dk, *dv;
  float* delta;                                   // (B, nheads, Nq)
  int tiles;
  GridMap map;
};

// p from a raw score.  The product and the difference are rounded apart: a row with a single key, whose log-sum IS its
// rounded score, gets exactly 1.
__device__ __forceinline__ float prob(float s, float scale, float lse) {
#pragma clang fp contract(off)
  const float t = s * scale;
  return __builtin_amdgcn_exp2f((t - lse) * kLog2e);
}

// half precision: p in [0, 1] takes this factor into the product (p = 1 / Nk of a long list would be subnormal)
constexpr float kHalfP = 4096.0f;

template <typename T, int DP, int TK>
constexpr int dq_lds() {
  constexpr int rows = TK * row_pitch<T, DP>() * (int)sizeof(T);
  return 2 * rows + (sizeof(T) == 2 ? DP * tr_pitch<TK>() * (int)sizeof(T) : 0);
}

template <typename T, int DP, int NW, bool VEC>
__global__ void __launch_bounds__(64 * NW, 2) dq_kernel(BwdArgs a) {
  constexpr int NT = 64 * NW, TK = 32, ROWS = 32 * NW;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  int* list = reinterpret_cast<int*>(lds + dq_lds<T, DP, TK>());
  int* qlist = list + kChunk + 64 + 4;
  const Shape sh = a.sh;
  int unit, item;
  if (!a.map.decode(blockIdx.x, unit, item)) return;
  const int pair = a.map.units == sh.B ? unit * sh.nkv + item / a.tiles : unit, tile = item % a.tiles;
  const int b = pair / sh.nkv, hk = pair - b * sh.nkv;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, col = lane & 31, h = lane >> 5;
  const int R = sh.g * sh.Nq, r0 = tile * ROWS;
  const float* mq = a.mq ? a.mq + (int64_t)b * sh.Nq : nullptr;
  const float* mk = a.mk ? a.mk + (int64_t)b * sh.Nk : nullptr;
  RowTile rt = {r0 / sh.g, sh.g, qlist};
  if (mq) {
    if (threadIdx.x < 64) compact_select(mq, sh.Nq, rt.first_c, min(ROWS, R) / sh.g + 2, qlist);
    zero_masked_rows<NT>((T*)a.dq + (int64_t)b * sh.Nq * a.dq_ld + (int64_t)hk * sh.g * sh.D, a.dq_ld, mq, r0, min(ROWS, R - r0), sh.g, sh.D);
    __syncthreads();
    if (qlist[0] < 0) return;
  }
  const int row = r0 + wave * 32 + col;
  int n = -1, gi = 0;
  const bool live = row < R && rt.locate(row, sh.Nq, mq != nullptr, n, gi);
  const int head = hk * sh.g + gi;
  const int64_t flat = (int64_t)b * sh.Nq + (live ? n : 0);

  constexpr int E = Traits<T>::EPC, S = DP / (2 * E);
  u32x4 qf[S], gf[S];
  load_row<T, DP, VEC>(qf, (const T*)a.q + flat * a.q_ld + (int64_t)head * sh.D, sh.D, live);
  load_row<T, DP, VEC>(gf, (const T*)a.dout + flat * a.dout_ld + (int64_t)head * sh.D, sh.D, live);
  const int64_t stat = ((int64_t)b * sh.nh + head) * sh.Nq + n;
  float lse = live ? a.lse[stat] : INFINITY;
  if (lse == -INFINITY) lse = INFINITY;           // a row without a key (or only scores of -inf): p = 0
  float delta = 0.0f;
  {
    u32x4 of[S];
    load_row<T, DP, VEC>(of, (const T*)a.out + flat * a.out_ld + (int64_t)head * sh.D, sh.D, live);
#pragma unroll
    for (int s = 0; s < S; ++s) {
      T x[E], y[E];
      __builtin_memcpy(x, &of[s], 16);
      __builtin_memcpy(y, &gf[s], 16);
#pragma unroll
      for (int i = 0; i < E; ++i) delta = fmaf((float)x[i], (float)y[i], delta);
    }
    delta += __shfl_xor(delta, 32);
  }
  f32x16 acc[DP / 32];
#pragma unroll
  for (int t = 0; t < DP / 32; ++t) acc[t] = zero16();

  T* Ks = reinterpret_cast<T*>(lds);
  T* Vs = Ks + TK * row_pitch<T, DP>();
  T* Kt = sizeof(T) == 2 ? Vs + TK * row_pitch<T, DP>() : Ks;
  SlotTiles<NW> keys;
  keys.init(mk, 0, sh.Nk, list, list + kChunk + 64);
  const T* kb = (const T*)a.k + (int64_t)b * sh.Nk * a.k_ld + (int64_t)hk * sh.D;
  const T* vb = (const T*)a.v + (int64_t)b * sh.Nk * a.v_ld + (int64_t)hk * sh.D;
  TileRegs<T, DP, TK, NT> kr, vr;
  int nk = keys.next(TK);
  kr.template load<VEC>(threadIdx.x, nk, sh.D, [&](int i) { return kb + (int64_t)keys.slot(i) * a.k_ld; });
  vr.template load<VEC>(threadIdx.x, nk, sh.D, [&](int i) { return vb + (int64_t)keys.slot(i) * a.v_ld; });
  bool first = true;
  ColScale scale;
  while (nk > 0) {
    SlotTiles<NW>::sync();
    kr.store_rows(threadIdx.x, Ks);
    vr.store_rows(threadIdx.x, Vs);
    kr.store_tr(threadIdx.x, Kt);
    const int nn = keys.next(TK);
    kr.template load<VEC>(threadIdx.x, nn, sh.D, [&](int i) { return kb + (int64_t)keys.slot(i) * a.k_ld; });
    vr.template load<VEC>(threadIdx.x, nn, sh.D, [&](int i) { return vb + (int64_t)keys.slot(i) * a.v_ld; });
    SlotTiles<NW>::sync();
    f32x16 s = dot_rows<T, DP>(Ks, 0, qf, zero16());
    f32x16 dp = dot_rows<T, DP>(Vs, 0, gf, zero16());
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = crow(r, h) < nk ? prob(s[r], a.scale, lse) : 0.0f;
    if (first && nn == 0) {                       // the whole row is here: delta from p and dp, free of out's rounding
      delta = 0.0f;
#pragma unroll
      for (int r = 0; r < 16; ++r) delta = fmaf(s[r], dp[r], delta);
      delta += __shfl_xor(delta, 32);
    }
    // ds is rounded to the inputs' type for the product, like p in the forward; the sum over keys stays in 32 bits
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] *= dp[r] - delta;
    if constexpr (__is_same(T, _Float16)) scale.fit(s, acc, DP / 32);
    dot_cols<T, DP, TK>(Kt, 0, s, acc);
    first = false;
    nk = nn;
  }
  if (!live) return;
  if (h == 0) a.delta[stat] = delta;
  store_col<T, DP, VEC>((T*)a.dq + flat * a.dq_ld + (int64_t)head * sh.D, acc,
                        __is_same(T, _Float16) ? a.scale / scale.sc : a.scale, sh.D);
}

template <typename T, int DP>
constexpr int dkv_lds() {
  constexpr int rows = 32 * row_pitch<T, DP>() * (int)sizeof(T);
  return 2 * rows + (sizeof(T) == 2 ? 2 * DP * tr_pitch<32>() * (int)sizeof(T) : 0);
}

template <typename T, int DP, int NW, bool VEC>
__global__ void __launch_bounds__(64 * NW, DP == 128 && sizeof(T) == 4 ? 1 : 2) dkv_kernel(BwdArgs a) {
  constexpr int NT = 64 * NW, TQ = 32, COLS = 32 * NW;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  float* stats = reinterpret_cast<float*>(lds + dkv_lds<T, DP>());          // lse[32], delta[32]
  int* list = reinterpret_cast<int*>(stats + 64);
  int* klist = list + kChunk + 64 + 4;
  const Shape sh = a.sh;
  int unit, item;
  if (!a.map.decode(blockIdx.x, unit, item)) return;
  const int pair = a.map.units == sh.B ? unit * sh.nkv + item / a.tiles : unit, tile = item % a.tiles;
  const int b = pair / sh.nkv, hk = pair - b * sh.nkv;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, col = lane & 31, h = lane >> 5;
  const int k0 = tile * COLS;
  const float* mq = a.mq ? a.mq + (int64_t)b * sh.Nq : nullptr;
  const float* mk = a.mk ? a.mk + (int64_t)b * sh.Nk : nullptr;
  if (mk) {
    if (threadIdx.x < 64) compact_select(mk, sh.Nk, k0, COLS, klist);
    const int rows = min(COLS, sh.Nk - k0);
    zero_masked_rows<NT>((T*)a.dk + (int64_t)b * sh.Nk * a.dk_ld + (int64_t)hk * sh.D, a.dk_ld, mk, k0, rows, 1, sh.D);
    zero_masked_rows<NT>((T*)a.dv + (int64_t)b * sh.Nk * a.dv_ld + (int64_t)hk * sh.D, a.dv_ld, mk, k0, rows, 1, sh.D);
    __syncthreads();
    if (klist[0] < 0) return;
  }
  const int kc = k0 + wave * 32 + col;
  const int key = mk ? klist[wave * 32 + col] : (kc < sh.Nk ? kc : -1);
  const int64_t flat = (int64_t)b * sh.Nk + (key >= 0 ? key : 0);
  constexpr int E = Traits<T>::EPC, S = DP / (2 * E);
  u32x4 kf[S], vf[S];
  load_row<T, DP, VEC>(kf, (const T*)a.k + flat * a.k_ld + (int64_t)hk * sh.D, sh.D, key >= 0);
  load_row<T, DP, VEC>(vf, (const T*)a.v + flat * a.v_ld + (int64_t)hk * sh.D, sh.D, key >= 0);
  f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
  for (int t = 0; t < DP / 32; ++t) {
    dk[t] = zero16();
    dv[t] = zero16();
  }
  T* Qs = reinterpret_cast<T*>(lds);
  T* Gs = Qs + TQ * row_pitch<T, DP>();
  T* Qt = sizeof(T) == 2 ? Gs + TQ * row_pitch<T, DP>() : Qs;
  T* Gt = sizeof(T) == 2 ? Qt + DP * tr_pitch<TQ>() : Gs;
  TileRegs<T, DP, TQ, NT> qr, gr;
  ColScale scale;
  for (int gi = 0; gi < sh.g; ++gi) {
    const int head = hk * sh.g + gi;
    const T* qb = (const T*)a.q + (int64_t)b * sh.Nq * a.q_ld + (int64_t)head * sh.D;
    const T* gb = (const T*)a.dout + (int64_t)b * sh.Nq * a.dout_ld + (int64_t)head * sh.D;
    const int64_t stat = ((int64_t)b * sh.nh + head) * sh.Nq;
    float st_l = 0.0f, st_d = 0.0f;
    SlotTiles<NW> rows;
    SlotTiles<NW>::sync();                        // the list of the head before this one has been read
    rows.init(mq, 0, sh.Nq, list, list + kChunk + 64);
    int nq = rows.next(TQ);
    auto fetch = [&](int n) {
      qr.template load<VEC>(threadIdx.x, n, sh.D, [&](int i) { return qb + (int64_t)rows.slot(i) * a.q_ld; });
      gr.template load<VEC>(threadIdx.x, n, sh.D, [&](int i) { return gb + (int64_t)rows.slot(i) * a.dout_ld; });
      st_l = INFINITY;                            // rows past the end, and rows without a key: p = 0
      st_d = 0.0f;
      if (threadIdx.x < 32 && threadIdx.x < n) {
        const int s = rows.slot(threadIdx.x);
        const float v = a.lse[stat + s];
        if (v != -INFINITY) {
          st_l = v;
          st_d = a.delta[stat + s];
        }
      }
    };
    fetch(nq);
    while (nq > 0) {
      SlotTiles<NW>::sync();
      qr.store_rows(threadIdx.x, Qs);
      gr.store_rows(threadIdx.x, Gs);
      qr.store_tr(threadIdx.x, Qt);
      gr.store_tr(threadIdx.x, Gt);
      if (threadIdx.x < 32) {
        stats[threadIdx.x] = st_l;
        stats[32 + threadIdx.x] = st_d;
      }
      const int nn = rows.next(TQ);
      fetch(nn);
      SlotTiles<NW>::sync();
      f32x16 s = dot_rows<T, DP>(Qs, 0, kf, zero16());
      f32x16 dp = dot_rows<T, DP>(Gs, 0, vf, zero16());
#pragma unroll
      for (int g4 = 0; g4 < 4; ++g4) {
        const float4 ls = *reinterpret_cast<const float4*>(stats + 8 * g4 + 4 * h);
        const float4 dl = *reinterpret_cast<const float4*>(stats + 32 + 8 * g4 + 4 * h);
        const float lv[4] = {ls.x, ls.y, ls.z, ls.w}, dv4[4] = {dl.x, dl.y, dl.z, dl.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = 4 * g4 + i;
          s[r] = prob(s[r], a.scale, lv[i]);
          dp[r] = s[r] * (dp[r] - dv4[i]);
        }
      }
      if constexpr (__is_same(T, _Float16)) {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] *= kHalfP;
        scale.fit(dp, dk, DP / 32);
      }
      dot_cols<T, DP, TQ>(Gt, 0, s, dv);
      dot_cols<T, DP, TQ>(Qt, 0, dp, dk);
      nq = nn;
    }
  }
  if (key < 0) return;
  store_col<T, DP, VEC>((T*)a.dk + flat * a.dk_ld + (int64_t)hk * sh.D, dk,
                        __is_same(T, _Float16) ? a.scale / scale.sc : a.scale, sh.D);
  store_col<T, DP, VEC>((T*)a.dv + flat * a.dv_ld + (int64_t)hk * sh.D, dv,
                        __is_same(T, _Float16) ? 1.0f / kHalfP : 1.0f, sh.D);
}

// ---- host --------------------------------------------------------------------------------------------------------
static int waves_for(int64_t rows) { return rows > 64 ? 4 : rows > 32 ? 2 : 1; }

template <typename K>
static int launch(K kern, PerDeviceOnce& once, const BwdArgs& a, int threads, int bytes, hipStream_t st, const char* what) {
  if (bytes > 64 * 1024 &&
      !once.run([&] { return hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) == hipSuccess; })) {
    set_error("%s: the runtime refuses %d bytes of LDS", what, bytes);
    return MMB_ERR_LAUNCH;
  }
  kern<<<dim3((unsigned)a.map.blocks()), dim3(threads), bytes, st>>>(a);
  return check_launch(what);
}

template <typename T, int DP, int NW, bool VEC>
static int launch_dq(const BwdArgs& a, hipStream_t st) {
  static PerDeviceOnce once;
  constexpr int bytes = dq_lds<T, DP, 32>() + (kChunk + 64 + 4 + 32 * NW + 4) * 4;
  return launch(dq_kernel<T, DP, NW, VEC>, once, a, 64 * NW, bytes, st, "mmb_cross_attention_bwd (dq)");
}
template <typename T, int DP, int NW, bool VEC>
static int launch_dkv(const BwdArgs& a, hipStream_t st) {
  static PerDeviceOnce once;
  constexpr int bytes = dkv_lds<T, DP>() + (64 + kChunk + 64 + 4 + 32 * NW + 4) * 4;
  return launch(dkv_kernel<T, DP, NW, VEC>, once, a, 64 * NW, bytes, st, "mmb_cross_attention_bwd (dk, dv)");
}

template <typename T, int DP, bool VEC>
static int run_bwd(BwdArgs& a, hipStream_t st) {
  const int64_t R = (int64_t)a.sh.g * a.sh.Nq;
  const int nw_q = waves_for(R), nw_k = waves_for(a.sh.Nk);
  a.tiles = (int)((R + 32 * nw_q - 1) / (32 * nw_q));
  a.map = grid_map(a.sh.B, a.sh.nkv, a.tiles);
  MMB_REQUIRE(a.map.blocks() <= 0x7fffffffLL, "mmb_cross_attention_bwd: %lld workgroups", (long long)a.map.blocks());
  int rc = nw_q == 4 ? launch_dq<T, DP, 4, VEC>(a, st) : nw_q == 2 ? launch_dq<T, DP, 2, VEC>(a, st) : launch_dq<T, DP, 1, VEC>(a, st);
  if (rc != MMB_OK) return rc;
  a.tiles = (int)(((int64_t)a.sh.Nk + 32 * nw_k - 1) / (32 * nw_k));
  a.map = grid_map(a.sh.B, a.sh.nkv, a.tiles);
  MMB_REQUIRE(a.map.blocks() <= 0x7fffffffLL, "mmb_cross_attention_bwd: %lld workgroups", (long long)a.map.blocks());
  return nw_k == 4 ? launch_dkv<T, DP, 4, VEC>(a, st) : nw_k == 2 ? launch_dkv<T, DP, 2, VEC>(a, st) : launch_dkv<T, DP, 1, VEC>(a, st);
}
template <typename T, bool VEC>
static int pick_dp(BwdArgs& a, hipStream_t st) {
  switch (pad_width(a.sh.D)) {
    case 32: return run_bwd<T, 32, VEC>(a, st);
    case 64: return run_bwd<T, 64, VEC>(a, st);
    default: return run_bwd<T, 128, VEC>(a, st);
  }
}

}  // namespace xattn
}  // namespace mmb

using namespace mmb;
using namespace mmb::xattn;

extern "C" int mmb_cross_attention_bwd(int B, int Nq, int Nk, int nheads, int nheads_kv, int D, int dtype, const void* q,
                                       int64_t q_ld, const void* k, int64_t k_ld, const void* v, int64_t v_ld,
                                       const float* maskf_q, const float* maskf_k, float scale, const void* out, int64_t out_ld,
                                       const void* dout, int64_t dout_ld, const float* lse, void* dq, int64_t dq_ld, void* dk,
                                       int64_t dk_ld, void* dv, int64_t dv_ld, void* workspace, int64_t workspace_bytes,
                                       void* stream) {
  if (int rc = check_shape("mmb_cross_attention_bwd", B, Nq, Nk, nheads, nheads_kv, D, dtype, scale)) return rc;
  MMB_REQUIRE(q && k && v && out && dout && lse && dq && dk && dv,
              "mmb_cross_attention_bwd: q, k, v, out, dout, lse, dq, dk, dv must not be NULL");
  const int64_t wq = (int64_t)nheads * D, wk = (int64_t)nheads_kv * D;
  MMB_REQUIRE(q_ld >= wq && out_ld >= wq && dout_ld >= wq && dq_ld >= wq && k_ld >= wk && v_ld >= wk && dk_ld >= wk && dv_ld >= wk,
              "mmb_cross_attention_bwd: a leading dimension is smaller than its row");
  const int64_t need = (int64_t)B * nheads * Nq * 4;
  MMB_REQUIRE(workspace && workspace_bytes >= need, "mmb_cross_attention_bwd: workspace of %lld bytes needed, got %lld",
              (long long)need, (long long)(workspace ? workspace_bytes : 0));
  BwdArgs a = {{B, Nq, Nk, nheads, nheads_kv, D, nheads / nheads_kv}, q, k, v, out, dout, q_ld, k_ld, v_ld, out_ld, dout_ld,
               dq_ld, dk_ld, dv_ld, maskf_q, maskf_k, lse, scale, dq, dk, dv, (float*)workspace, 0, {}};
  const int es = dtype == MMB_DT_F32 ? 4 : 2;
  const bool vec = D * es % 16 == 0 && chunk_aligned(q, q_ld, es) && chunk_aligned(k, k_ld, es) && chunk_aligned(v, v_ld, es) &&
                   chunk_aligned(out, out_ld, es) && chunk_aligned(dout, dout_ld, es) && chunk_aligned(dq, dq_ld, es) &&
                   chunk_aligned(dk, dk_ld, es) && chunk_aligned(dv, dv_ld, es);
  hipStream_t st = as_stream(stream);
  if (dtype == MMB_DT_F32) return vec ? pick_dp<float, true>(a, st) : pick_dp<float, false>(a, st);
  if (dtype == MMB_DT_BF16) return vec ? pick_dp<__bf16, true>(a, st) : pick_dp<__bf16, false>(a, st);
  return vec ? pick_dp<_Float16, true>(a, st) : pick_dp<_Float16, false>(a, st);
}
