// Cross attention of the slots of one cloud to the slots of another, reverse.
//
//   p_ij  = exp(s_ij - lse_i)                     recomputed from q, k and the forward's log-sum
//   dp_ij = do_i . v_j      delta_i = sum_j p_ij dp_ij = do_i . o_i      ds_ij = p_ij (dp_ij - delta_i)
//   dv_j  = sum_i p_ij do_i      dq_i = scale sum_j ds_ij k_j      dk_j = scale sum_i ds_ij q_i
//
// Two kinds of workgroups, each owning its outputs, so that every sum runs in a fixed order and nothing is accumulated with
// atomics: for dq a wave owns 32 query rows and walks the keys, for dk and dv a wave owns 32 keys and walks the queries of
// every head that shares them.  That recomputes s and dp once: 7 products instead of the 5 that one kind with atomically
// summed dq would need.  Both need delta: a short launch computes it and both kinds then run side by side in one launch (the
// waves of one kind alone are too few to cover each other's latencies); with so few keys that a row is in registers at once,
// the dq workgroups run first and take delta from p and dp themselves, free of the rounding of out.
#include "cross_attention.h"
#include "regions.h"

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
  bool few_keys;                                  // dq workgroups find delta themselves
  bool pack_heads;                                // dk, dv: rows of several query heads in one tile
  int tiles_q, tiles_k;
  GridMap map_q, map_k;
  unsigned n_dkv;                                 // workgroups of this launch that own keys
};


// keys of a dq tile, queries of a dk / dv tile: as many as leave two workgroups on a CU room for their registers
template <typename T, int DP> constexpr int dq_tile() { return sizeof(T) == 2 ? 64 : 32; }
template <typename T, int DP> constexpr int dkv_tile() { return sizeof(T) == 2 && DP <= 64 ? 64 : 32; }

constexpr int kListInts = kChunk + 64 + 4;
// The thread's number; as another value each time, so that what follows from it is found again, in the instances for which 256
// registers would otherwise not do (elsewhere keeping it is 3..5 % faster).
template <typename T, int DP, int NW>
__device__ __forceinline__ int thread_again() {
  return DP == 64 && (sizeof(T) == 2 || NW < 4) ? again(threadIdx.x) : (int)threadIdx.x;
}

template <typename T, int DP, int NW>
constexpr int bwd_lds() {
  constexpr int a = 4 * tile_bytes<T, DP, dq_tile<T, DP>()>(), b = 4 * tile_bytes<T, DP, dkv_tile<T, DP>()>() + 4 * dkv_tile<T, DP>() * 4;
  return (a > b ? a : b) + (kListInts + 32 * NW + 4) * 4;
}

template <typename T, int DP, int NW, bool VEC>
__device__ __forceinline__ void dq_body(const BwdArgs& a, int64_t id, char* lds) {
  constexpr int NT = 64 * NW, TK = dq_tile<T, DP>(), ROWS = 32 * NW, TILE_E = TK * row_pitch<T, DP>();
  int* list = reinterpret_cast<int*>(lds + 4 * tile_bytes<T, DP, TK>());
  int* qlist = list + kListInts;
  const Shape& sh = a.sh;
  int unit, item;
  if (!a.map_q.decode(id, unit, item)) return;
  const int pair = a.map_q.units == sh.B ? unit * sh.nkv + item / a.tiles_q : unit, tile = item % a.tiles_q;
  const int b = pair / sh.nkv, hk = pair - b * sh.nkv;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, col = lane & 31, h = lane >> 5;
  const int R = sh.g * sh.Nq, r0 = tile * ROWS;
  const float* mq = a.mq ? a.mq + (int64_t)b * sh.Nq : nullptr;
  const float* mk = a.mk ? a.mk + (int64_t)b * sh.Nk : nullptr;
  RowTile rt = {r0 / sh.g, sh.g, qlist};
  if (mq) {
    if (threadIdx.x < 64) compact_select(mq, sh.Nq, rt.first_c, min(ROWS, R) / sh.g + 2, qlist);
    zero_masked_rows<NT, VEC>((T*)a.dq + (int64_t)b * sh.Nq * a.dq_ld + (int64_t)hk * sh.g * sh.D, a.dq_ld, mq, r0, min(ROWS, R - r0), sh.g, sh.D);
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
  const float lse = live ? row_stat<T>(a.lse[stat]) : INFINITY;
  float delta = live && !a.few_keys ? a.delta[stat] : 0.0f;
  const float c = a.scale * kLog2e;
  f32x16 acc[DP / 32];
#pragma unroll
  for (int t = 0; t < DP / 32; ++t) acc[t] = zero16();

  T* tiles = reinterpret_cast<T*>(lds);
  SlotTiles<NW> keys;
  keys.init(mk, 0, sh.Nk, list, list + kChunk + 64);
  const T* kb = (const T*)a.k + (int64_t)b * sh.Nk * a.k_ld + (int64_t)hk * sh.D;
  const T* vb = (const T*)a.v + (int64_t)b * sh.Nk * a.v_ld + (int64_t)hk * sh.D;
  TileRegs<T, DP, TK, NT> kr, vr;
  int nk = keys.next(TK);
  kr.template load<VEC>(threadIdx.x, nk, sh.D, [&](int i) { return kb + (int64_t)keys.slot(i) * a.k_ld; });
  vr.template load<VEC>(threadIdx.x, nk, sh.D, [&](int i) { return vb + (int64_t)keys.slot(i) * a.v_ld; });
  const bool wave_live = __any(live);
  ColScale cs;
  float st = lse;
  if constexpr (__is_same(T, _Float16)) st -= log2_pow2(cs.sc);              // the scale rides on p
  for (int buf = 0; nk > 0; buf ^= 1) {
    T* Ks = tiles + buf * 2 * TILE_E;
    T* Vs = Ks + TILE_E;
    kr.store(threadIdx.x, Ks);
    vr.store(threadIdx.x, Vs);
    const int nn = keys.next(TK);
    SlotTiles<NW>::sync();
    const int lt = thread_again<T, DP, NW>();
    kr.template load<VEC>(lt, nn, sh.D, [&](int i) { return kb + (int64_t)keys.slot(i) * a.k_ld; });
    vr.template load<VEC>(lt, nn, sh.D, [&](int i) { return vb + (int64_t)keys.slot(i) * a.v_ld; });
    if (!wave_live) {                             // a wave without rows only helps to load
      nk = nn;
      continue;
    }
    if (a.few_keys) {                             // at most 32 keys, all of them here: p normalised by its own sum
      f32x16 s = dot_rows<T, DP>(Ks, 0, qf, zero16());
      const f32x16 dp = dot_rows<T, DP>(Vs, 0, gf, zero16());
      float sum = 0.0f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[r] = crow(r, h) < nk ? prob<T>(s[r], a.scale, c, lse) : 0.0f;
        sum += s[r];
      }
      sum += __shfl_xor(sum, 32);
#pragma unroll
      for (int r = 0; r < 16; ++r) delta = fmaf(sum == 0.0f ? 0.0f : s[r] / sum, dp[r], delta);
      delta += __shfl_xor(delta, 32);
    }
    // all score tiles, then all second products: the matrix work of one tile beside the element work of another
    constexpr int SUBS = TK / 32;
    f32x16 s[SUBS];
#pragma unroll
    for (int u = 0; u < SUBS; ++u) {
      s[u] = dot_rows<T, DP>(Ks, 32 * u, qf, zero16());
      const f32x16 dp = dot_rows<T, DP>(Vs, 32 * u, gf, zero16());
#pragma unroll
      for (int r = 0; r < 16; ++r) s[u][r] = prob<T>(s[u][r], a.scale, c, st) * (dp[r] - delta);
    }
    if (nk < TK) {
      rarely();
#pragma unroll
      for (int u = 0; u < SUBS; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (32 * u + crow(r, h) >= nk) s[u][r] = 0.0f;
    }
    if constexpr (__is_same(T, _Float16)) {
      if (cs.fit<SUBS>(s, acc, DP / 32)) st = lse - log2_pow2(cs.sc);
    }
    // ds is rounded to the inputs' type for the product, like p in the forward; the sum over keys stays in 32 bits
#pragma unroll
    for (int u = 0; u < SUBS; ++u) dot_cols<T, DP>(Ks, 32 * u, s[u], acc);
    nk = nn;
  }
  if (!live) return;
  const int tid = thread_again<T, DP, NW>();              // (places found again, not kept in registers through the walk)
  int n_out = -1, gi_out = 0;
  rt.locate(again(r0) + (tid >> 6) * 32 + (tid & 31), sh.Nq, mq != nullptr, n_out, gi_out);
  const int head_out = hk * sh.g + gi_out;
  if (a.few_keys && (tid & 32) == 0) a.delta[((int64_t)b * sh.nh + head_out) * sh.Nq + n_out] = delta;
  store_col<T, DP, VEC>((T*)a.dq + ((int64_t)b * sh.Nq + n_out) * a.dq_ld + (int64_t)head_out * sh.D, acc,
                        __is_same(T, _Float16) ? a.scale / cs.sc : a.scale, sh.D, tid);
}

template <typename T, int DP, int NW, bool VEC>
__device__ __forceinline__ void dkv_body(const BwdArgs& a, int64_t id, char* lds) {
  constexpr int NT = 64 * NW, TQ = dkv_tile<T, DP>(), COLS = 32 * NW, TILE_E = TQ * row_pitch<T, DP>();
  float* stats = reinterpret_cast<float*>(lds + 4 * tile_bytes<T, DP, TQ>());          // two of lse[TQ], delta[TQ]
  int* list = reinterpret_cast<int*>(stats + 4 * TQ);
  int* klist = list + kListInts;
  const Shape& sh = a.sh;
  int unit, item;
  if (!a.map_k.decode(id, unit, item)) return;
  const int pair = a.map_k.units == sh.B ? unit * sh.nkv + item / a.tiles_k : unit, tile = item % a.tiles_k;
  const int b = pair / sh.nkv, hk = pair - b * sh.nkv;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, col = lane & 31, h = lane >> 5;
  const int k0 = tile * COLS;
  const float* mq = a.mq ? a.mq + (int64_t)b * sh.Nq : nullptr;
  const float* mk = a.mk ? a.mk + (int64_t)b * sh.Nk : nullptr;
  if (mk) {
    if (threadIdx.x < 64) compact_select(mk, sh.Nk, k0, COLS, klist);
    const int rows = min(COLS, sh.Nk - k0);
    zero_masked_rows<NT, VEC>((T*)a.dk + (int64_t)b * sh.Nk * a.dk_ld + (int64_t)hk * sh.D, a.dk_ld, mk, k0, rows, 1, sh.D);
    zero_masked_rows<NT, VEC>((T*)a.dv + (int64_t)b * sh.Nk * a.dv_ld + (int64_t)hk * sh.D, a.dv_ld, mk, k0, rows, 1, sh.D);
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
  const float c = a.scale * kLog2e;
  const bool wave_live = __any(key >= 0);
  T* tiles = reinterpret_cast<T*>(lds);
  TileRegs<T, DP, TQ, NT> qr, gr;
  ColScale cs;
  int buf = 0;
  // rows of a tile: (slot, head) with gh heads beside each other -- 1 where the slots of one head fill a tile, else as many of
  // the heads that share this key head as a tile holds
  const int gh = a.pack_heads ? min(sh.g, TQ) : 1, per_tile = TQ / gh;
  for (int gi = 0; gi < sh.g; gi += gh) {
    const int head0 = hk * sh.g + gi, nh = min(gh, sh.g - gi);
    const T* qb = (const T*)a.q + (int64_t)b * sh.Nq * a.q_ld + (int64_t)head0 * sh.D;
    const T* gb = (const T*)a.dout + (int64_t)b * sh.Nq * a.dout_ld + (int64_t)head0 * sh.D;
    const int64_t stat = ((int64_t)b * sh.nh + head0) * sh.Nq;
    float st_l = 0.0f, st_d = 0.0f;
    SlotTiles<NW> rows;
    rows.init(mq, 0, sh.Nq, list, list + kChunk + 64);
    int nq = rows.next(per_tile) * nh;            // rows, not slots
    auto fetch = [&](int n) {
      auto at = [&](int i, const T* base, int64_t ld) {
        if (nh == 1) return base + (int64_t)rows.slot(i) * ld;
        const int s = i / nh;
        return base + (int64_t)rows.slot(s) * ld + (i - s * nh) * sh.D;
      };
      const int lt = thread_again<T, DP, NW>();
      qr.template load<VEC>(lt, n, sh.D, [&](int i) { return at(i, qb, a.q_ld); });
      gr.template load<VEC>(lt, n, sh.D, [&](int i) { return at(i, gb, a.dout_ld); });
      st_l = -INFINITY;
      if (threadIdx.x < TQ && threadIdx.x < n) {  // (both loads at once; looked at when the tile is stored)
        const int s = (int)threadIdx.x / nh;
        const int64_t o = stat + (int64_t)(threadIdx.x - s * nh) * sh.Nq + rows.slot(s);
        st_l = a.lse[o];
        st_d = a.delta[o];
      }
    };
    fetch(nq);
    for (; nq > 0; buf ^= 1) {
      T* Qs = tiles + buf * 2 * TILE_E;
      T* Gs = Qs + TILE_E;
      float* sl = stats + buf * 2 * TQ;
      const int ts = thread_again<T, DP, NW>();
      qr.store(ts, Qs);
      gr.store(ts, Gs);
      if (threadIdx.x < TQ) {
        const float x = row_stat<T>(st_l);        // rows past the end, and rows without a key: p = 0
        sl[threadIdx.x] = __is_same(T, _Float16) ? x - kHalfLog : x;
        sl[TQ + threadIdx.x] = x < INFINITY ? st_d : 0.0f;
      }
      const int nn = rows.next(per_tile) * nh;
      SlotTiles<NW>::sync();
      fetch(nn);
      if (!wave_live) {                           // a wave without keys only helps to load
        nq = nn;
        continue;
      }
      constexpr int SUBS = TQ / 32;
      f32x16 s[SUBS], dp[SUBS];
#pragma unroll
      for (int u = 0; u < SUBS; ++u) {
        s[u] = dot_rows<T, DP>(Qs, 32 * u, kf, zero16());
        dp[u] = dot_rows<T, DP>(Gs, 32 * u, vf, zero16());
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4) {
          const f32x4 ls = *reinterpret_cast<const f32x4*>(sl + 32 * u + 8 * g4 + 4 * h);
          const f32x4 dl = *reinterpret_cast<const f32x4*>(sl + TQ + 32 * u + 8 * g4 + 4 * h);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = 4 * g4 + i;
            s[u][r] = prob<T>(s[u][r], a.scale, c, ls[i]);
            dp[u][r] = s[u][r] * (dp[u][r] - dl[i]);
            if constexpr (__is_same(T, _Float16)) dp[u][r] *= cs.sc;
          }
        }
      }
      if constexpr (__is_same(T, _Float16)) cs.fit<SUBS>(dp, dk, DP / 32);
#pragma unroll
      for (int u = 0; u < SUBS; ++u) {
        dot_cols<T, DP>(Gs, 32 * u, s[u], dv);
        dot_cols<T, DP>(Qs, 32 * u, dp[u], dk);
      }
      nq = nn;
    }
  }
  const int tid = thread_again<T, DP, NW>(), place = (tid >> 6) * 32 + (tid & 31), kc_out = again(k0) + place;
  const int key_out = mk ? klist[place] : (kc_out < sh.Nk ? kc_out : -1);
  if (key_out < 0) return;
  const int64_t out = (int64_t)b * sh.Nk + key_out;
  // (dp carried p's 2^12 too)
  store_col<T, DP, VEC>((T*)a.dk + out * a.dk_ld + (int64_t)hk * sh.D, dk,
                        __is_same(T, _Float16) ? a.scale / kHalfP / cs.sc : a.scale, sh.D, tid);
  store_col<T, DP, VEC>((T*)a.dv + out * a.dv_ld + (int64_t)hk * sh.D, dv,
                        __is_same(T, _Float16) ? 1.0f / kHalfP : 1.0f, sh.D, tid);
}

// Waves a SIMD that an instance leaves registers for.  None may spill: the compiler stored a spilled register under a narrowed
// exec mask and read it back for all lanes (bfloat16 heads of 33 .. 63 off the chunk of eight on two waves: delta went to
// whatever address scratch memory held).  So two only where 256 registers are enough; again() keeps what is cheap to find out of
// them.
template <typename T, int DP, int NW, bool VEC>
constexpr int bwd_waves() {
  if (DP == 128) return 1;
  if (DP == 64 && (NW == 1 || (NW == 2 && sizeof(T) == 2 && !VEC))) return 1;
  return 2;
}

// workgroups [0, n_dkv) own keys, the others query rows
template <typename T, int DP, int NW, bool VEC>
__global__ void __launch_bounds__(64 * NW, (bwd_waves<T, DP, NW, VEC>())) bwd_kernel(BwdArgs a) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  if (blockIdx.x < a.n_dkv) dkv_body<T, DP, NW, VEC>(a, blockIdx.x, lds);
  else dq_body<T, DP, NW, VEC>(a, blockIdx.x - a.n_dkv, lds);
}

// delta of every (row, head) of a kept slot: LP lanes a head, its chunks dealt to them
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) delta_kernel(BwdArgs a, int lp) {
  constexpr int E = Traits<T>::EPC;
  const Shape sh = a.sh;
  const int64_t items = (int64_t)sh.B * sh.Nq * sh.nh, per = 256 / lp;
  const int sub = threadIdx.x % lp;
  for (int64_t it = (int64_t)blockIdx.x * per + threadIdx.x / lp; it < items; it += (int64_t)gridDim.x * per) {
    const int64_t row = it / sh.nh;
    if (a.mq && a.mq[row] == 0.0f) continue;      // (a masked slot's rows are not read; all lanes of the head leave)
    const int head = (int)(it - row * sh.nh);
    const T* o = (const T*)a.out + row * a.out_ld + (int64_t)head * sh.D;
    const T* g = (const T*)a.dout + row * a.dout_ld + (int64_t)head * sh.D;
    float s = 0.0f;
    for (int ch = sub; ch * E < sh.D; ch += lp) {
      T x[E], y[E];
      const u32x4 u = load_chunk<T, VEC>(o, ch * E, sh.D, true), v = load_chunk<T, VEC>(g, ch * E, sh.D, true);
      __builtin_memcpy(x, &u, 16);
      __builtin_memcpy(y, &v, 16);
#pragma unroll
      for (int i = 0; i < E; ++i) s = fmaf((float)x[i], (float)y[i], s);
    }
    for (int o2 = lp >> 1; o2 > 0; o2 >>= 1) s += __shfl_xor(s, o2, 64);
    if (sub == 0) {
      const int64_t bb = row / sh.Nq;
      a.delta[(bb * sh.nh + head) * sh.Nq + (row - bb * sh.Nq)] = s;
    }
  }
}

// ---- host --------------------------------------------------------------------------------------------------------
template <typename T, int DP, int NW, bool VEC>
static int run_bwd(BwdArgs& a, hipStream_t st) {
  constexpr int bytes = bwd_lds<T, DP, NW>();
  static_assert(bytes <= 160 * 1024, "LDS");
  const Shape& s = a.sh;
  a.tiles_q = (int)(((int64_t)s.g * s.Nq + 32 * NW - 1) / (32 * NW));
  a.tiles_k = (int)(((int64_t)s.Nk + 32 * NW - 1) / (32 * NW));
  a.map_q = grid_map(s.B, s.nkv, a.tiles_q);
  a.map_k = grid_map(s.B, s.nkv, a.tiles_k);
  const int64_t nq = a.map_q.blocks(), nk = a.map_k.blocks();
  MMB_REQUIRE(grid_fits(nq + nk, 64 * NW), "mmb_cross_attention_bwd: %lld workgroups are more than a launch takes", (long long)(nq + nk));
  auto kern = bwd_kernel<T, DP, NW, VEC>;
  static PerDeviceOnce once;
  if (bytes > 64 * 1024 &&
      !once.run([&] { return hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) == hipSuccess; })) {
    set_error("mmb_cross_attention_bwd: the runtime refuses %d bytes of LDS", bytes);
    return MMB_ERR_LAUNCH;
  }
  a.few_keys = s.Nk <= 32;
  // (818 clouds of 2 x 1306 slots, 15 heads on 3: 903 -> 557 us a training step)
  a.pack_heads = s.g > 1 && s.Nq < dkv_tile<T, DP>();
  if (a.few_keys) {
    a.n_dkv = 0;
    kern<<<dim3((unsigned)nq), dim3(64 * NW), bytes, st>>>(a);
    if (int rc = check_launch("mmb_cross_attention_bwd (dq)")) return rc;
    a.n_dkv = (unsigned)nk;
    kern<<<dim3((unsigned)nk), dim3(64 * NW), bytes, st>>>(a);
    return check_launch("mmb_cross_attention_bwd (dk, dv)");
  }
  constexpr int E = Traits<T>::EPC;
  int lp = 1;
  while (lp * E < s.D && lp < 16) lp *= 2;
  delta_kernel<T, VEC><<<stream_grid((int64_t)s.B * s.Nq * s.nh * lp, 256), 256, 0, st>>>(a, lp);
  if (int rc = check_launch("mmb_cross_attention_bwd (delta)")) return rc;
  a.n_dkv = (unsigned)nk;
  kern<<<dim3((unsigned)(nq + nk)), dim3(64 * NW), bytes, st>>>(a);
  return check_launch("mmb_cross_attention_bwd");
}
// waves of a workgroup (32 rows or keys each): as many as the longer side fills; where the shorter side leaves waves without
// rows of their own they still share the loading
template <typename T, int DP, bool VEC>
static int pick_nw(BwdArgs& a, hipStream_t st) {
  const int64_t R = (int64_t)a.sh.g * a.sh.Nq, m = R > a.sh.Nk ? R : a.sh.Nk;
  if (m > 64) return run_bwd<T, DP, 4, VEC>(a, st);
  // (one wave alone would need more than 512 registers for tiles of 128-wide heads)
  if constexpr (DP < 128)
    if (m <= 32) return run_bwd<T, DP, 1, VEC>(a, st);
  return run_bwd<T, DP, 2, VEC>(a, st);
}
template <typename T, bool VEC>
static int pick_dp(BwdArgs& a, hipStream_t st) {
  switch (pad_width(a.sh.D)) {
    case 32: return pick_nw<T, 32, VEC>(a, st);
    case 64: return pick_nw<T, 64, VEC>(a, st);
    default: return pick_nw<T, 128, VEC>(a, st);
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
  const int es = dtype == MMB_DT_F32 ? 4 : 2;
  const int64_t rq = (int64_t)B * Nq, rk = (int64_t)B * Nk;
  const Region outs[] = {row_region(dq, rq, wq, dq_ld, es), row_region(dk, rk, wk, dk_ld, es), row_region(dv, rk, wk, dv_ld, es),
                         flat_region(workspace, need)};
  const Region ins[] = {row_region(q, rq, wq, q_ld, es), row_region(k, rk, wk, k_ld, es), row_region(v, rk, wk, v_ld, es),
                        row_region(out, rq, wq, out_ld, es), row_region(dout, rq, wq, dout_ld, es), flat_region(lse, need),
                        flat_region(maskf_q, rq * 4), flat_region(maskf_k, rk * 4)};
  if (int rc = check_apart("mmb_cross_attention_bwd", outs, 4, ins, 8)) return rc;
  BwdArgs a = {{B, Nq, Nk, nheads, nheads_kv, D, nheads / nheads_kv}, q, k, v, out, dout, q_ld, k_ld, v_ld, out_ld, dout_ld,
               dq_ld, dk_ld, dv_ld, maskf_q, maskf_k, lse, scale, dq, dk, dv, (float*)workspace, false, false, 0, 0, {}, {}, 0};
  const bool vec = D * es % 16 == 0 && chunk_aligned(q, q_ld, es) && chunk_aligned(k, k_ld, es) && chunk_aligned(v, v_ld, es) &&
                   chunk_aligned(out, out_ld, es) && chunk_aligned(dout, dout_ld, es) && chunk_aligned(dq, dq_ld, es) &&
                   chunk_aligned(dk, dk_ld, es) && chunk_aligned(dv, dv_ld, es);
  hipStream_t st = as_stream(stream);
  if (jets_fit(a.sh, dtype, true))
    return jets_bwd(a.sh, vec, (const float*)q, q_ld, (const float*)k, k_ld, (const float*)v, v_ld, maskf_q, maskf_k, scale, (const float*)out,
                    out_ld, (const float*)dout, dout_ld, lse, (float*)dq, dq_ld, (float*)dk, dk_ld, (float*)dv, dv_ld, st);
  if (resident_fits(a.sh, dtype, true))
    return resident_bwd(a.sh, dtype, vec, q, q_ld, k, k_ld, v, v_ld, maskf_q, maskf_k, scale, out, out_ld, dout, dout_ld, lse, dq,
                        dq_ld, dk, dk_ld, dv, dv_ld, st);
  if (dtype == MMB_DT_F32) return vec ? pick_dp<float, true>(a, st) : pick_dp<float, false>(a, st);
  if (dtype == MMB_DT_BF16) return vec ? pick_dp<__bf16, true>(a, st) : pick_dp<__bf16, false>(a, st);
  return vec ? pick_dp<_Float16, true>(a, st) : pick_dp<_Float16, false>(a, st);
}
