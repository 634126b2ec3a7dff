// Cross attention of the slots of one cloud to the slots of another, forward.
//
//   s_ij = scale q_i . k_j over the kept keys j;   p_i = softmax_j s_ij;   o_i = sum_j p_ij v_j;   lse_i = log sum_j e^s_ij
//
// One pass over the keys with a running maximum m and sum l: when a tile raises m, what was summed so far is scaled by
// exp(m_old - m_new).  Rows of query heads that share a key head are rows of one problem (row = query * g + head in group),
// so a single token with g heads reads its keys once.
//
// Two forms of one kernel body:
//   team    NW waves of one workgroup share every key tile through LDS, each owns 32 rows; many keys of few clouds go in two
//           ranges to two workgroups, whose results a second launch joins;
//   split   every wave walks its own range of keys with its own LDS tiles (no workgroup barrier while it runs); the
//           four partial sums of a workgroup are joined in LDS, those of several workgroups by a second launch.  For a
//           few rows against many keys, where the team form would leave most of the chip idle.
#include "cross_attention.h"
#include "regions.h"
#include <cmath>

namespace mmb {
namespace xattn {

struct FwdArgs {
  Shape sh;
  const void *q, *k, *v;
  int64_t q_ld, k_ld, v_ld, out_ld;
  const float *mq, *mk;
  float scale;
  void* out;
  float* lse;
  float* part;                                    // key splits: partial results of every 32 rows
  bool vec;
  int tiles, nsplit, chunk;                       // row tiles per (cloud, key head); key splits; keys of one (split form: of one wave)
  GridMap map;
};

// K and V tiles; the team form has two of each, so that one barrier a tile is enough
template <typename T, int DP, int TK, bool SPLIT>
constexpr int kv_lds() { return 2 * (SPLIT ? 1 : 2) * tile_bytes<T, DP, TK>(); }

// No instance may spill registers (the reverse says why): one wave a SIMD where the tiles in LDS admit no more anyway.
template <typename T, int DP, int NW, int TK, bool SPLIT, bool VEC>
__global__ void __launch_bounds__(64 * NW, DP == 128 && sizeof(T) == 4 && (NW < 4 || SPLIT) ? 1 : 2) fwd_kernel(FwdArgs a) {
  constexpr int NT = 64 * NW, TEAM = SPLIT ? 1 : NW, TT = 64 * TEAM, ROWS = SPLIT ? 32 : 32 * NW;
  constexpr int TILE = kv_lds<T, DP, TK, SPLIT>(), NTILE = SPLIT ? NW : 1;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  int* lists = reinterpret_cast<int*>(lds + TILE * NTILE);                  // key list(s), then the row list
  int* qlist = lists + NTILE * (kChunk + 64 + 4);
  const Shape sh = a.sh;
  int unit, item;
  if (!a.map.decode(blockIdx.x, unit, item)) return;
  const int per = a.tiles * a.nsplit;
  const int pair = a.map.units == sh.B ? unit * sh.nkv + item / per : unit;
  item %= per;
  const int b = pair / sh.nkv, hk = pair - b * sh.nkv, tile = item / a.nsplit, split = item - tile * a.nsplit;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, col = lane & 31, h = lane >> 5;
  const int team = SPLIT ? wave : 0, tid = SPLIT ? lane : threadIdx.x;
  const int R = sh.g * sh.Nq, r0 = tile * ROWS;
  const float* mq = a.mq ? a.mq + (int64_t)b * sh.Nq : nullptr;
  const float* mk = a.mk ? a.mk + (int64_t)b * sh.Nk : nullptr;

  RowTile rt = {r0 / sh.g, sh.g, qlist};
  if (mq) {
    if (threadIdx.x < 64) compact_select(mq, sh.Nq, rt.first_c, min(ROWS, R) / sh.g + 2, qlist);
    if (split == 0) {                             // slots of masked queries: zero rows, no log-sum
      const int rows = min(ROWS, R - r0);
      zero_masked_rows<NT, VEC>((T*)a.out + (int64_t)b * sh.Nq * a.out_ld + (int64_t)hk * sh.g * sh.D, a.out_ld, mq, r0, rows, sh.g, sh.D);
      for (int r = threadIdx.x; r < rows && a.lse; r += NT) {
        const int n = (r0 + r) / sh.g, gi = (r0 + r) - n * sh.g;
        if (mq[n] == 0.0f) a.lse[((int64_t)b * sh.nh + hk * sh.g + gi) * sh.Nq + n] = -INFINITY;
      }
    }
    __syncthreads();
    if (qlist[0] < 0) return;                        // no query left for this tile
  }
  const int row = r0 + (SPLIT ? 0 : wave * 32) + col;
  int n = -1, gi = 0;
  const bool live = row < R && rt.locate(row, sh.Nq, mq != nullptr, n, gi);
  const bool wave_live = __any(live);
  const int head = hk * sh.g + gi;

  u32x4 qf[DP / (2 * Traits<T>::EPC)];
  load_row<T, DP, VEC>(qf, (const T*)a.q + ((int64_t)b * sh.Nq + (live ? n : 0)) * a.q_ld + (int64_t)head * sh.D, sh.D, live);
  f32x16 acc[DP / 32];
#pragma unroll
  for (int t = 0; t < DP / 32; ++t) acc[t] = zero16();
  float m = -INFINITY, l = 0.0f;
  const float c = a.scale * kLog2e;

  int lo = 0, hi = sh.Nk;
  if (SPLIT || a.nsplit > 1) {
    lo = (int)min((int64_t)sh.Nk, (int64_t)(SPLIT ? split * NW + wave : split) * a.chunk);
    hi = (int)min((int64_t)sh.Nk, (int64_t)lo + a.chunk);
  }
  T* tiles = reinterpret_cast<T*>(lds + team * TILE);
  constexpr int TILE_E = TK * row_pitch<T, DP>();
  int* list = lists + team * (kChunk + 64 + 4);
  SlotTiles<TEAM> keys;
  keys.init(mk, lo, hi, list, list + kChunk + 64);
  const T* kb = (const T*)a.k + (int64_t)b * sh.Nk * a.k_ld + (int64_t)hk * sh.D;
  const T* vb = (const T*)a.v + (int64_t)b * sh.Nk * a.v_ld + (int64_t)hk * sh.D;
  TileRegs<T, DP, TK, TT> kr, vr;
  int nk = keys.next(TK);
  kr.template load<VEC>(tid, nk, sh.D, [&](int i) { return kb + (int64_t)keys.slot(i) * a.k_ld; });
  vr.template load<VEC>(tid, nk, sh.D, [&](int i) { return vb + (int64_t)keys.slot(i) * a.v_ld; });
  for (int buf = 0; nk > 0; buf ^= SPLIT ? 0 : 1) {
    if constexpr (SPLIT) wave_sync();             // one buffer: the tile before this one has been read (LDS is in order)
    T* Ks = tiles + buf * 2 * TILE_E;
    T* Vs = Ks + TILE_E;
    kr.store(tid, Ks);
    vr.store(tid, Vs);
    const int nn = keys.next(TK);
    SlotTiles<TEAM>::sync();                      // (team: whoever passes here has read the other buffer)
    // the next tile's rows come in while this one is worked on; issued behind the barrier, where finding their addresses
    // overlaps with this tile's products
    const int lt = SPLIT ? again(threadIdx.x) & 63 : VEC ? tid : again(threadIdx.x);
    kr.template load<VEC>(lt, nn, sh.D, [&](int i) { return kb + (int64_t)keys.slot(i) * a.k_ld; });
    vr.template load<VEC>(lt, nn, sh.D, [&](int i) { return vb + (int64_t)keys.slot(i) * a.v_ld; });
    if (wave_live) attend<T, DP, TK>(Ks, Vs, nk, qf, c, m, l, acc);         // (a wave without rows only helps to load)
    nk = nn;
  }
  l += __shfl_xor(l, 32);

  if constexpr (SPLIT) {                          // join the waves' partial sums: LDS, [wave][feature][row]
    __syncthreads();
    float* ml = reinterpret_cast<float*>(lds);                              // [wave][2][32]
    float* os = ml + NW * 64;
    if (h == 0) {
      ml[wave * 64 + col] = m;
      ml[wave * 64 + 32 + col] = l;
    }
#pragma unroll
    for (int t = 0; t < DP / 32; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) os[(wave * DP + 32 * t + crow(r, h)) * 33 + col] = acc[t][r];
    __syncthreads();
    // thread -> (row, features): rows of 32 threads each
    const int rr = threadIdx.x & 31;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, ml[w * 64 + rr]);
    const float Ms = M == -INFINITY ? 0.0f : M;
    float f[NW], L = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      f[w] = __builtin_amdgcn_exp2f((ml[w * 64 + rr] - Ms) * c);
      L += f[w] * ml[w * 64 + 32 + rr];
    }
    const int row2 = r0 + rr;
    int n2 = -1, g2 = 0;
    const bool live2 = row2 < R && rt.locate(row2, sh.Nq, mq != nullptr, n2, g2);
    const int head2 = hk * sh.g + g2;
    if (a.nsplit > 1) {
      float* p = a.part + ((int64_t)(pair * a.tiles + tile) * a.nsplit + split) * (32 * (DP + 2));
      if (threadIdx.x < 32) {
        p[rr] = M;
        p[32 + rr] = L;
      }
      for (int d = threadIdx.x >> 5; d < DP; d += NT / 32) {
        float o = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) o += f[w] * os[(w * DP + d) * 33 + rr];
        p[64 + d * 32 + rr] = o;
      }
      return;
    }
    if (!live2) return;
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;          // no key (or only scores of -inf): zeros
    T* o = (T*)a.out + ((int64_t)b * sh.Nq + n2) * a.out_ld + (int64_t)head2 * sh.D;
    for (int d = threadIdx.x >> 5; d < sh.D; d += NT / 32) {
      float s = 0.0f;
#pragma unroll
      for (int w = 0; w < NW; ++w) s += f[w] * os[(w * DP + d) * 33 + rr];
      o[d] = round_to<T>(s * inv);
    }
    if (a.lse && threadIdx.x < 32)
      a.lse[((int64_t)b * sh.nh + head2) * sh.Nq + n2] = row_lse<T>(M, L, a.scale);
  } else {
    if (a.nsplit > 1) {                           // this range's sums of the wave's 32 rows
      if (!wave_live) return;
      float* p = a.part + ((int64_t)((pair * a.tiles + tile) * NW + wave) * a.nsplit + split) * (32 * (DP + 2));
      if (h == 0) {
        p[col] = m;
        p[32 + col] = l;
      }
#pragma unroll
      for (int t = 0; t < DP / 32; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) p[64 + (32 * t + crow(r, h)) * 32 + col] = acc[t][r];
      return;
    }
    if (!live) return;
    const int t = again(threadIdx.x);             // (places found again, not kept in registers through the walk)
    int n_out = -1, gi_out = 0;
    rt.locate(again(r0) + (t >> 6) * 32 + (t & 31), sh.Nq, mq != nullptr, n_out, gi_out);
    const int head_out = hk * sh.g + gi_out;
    store_col<T, DP, VEC>((T*)a.out + ((int64_t)b * sh.Nq + n_out) * a.out_ld + (int64_t)head_out * sh.D, acc, l == 0.0f ? 0.0f : 1.0f / l, sh.D, t);
    if (a.lse && (t & 32) == 0) a.lse[((int64_t)b * sh.nh + head_out) * sh.Nq + n_out] = row_lse<T>(m, l, a.scale);
  }
}

// joins the key splits of 32 rows; workgroup = (pair, 32-row tile), a thread has an eighth of a row's features.  a.tiles: 32-row
// tiles.
template <typename T, int DP>
__global__ void __launch_bounds__(256) fwd_join_kernel(FwdArgs a) {
  __shared__ int qlist[34];
  const Shape sh = a.sh;
  const int pair = blockIdx.x / a.tiles, tile = blockIdx.x - pair * a.tiles, b = pair / sh.nkv, hk = pair - b * sh.nkv;
  const int r0 = tile * 32, R = sh.g * sh.Nq, rr = threadIdx.x & 31;
  const float* mq = a.mq ? a.mq + (int64_t)b * sh.Nq : nullptr;
  RowTile rt = {r0 / sh.g, sh.g, qlist};
  if (mq) {
    if (threadIdx.x < 64) compact_select(mq, sh.Nq, rt.first_c, min(32, R) / sh.g + 2, qlist);
    __syncthreads();
  }
  int n = -1, gi = 0;
  if (r0 + rr >= R || !rt.locate(r0 + rr, sh.Nq, mq != nullptr, n, gi)) return;
  const int head = hk * sh.g + gi;
  const float c = a.scale * kLog2e;
  const float* p = a.part + (int64_t)blockIdx.x * a.nsplit * (32 * (DP + 2));
  float M = -INFINITY;
  for (int s = 0; s < a.nsplit; ++s) M = fmaxf(M, p[(int64_t)s * 32 * (DP + 2) + rr]);
  const float Ms = M == -INFINITY ? 0.0f : M;
  const int d0 = (threadIdx.x >> 5) * (DP / 8);
  float L = 0.0f, o[DP / 8];
#pragma unroll
  for (int i = 0; i < DP / 8; ++i) o[i] = 0.0f;
  for (int s = 0; s < a.nsplit; ++s) {
    const float* ps = p + (int64_t)s * 32 * (DP + 2);
    const float f = __builtin_amdgcn_exp2f((ps[rr] - Ms) * c);
    L += f * ps[32 + rr];
#pragma unroll
    for (int i = 0; i < DP / 8; ++i) o[i] += f * ps[64 + (d0 + i) * 32 + rr];
  }
  const float inv = L == 0.0f ? 0.0f : 1.0f / L;
  T* op = (T*)a.out + ((int64_t)b * sh.Nq + n) * a.out_ld + (int64_t)head * sh.D;
  T v[DP / 8];
#pragma unroll
  for (int i = 0; i < DP / 8; ++i) v[i] = round_to<T>(o[i] * inv);
  if (a.vec) {                                    // (rows 16-byte aligned, D a multiple of a chunk)
    constexpr int W = 4;                          // four elements at a time: every DP / 8 is a multiple
#pragma unroll
    for (int i = 0; i < DP / 8; i += W)
      if (d0 + i < sh.D) __builtin_memcpy(__builtin_assume_aligned(op + d0 + i, W * sizeof(T)), v + i, W * sizeof(T));
  } else {
#pragma unroll
    for (int i = 0; i < DP / 8; ++i)
      if (d0 + i < sh.D) op[d0 + i] = v[i];
  }
  if (a.lse && threadIdx.x < 32)
    a.lse[((int64_t)b * sh.nh + head) * sh.Nq + n] = row_lse<T>(M, L, a.scale);
}

// ---- host --------------------------------------------------------------------------------------------------------
struct Plan {
  bool split;
  int nw, tiles, nsplit, chunk;
  int64_t part_bytes(const Shape& s) const {      // partial sums of every 32 rows and key range
    return nsplit > 1 ? (int64_t)s.B * s.nkv * tiles * (split ? 1 : nw) * nsplit * 32 * (pad_width(s.D) + 2) * 4 : 0;
  }
};
// Team form: 32 rows a wave, as many waves (1, 2, 4) as a cloud's rows fill, eight where that still leaves every CU two
// workgroups (they run one after the other, two waves a SIMD): the more waves share a tile, the less of it each has to load
// (4096 x 5000 slots, bf16: 364..388 us with eight, 424 with four; 2047 x 4099, where eight would leave CUs idle: 325 against
// 298).  Split form when the team form would put fewer than one workgroup on each of the 256 CUs, or one 32-row tile holds all
// rows, and there are keys to split.
static Plan fwd_plan(const Shape& s) {
  const int64_t R = (int64_t)s.g * s.Nq, pairs = (int64_t)s.B * s.nkv;
  Plan p;
  p.nw = R > 128 && pairs * ((R + 255) / 256) >= 512 ? 8 : R > 64 ? 4 : R > 32 ? 2 : 1;
  p.tiles = (int)((R + 32 * p.nw - 1) / (32 * p.nw));
  p.nsplit = 1;
  p.chunk = s.Nk;
  p.split = s.Nk > 128 && (pairs * p.tiles < 256 || R <= 32);
  if (p.split) {
    p.nw = 4;
    p.tiles = (int)((R + 31) / 32);
    // two workgroups on every CU, no wave with fewer than 128 keys (four tiles: below, joining costs more than it saves)
    const int64_t want = (512 + pairs * p.tiles - 1) / (pairs * p.tiles), most = (s.Nk + 511) / 512;
    p.nsplit = (int)(want < most ? want : most);
    if (p.nsplit < 1) p.nsplit = 1;
    p.chunk = (s.Nk + p.nsplit * 4 - 1) / (p.nsplit * 4);
    p.chunk = (p.chunk + 31) / 32 * 32;
  } else if (p.nw == 4 && s.Nk >= 2560 && pairs * p.tiles < 512) {
    // the team form alone leaves CUs with one workgroup, whose four waves do not hide each other's latencies: the keys in two
    // ranges and a second launch that joins them.  us with two ranges, with one, for 2047 slots, 16 heads on 8:
    //   fp16, D = 64     2560 keys 49, 55    4099 keys 69, 85    (masked 63, 73 and 54, 70)
    //   bf16, D = 128    2560 keys 71, 92    4099 keys 103, 144
    //   float, D = 32    2560 keys 114, 129  4099 keys 180, 206
    // Shorter lists gain less (fp16: 2048 keys 44, 46; 1800 keys 44, 45) and keep one range and one launch; two such clouds,
    // masked: the same within 3 %.
    p.nsplit = 2;
    p.chunk = ((s.Nk + 1) / 2 + 63) / 64 * 64;
  }
  return p;
}

template <typename T, int DP, int NW, int TK, bool SPLIT, bool VEC>
static int launch_fwd(const FwdArgs& a, hipStream_t st) {
  constexpr int NTILE = SPLIT ? NW : 1, tiles = kv_lds<T, DP, TK, SPLIT>() * NTILE, lists = NTILE * (kChunk + 64 + 4) * 4;
  constexpr int bytes = tiles + lists + (32 * NW + 4) * 4;
  static_assert(bytes <= 160 * 1024, "LDS");
  // the join buffers may not reach the row list behind tiles and key lists
  static_assert(!SPLIT || (NW * 64 + NW * DP * 33) * 4 <= tiles + lists, "join");
  auto kern = fwd_kernel<T, DP, NW, TK, SPLIT, VEC>;
  static PerDeviceOnce once;
  if (bytes > 64 * 1024 &&
      !once.run([&] { return hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) == hipSuccess; })) {
    set_error("mmb_cross_attention_fwd: the runtime refuses %d bytes of LDS", bytes);
    return MMB_ERR_LAUNCH;
  }
  kern<<<dim3((unsigned)a.map.blocks()), dim3(64 * NW), bytes, st>>>(a);
  int rc = check_launch("mmb_cross_attention_fwd");
  if (rc == MMB_OK && a.nsplit > 1) {
    FwdArgs j = a;
    j.tiles = a.tiles * (SPLIT ? 1 : NW);
    fwd_join_kernel<T, DP><<<dim3((unsigned)(j.sh.B * j.sh.nkv * j.tiles)), dim3(256), 0, st>>>(j);
    rc = check_launch("mmb_cross_attention_fwd (join)");
  }
  return rc;
}

template <typename T, int DP, bool VEC>
static int pick_nw(const Plan& p, const FwdArgs& a, hipStream_t st) {
  // keys per tile: 64 in 16 bits (two K and V tiles of a 128-wide head: 64 KB), 32 in float (68 KB)
  constexpr int TK = sizeof(T) == 2 ? 64 : 32;
  if (p.split) return launch_fwd<T, DP, 4, 32, true, VEC>(a, st);
  if (p.nw == 8) return launch_fwd<T, DP, 8, TK, false, VEC>(a, st);
  if (p.nw == 4) return launch_fwd<T, DP, 4, TK, false, VEC>(a, st);
  if (p.nw == 2) return launch_fwd<T, DP, 2, DP == 128 ? 32 : TK, false, VEC>(a, st);
  return launch_fwd<T, DP, 1, 32, false, VEC>(a, st);
}
template <typename T, bool VEC>
static int pick_dp(const Plan& p, const FwdArgs& a, hipStream_t st) {
  switch (pad_width(a.sh.D)) {
    case 32: return pick_nw<T, 32, VEC>(p, a, st);
    case 64: return pick_nw<T, 64, VEC>(p, a, st);
    default: return pick_nw<T, 128, VEC>(p, a, st);
  }
}

int check_shape(const char* who, int B, int Nq, int Nk, int nh, int nkv, int D, int dtype, float scale) {
  MMB_REQUIRE(B > 0 && Nq > 0 && Nk > 0, "%s: B, Nq, Nk must be positive (got %d, %d, %d)", who, B, Nq, Nk);
  MMB_REQUIRE(nkv > 0 && nh > 0 && nh % nkv == 0, "%s: nheads (%d) must be a positive multiple of nheads_kv (%d)", who, nh, nkv);
  MMB_REQUIRE(D > 0 && D <= 128, "%s: head width must be 1..128 (got %d)", who, D);
  MMB_REQUIRE(dtype == MMB_DT_F32 || dtype == MMB_DT_BF16 || dtype == MMB_DT_F16, "%s: unknown dtype %d", who, dtype);
  MMB_REQUIRE(scale > 0.0f && std::isfinite(scale), "%s: scale must be positive and finite", who);
  // 32-bit slot counters run a compaction step past the last slot, and the plan's divisions round up
  constexpr int most = 0x7fffffff - 4096;
  MMB_REQUIRE(Nk <= most, "%s: Nk must not exceed 2^31 - 4097 (got %d)", who, Nk);
  MMB_REQUIRE((int64_t)nh * Nq <= (1 << 30) && (int64_t)B * nh <= (1 << 30), "%s: nheads * Nq and B * nheads must stay below 2^30", who);
  return MMB_OK;
}

}  // namespace xattn
}  // namespace mmb

using namespace mmb;
using namespace mmb::xattn;

extern "C" int mmb_cross_attention_workspace(int B, int Nq, int Nk, int nheads, int nheads_kv, int D, int dtype, int backward,
                                             int64_t* bytes_host) {
  if (int rc = check_shape("mmb_cross_attention_workspace", B, Nq, Nk, nheads, nheads_kv, D, dtype, 1.0f)) return rc;
  MMB_REQUIRE(bytes_host != nullptr, "mmb_cross_attention_workspace: bytes_host is NULL");
  const Shape s = {B, Nq, Nk, nheads, nheads_kv, D, nheads / nheads_kv};
  if (backward) {
    *bytes_host = (int64_t)B * nheads * Nq * 4;
    return MMB_OK;
  }
  *bytes_host = resident_fits(s, dtype, false) || jets_fit(s, dtype, false) ? 0 : fwd_plan(s).part_bytes(s);
  return MMB_OK;
}

extern "C" int mmb_cross_attention_fwd(int B, int Nq, int Nk, int nheads, int nheads_kv, int D, int dtype, const void* q,
                                       int64_t q_ld, const void* k, int64_t k_ld, const void* v, int64_t v_ld,
                                       const float* maskf_q, const float* maskf_k, float scale, void* out, int64_t out_ld,
                                       float* lse, void* workspace, int64_t workspace_bytes, void* stream) {
  if (int rc = check_shape("mmb_cross_attention_fwd", B, Nq, Nk, nheads, nheads_kv, D, dtype, scale)) return rc;
  MMB_REQUIRE(q && k && v && out, "mmb_cross_attention_fwd: q, k, v, out must not be NULL");
  MMB_REQUIRE(q_ld >= (int64_t)nheads * D && out_ld >= (int64_t)nheads * D && k_ld >= (int64_t)nheads_kv * D &&
                  v_ld >= (int64_t)nheads_kv * D,
              "mmb_cross_attention_fwd: a leading dimension is smaller than its row");
  const Shape s = {B, Nq, Nk, nheads, nheads_kv, D, nheads / nheads_kv};
  const int es = dtype == MMB_DT_F32 ? 4 : 2;
  const bool vec = D * es % 16 == 0 && chunk_aligned(q, q_ld, es) && chunk_aligned(k, k_ld, es) && chunk_aligned(v, v_ld, es) &&
                   chunk_aligned(out, out_ld, es);
  const bool jets = jets_fit(s, dtype, false), resident = resident_fits(s, dtype, false);
  const Plan p = fwd_plan(s);
  const int64_t need = jets || resident ? 0 : p.part_bytes(s);
  MMB_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), "mmb_cross_attention_fwd: workspace of %lld bytes needed, got %lld",
              (long long)need, (long long)(workspace ? workspace_bytes : 0));
  const int64_t rq = (int64_t)B * Nq, rk = (int64_t)B * Nk, wq = (int64_t)nheads * D, wk = (int64_t)nheads_kv * D;
  const Region outs[] = {row_region(out, rq, wq, out_ld, es), flat_region(lse, rq * nheads * 4), flat_region(workspace, need)};
  const Region ins[] = {row_region(q, rq, wq, q_ld, es), row_region(k, rk, wk, k_ld, es), row_region(v, rk, wk, v_ld, es),
                        flat_region(maskf_q, rq * 4), flat_region(maskf_k, rk * 4)};
  if (int rc = check_apart("mmb_cross_attention_fwd", outs, 3, ins, 5)) return rc;
  if (jets)
    return jets_fwd(s, vec, (const float*)q, q_ld, (const float*)k, k_ld, (const float*)v, v_ld, maskf_q, maskf_k, scale, (float*)out, out_ld,
                    lse, as_stream(stream));
  if (resident)
    return resident_fwd(s, dtype, vec, q, q_ld, k, k_ld, v, v_ld, maskf_q, maskf_k, scale, out, out_ld, lse, as_stream(stream));
  FwdArgs a = {s, q, k, v, q_ld, k_ld, v_ld, out_ld, maskf_q, maskf_k, scale, out, lse, (float*)workspace, vec, p.tiles, p.nsplit, p.chunk,
               grid_map(B, nheads_kv, p.tiles * p.nsplit)};
  MMB_REQUIRE(grid_fits(a.map.blocks(), 64 * p.nw), "mmb_cross_attention_fwd: %lld workgroups are more than a launch takes", (long long)a.map.blocks());
  hipStream_t st = as_stream(stream);
  if (dtype == MMB_DT_F32) return vec ? pick_dp<float, true>(p, a, st) : pick_dp<float, false>(p, a, st);
  if (dtype == MMB_DT_BF16) return vec ? pick_dp<__bf16, true>(p, a, st) : pick_dp<__bf16, false>(p, a, st);
  return vec ? pick_dp<_Float16, true>(p, a, st) : pick_dp<_Float16, false>(p, a, st);
}
