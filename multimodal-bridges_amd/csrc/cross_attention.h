// Shared parts of the cross-attention kernels (cross_attention.hip: forward, cross_attention_bwd.hip: reverse).
//
// Both passes are built from 32x32 matrix-core tiles in which a lane owns one COLUMN of the score matrix:
//   forward / dq :  S^T (keys x queries)  = K Q^T      a lane holds 16 keys of one query per tile
//   dk, dv       :  S   (queries x keys)  = Q K^T      a lane holds 16 queries of one key per tile
// so softmax statistics are per-lane scalars, and the accumulator registers of S (or P, dS) ARE the B operand of the
// next product: 32x32x16 wants, for one column, eight contraction indices per lane half, the accumulator holds
// {4h..4h+3, 8+4h..8+4h+3} of every 16 -- a permutation of the contraction index, which the A operand is read with.  No
// cross-lane traffic, no LDS round trip for P.  The A operand of that product is the transpose of a tile that lies row by
// row in LDS; in 16 bits the transposing LDS read supplies it, so a tile is stored once and serves both products.
#pragma once
#include "common.h"

namespace mmb {
namespace xattn {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;

// row of accumulator register r in a 32x32 tile, for lane half h
__device__ __forceinline__ int crow(int r, int h) { return (r >> 2) * 8 + h * 4 + (r & 3); }

template <typename T> struct Traits;
template <> struct Traits<float> { static constexpr int EPC = 4; };       // elements of one 16-byte chunk
template <> struct Traits<__bf16> { static constexpr int EPC = 8; };
template <> struct Traits<_Float16> { static constexpr int EPC = 8; };

// 8 (16-bit types) or 4 (float) elements, one 16-byte chunk
template <typename T, bool VEC>
__device__ __forceinline__ u32x4 load_chunk(const T* __restrict__ p, int d, int D, bool ok) {
  constexpr int E = Traits<T>::EPC;
  u32x4 r = {0u, 0u, 0u, 0u};
  if constexpr (VEC) {
    if (ok && d < D) r = *reinterpret_cast<const u32x4*>(p + d);
  } else {
    if (ok) {
      T t[E];
#pragma unroll
      for (int i = 0; i < E; ++i) t[i] = d + i < D ? p[d + i] : (T)0.0f;
      __builtin_memcpy(&r, t, 16);
    }
  }
  return r;
}

template <typename T>
__device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (sizeof(T) == 2) {
    if constexpr (__is_same(T, __bf16))
      return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
      return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  } else {
    // four steps of two: lane half h supplies contraction indices 4h .. 4h+3 of the eight that the chunk pair covers
    const f32x4 af = __builtin_bit_cast(f32x4, a), bf = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(af[i], bf[i], c, 0, 0, 0);
    return c;
  }
}

// eight accumulator values, rounded to T (nearest even): one B operand of the next product
template <typename T>
__device__ __forceinline__ u32x4 pack8(const f32x16& s, int r0) {
  T t[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) t[i] = (T)s[r0 + i];
  u32x4 r;
  __builtin_memcpy(&r, t, 16);
  return r;
}

__device__ __forceinline__ f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.0f;
  return z;
}

// LDS hand-over inside one wave (in order in hardware; the fence keeps the compiler from moving accesses across)
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// First statement of a branch that is rarely taken: keeps the compiler from executing the branch's arithmetic always and
// selecting afterwards (it does so for the tail of the keys and for rescaling, at three instructions an element).
__device__ __forceinline__ void rarely() { asm volatile(""); }

// a value that the compiler takes for another one: what is computed from it is computed again, not kept
__device__ __forceinline__ int again(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

constexpr int kChunk = 512;                       // raw slots one compaction step looks at

// Appends the slots n in [lo, min(lo + kChunk, hi)) with maskf[n] != 0 to list[], in order; returns how many.
// One wave; all eight loads are in flight together.
__device__ __forceinline__ int compact_chunk(const float* __restrict__ maskf, int lo, int hi, int* list) {
  const int lane = threadIdx.x & 63;
  float f[kChunk / 64];
#pragma unroll
  for (int c = 0; c < kChunk / 64; ++c) {
    const int n = lo + c * 64 + lane;
    f[c] = n < hi ? maskf[n] : 0.0f;
  }
  int at = 0;
#pragma unroll
  for (int c = 0; c < kChunk / 64; ++c) {
    const bool ok = f[c] != 0.0f;
    const unsigned long long bal = __ballot(ok);
    if (ok) list[at + __popcll(bal & ((1ull << lane) - 1ull))] = lo + c * 64 + lane;
    at += __popcll(bal);
  }
  return at;
}

// list[i] = slot of the (first + i)-th kept slot of maskf[0, N), for i < n; -1 where there is none.  One wave.
__device__ __forceinline__ void compact_select(const float* __restrict__ maskf, int N, int first, int n, int* list) {
  const int lane = threadIdx.x & 63;
  for (int i = lane; i < n; i += 64) list[i] = -1;
  wave_sync();
  int at = 0;
  for (int lo = 0; lo < N && at < first + n; lo += kChunk) {
    float f[kChunk / 64];
#pragma unroll
    for (int c = 0; c < kChunk / 64; ++c) {
      const int s = lo + c * 64 + lane;
      f[c] = s < N ? maskf[s] : 0.0f;
    }
#pragma unroll
    for (int c = 0; c < kChunk / 64; ++c) {
      const bool ok = f[c] != 0.0f;
      const unsigned long long bal = __ballot(ok);
      const int o = at + __popcll(bal & ((1ull << lane) - 1ull)) - first;
      if (ok && o >= 0 && o < n) list[o] = lo + c * 64 + lane;
      at += __popcll(bal);
    }
  }
}

// The kept slots of [lo, hi), handed out in tiles.  list: LDS, kChunk + 64 ints, shared by the TEAM waves that walk
// together (TEAM == 1: one wave on its own).  Without a mask nothing is listed: slot(i) is lo + i.
template <int TEAM>
struct SlotTiles {
  const float* maskf;
  int raw, hi, head, cnt;
  int* list;
  int* cnt_sh;
  __device__ __forceinline__ void init(const float* m, int lo, int hi_, int* l, int* c) {
    maskf = m; raw = lo; hi = hi_; head = cnt = 0; list = l; cnt_sh = c;
  }
  static __device__ __forceinline__ void sync() {
    if constexpr (TEAM == 1) wave_sync();
    else __syncthreads();
  }
  // number of slots of the next tile (0: done); slot(i), i < number, stays valid until the next call
  __device__ __forceinline__ int next(int tile) {
    if (maskf == nullptr) {
      head = raw;
      const int n = min(tile, hi - raw);
      raw += max(n, 0);
      return max(n, 0);
    }
    head += cur;
    cur = 0;
    while (cnt - head < tile && raw < hi) {
      sync();                                     // everyone is done with the list
      if (TEAM == 1 || threadIdx.x < 64) {
        const int lane = threadIdx.x & 63, left = cnt - head;      // left < tile <= 64: one slot a lane
        const int keep = lane < left ? list[head + lane] : 0;
        wave_sync();
        if (lane < left) list[lane] = keep;
        wave_sync();
        const int c = left + compact_chunk(maskf, raw, hi, list + left);
        if (TEAM > 1 && lane == 0) *cnt_sh = c;
        if (TEAM == 1) cnt = c;
      }
      sync();
      if constexpr (TEAM > 1) cnt = *cnt_sh;
      head = 0;
      raw += kChunk;
    }
    cur = min(tile, cnt - head);
    return cur;
  }
  __device__ __forceinline__ int slot(int i) const { return maskf == nullptr ? head + i : list[head + i]; }
  int cur = 0;
};

// ---- one tile of rows in LDS -------------------------------------------------------------------------------------
// float:  row-major, pitch DP + 4 (b128 reads of 32 rows at one chunk column spread over all banks).
// 16-bit: row-major without padding, the 16-byte chunks of a row permuted by an exclusive-or with a function of the row
//         that serves both kinds of read: 16 rows at one chunk column (the scores) and four rows of 16 columns (the
//         transposing read of the second product) each fall on 64 different banks.
template <int DP> constexpr int feature_tiles() { return DP / 32; }      // 32-row accumulators of DP features
template <typename T, int DP> constexpr int row_pitch() { return sizeof(T) == 2 ? DP : DP + 4; }
template <int DP>
__device__ __forceinline__ int swizzle(int row) {
  return DP == 128 ? ((row & 3) << 2 | ((row >> 2) & 3)) : DP == 64 ? (((row >> 1) & 1) << 2 | ((row >> 2) & 3)) : (row >> 2) & 3;
}
template <typename T, int DP>
__device__ __forceinline__ int chunk_at(int row, int ch) {                  // element offset of chunk ch of a row
  constexpr int E = Traits<T>::EPC;
  if constexpr (sizeof(T) == 2) return row * DP + ((ch ^ swizzle<DP>(row)) * E);
  else return row * row_pitch<T, DP>() + ch * E;
}
template <typename T, int DP, int ROWS>
constexpr int tile_bytes() { return ROWS * row_pitch<T, DP>() * (int)sizeof(T); }

// Registers of one thread's share of a ROWS x DP tile: 16-byte chunks, the chunks of a row beside each other.
template <typename T, int DP, int ROWS, int NT>
struct TileRegs {
  static constexpr int E = Traits<T>::EPC, CH = DP / E, ITEMS = ROWS * CH, PER = (ITEMS + NT - 1) / NT;
  u32x4 r[PER];
  template <bool VEC, typename RowOf>
  __device__ __forceinline__ void load(int tid, int n, int D, RowOf row_of) {
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      const int it = p * NT + tid, row = it / CH;
      const bool ok = row < n && (ITEMS % NT == 0 || it < ITEMS);
      r[p] = load_chunk<T, VEC>(ok ? row_of(row) : nullptr, (it % CH) * E, D, ok);
    }
  }
  __device__ __forceinline__ void store(int tid, T* dst) const {
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      const int it = p * NT + tid;
      if (ITEMS % NT != 0 && it >= ITEMS) break;
      *reinterpret_cast<u32x4*>(dst + chunk_at<T, DP>(it / CH, it % CH)) = r[p];
    }
  }
};

// acc (32 x 32, register rows = contraction-major) += A_rows[row0 .. row0+31][:] . b, over the DP features of b's chunks
template <typename T, int DP>
__device__ __forceinline__ f32x16 dot_rows(const T* rows, int row0, const u32x4* b, f32x16 acc) {
  constexpr int E = Traits<T>::EPC;
  const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
#pragma unroll
  for (int s = 0; s < DP / (2 * E); ++s)
    acc = mfma<T>(*reinterpret_cast<const u32x4*>(rows + row0 * row_pitch<T, DP>() + chunk_at<T, DP>(r, 2 * s + h)), b[s], acc);
  return acc;
}

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// out[t] (features 32t.. x columns) += X^T . w, the contraction over the 32 rows row0.. that w's registers run over.
// 16-bit: X^T by the transposing read: the 16 lanes that hold 16 columns address four rows (lane j: row j >> 2, columns
// from 4 (j & 3)) and receive four rows of their own column.  float: one element a lane and step.
template <typename T, int DP>
__device__ __forceinline__ void dot_cols(const T* x, int row0, const f32x16& w, f32x16* out) {
  const int lane = threadIdx.x & 63, col = lane & 31, h = lane >> 5;
  if constexpr (sizeof(T) == 2) {
    const int r4 = 4 * h + ((lane & 15) >> 2), cc = ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1), half = (lane & 1) * 4;
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const u32x4 b = pack8<T>(w, 8 * g);
#pragma unroll
      for (int t = 0; t < feature_tiles<DP>(); ++t) {
        union { s16x4 v[2]; u32x4 a; } f;
#pragma unroll
        for (int r = 0; r < 2; ++r)
          f.v[r] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(x + (row0 + 16 * g) * DP + chunk_at<T, DP>(8 * r + r4, 4 * t + cc) + half));
        out[t] = mfma<T>(f.a, b, out[t]);
      }
    }
  } else {
#pragma unroll
    for (int r = 0; r < 16; ++r)
#pragma unroll
      for (int t = 0; t < feature_tiles<DP>(); ++t)
        out[t] = __builtin_amdgcn_mfma_f32_32x32x2f32(x[(row0 + crow(r, h)) * row_pitch<T, DP>() + 32 * t + col], w[r], out[t], 0, 0, 0);
  }
}

// chunks of one row as a B operand: chunk s of lane half h covers features (2s + h) * E ..
template <typename T, int DP, bool VEC>
__device__ __forceinline__ void load_row(u32x4* b, const T* __restrict__ p, int D, bool ok) {
  constexpr int E = Traits<T>::EPC;
  const int h = (threadIdx.x & 63) >> 5;
#pragma unroll
  for (int s = 0; s < DP / (2 * E); ++s) b[s] = load_chunk<T, VEC>(p, (2 * s + h) * E, D, ok);
}

// a 32-bit value rounded to T.  The barrier keeps the compiler from folding the product before it into a mixed-precision
// multiply in some instances and not in others (one rounding or two: results would depend on the alignment of a row).
template <typename T>
__device__ __forceinline__ T round_to(float x) {
  if constexpr (__is_same(T, _Float16)) asm("" : "+v"(x));
  return (T)x;
}

// Half precision holds nothing below 2^-24: gradients of scores (a probability times a small number) would vanish.  A lane's
// column of them is scaled by a power of two, chosen from the largest magnitude so far (kept between 2^12 and 2^14), and so is
// what the column has summed; values 2^-38 below the largest are lost, which is below the sum's own rounding.
struct ColScale {
  float sc = 0x1p60f;                              // (products of halves stay below 2^52: no overflow in 32 bits)
  // N tiles of values that already carry sc; true: the scale has changed
  template <int N>
  __device__ __forceinline__ bool fit(f32x16* w, f32x16* acc, int n_acc) {
    float top = 0.0f;
#pragma unroll
    for (int u = 0; u < N; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(w[u][r]));
    top = fmaxf(top, __shfl_xor(top, 32));
    if (!__any(top >= 0x1p14f)) return false;
    rarely();
    const int ex = (int)(__float_as_uint(top) >> 23);                         // 2^(ex - 127) <= top
    const float f = top >= 0x1p14f ? __uint_as_float((uint32_t)max(266 - ex, 12) << 23) : 1.0f;        // top * f in [2^12, 2^13)
#pragma unroll
    for (int t = 0; t < 4; ++t)
      if (t < n_acc)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[t][r] *= f;
#pragma unroll
    for (int u = 0; u < N; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) w[u][r] *= f;
    sc *= f;
    return true;
  }
};

// column `lane & 31` of acc (features x columns) times mul -> one row of D features
template <typename T, int DP, bool VEC>
__device__ __forceinline__ void store_col(T* __restrict__ p, const f32x16* acc, float mul, int D, int tid = threadIdx.x) {
  const int h = (tid & 63) >> 5;
#pragma unroll
  for (int t = 0; t < feature_tiles<DP>(); ++t)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = 32 * t + 8 * g + 4 * h;
      T v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = round_to<T>(acc[t][4 * g + i] * mul);
      if constexpr (VEC) {                        // D is a multiple of the chunk: four features are in or out together
        if (d < D) __builtin_memcpy(__builtin_assume_aligned(p + d, 4 * sizeof(T)), v, 4 * sizeof(T));
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (d + i < D) p[d + i] = v[i];
      }
    }
}

// Half precision: p in [0, 1] takes 2^12 into the product.  p = 1 / Nk of a long list would be subnormal, and below 2^-25 zero
// while the sum still counts it: a long tail of like scores would lose that share of the output.
constexpr float kHalfLog = 12.0f, kHalfP = 4096.0f;
template <typename T> constexpr float p_log() { return __is_same(T, _Float16) ? kHalfLog : 0.0f; }

// log-sum of a row from its maximum and sum; the forward's sums carry p's 2^12 in half precision
template <typename T>
__device__ __forceinline__ float row_lse(float m, float l, float scale) {
  return l == 0.0f ? -INFINITY : m * scale + logf(__is_same(T, _Float16) ? l * (1.0f / kHalfP) : l);
}

// Running softmax over one tile of n keys: raw scores in s become p; m, l and what acc has summed follow the maximum.
template <typename T, int DP, int TK>
__device__ __forceinline__ void softmax_step(f32x16* s, int n, float c, float& m, float& l, f32x16* acc) {
  const int h = (threadIdx.x & 63) >> 5;
  if (n < TK) {
#pragma unroll
    for (int st = 0; st < TK / 32; ++st)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (32 * st + crow(r, h) >= n) s[st][r] = -INFINITY;
  }
  float top = s[0][0];
#pragma unroll
  for (int st = 0; st < TK / 32; ++st)
#pragma unroll
    for (int r = 0; r < 16; ++r) top = fmaxf(top, s[st][r]);
  top = fmaxf(top, __shfl_xor(top, 32));
  const float mn = fmaxf(m, top);
  const float ms = mn == -INFINITY ? 0.0f : mn;   // every score so far -inf: nothing to subtract
  if (__any(mn > m)) {
    const float alpha = __builtin_amdgcn_exp2f((m - ms) * c);
    l *= alpha;
#pragma unroll
    for (int t = 0; t < feature_tiles<DP>(); ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[t][r] *= alpha;
    m = mn;
  }
  // 16-bit inputs: one fused step (the rounding of off moves all p of a row alike and cancels); float: the difference first,
  // which is exact next to the maximum
  const float off = fmaf(-ms, c, p_log<T>());
#pragma unroll
  for (int st = 0; st < TK / 32; ++st)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      s[st][r] = __builtin_amdgcn_exp2f(sizeof(T) == 2 ? fmaf(s[st][r], c, off) : (s[st][r] - ms) * c);
      l += s[st][r];
    }
}

// One tile of n keys (K rows and V in LDS): scores, running softmax, o += V^T P.
template <typename T, int DP, int TK>
__device__ __forceinline__ void attend(const T* Ks, const T* Vs, int n, const u32x4* qf, float c, float& m, float& l, f32x16* acc) {
  f32x16 s[TK / 32];
#pragma unroll
  for (int st = 0; st < TK / 32; ++st) s[st] = dot_rows<T, DP>(Ks, 32 * st, qf, zero16());
  softmax_step<T, DP, TK>(s, n, c, m, l, acc);
  // p is rounded to the inputs' type for the product (16-bit types: half a step relative to p, down to 2^-26 of the row's
  // largest in half precision and 2^-37 absolutely below; the size of the output's own rounding; l sums the unrounded
  // values), the sums over keys stay in 32 bits
#pragma unroll
  for (int st = 0; st < TK / 32; ++st) dot_cols<T, DP>(Vs, 32 * st, s[st], acc);
}

// p from a raw score; st: lse, for 16-bit types in units of log 2.  float: the product and the difference are rounded apart,
// so that a row with a single key, whose log-sum IS its rounded score, gets exactly 1.
template <typename T>
__device__ __forceinline__ float prob(float s, float scale, float c, float st) {
#pragma clang fp contract(off)
  if constexpr (sizeof(T) == 2) return __builtin_amdgcn_exp2f(__builtin_fmaf(s, c, -st));
  const float t = s * scale;
  return __builtin_amdgcn_exp2f((t - st) * kLog2e);
}
// a row without a key (or only scores of -inf): p = 0
template <typename T>
__device__ __forceinline__ float row_stat(float lse) {
  return lse == -INFINITY ? INFINITY : sizeof(T) == 2 ? lse * kLog2e : lse;
}

// log2 of a power of two
__device__ __forceinline__ float log2_pow2(float x) { return (float)((int)(__float_as_uint(x) >> 23) - 127); }

// Workgroup id -> (unit, item): units (clouds, or (cloud, key head) pairs when there are few clouds) are dealt to the
// eight XCDs in turn and all items of a unit stay on one XCD, whose L2 then holds the rows they share.
struct GridMap {
  int units, items, swizzle;
  __host__ __device__ int64_t blocks() const { return (int64_t)(swizzle ? (units + 7) / 8 * 8 : units) * items; }
  __device__ __forceinline__ bool decode(int64_t id, int& unit, int& item) const {
    if (!swizzle) {
      unit = (int)(id / items);
      item = (int)(id - (int64_t)unit * items);
      return true;
    }
    const int64_t y = id >> 3;
    unit = (int)(y / items) * 8 + (int)(id & 7);
    item = (int)(y % items);
    return unit < units;
  }
};
inline GridMap grid_map(int B, int nkv, int per_head) {
  GridMap g;
  if ((int64_t)nkv * per_head > 0x7fffffff) return {0x7fffffff, 0x7fffffff, 0};       // (more than any launch takes)
  if (B % 8 == 0 || B >= 64) g = {B, nkv * per_head, 1};
  else if ((int64_t)B * nkv >= 64 || (B * nkv) % 8 == 0) g = {B * nkv, per_head, 1};
  else g = {B * nkv, per_head, 0};
  return g;
}

// zeros in the rows r0 .. r0 + rows - 1 (row = slot * g + head of the group) whose slot the mask drops; four lanes a row
template <int NT, bool VEC, typename T>
__device__ __forceinline__ void zero_masked_rows(T* __restrict__ out, int64_t ld, const float* __restrict__ maskf, int r0, int rows,
                                                 int g, int D) {
  constexpr int E = Traits<T>::EPC;
  for (int r = threadIdx.x >> 2; r < rows; r += NT / 4) {
    const int n = g == 1 ? r0 + r : (r0 + r) / g, gi = r0 + r - n * g;
    if (maskf[n] != 0.0f) continue;
    T* o = out + (int64_t)n * ld + gi * D;
    if constexpr (VEC) {
      for (int d = (threadIdx.x & 3) * E; d < D; d += 4 * E) *reinterpret_cast<u32x4*>(o + d) = u32x4{0u, 0u, 0u, 0u};
    } else {
      for (int d = threadIdx.x & 3; d < D; d += 4) o[d] = (T)0.0f;
    }
  }
}

// the rows of a tile: list of compacted slots (from first_c on), row -> (slot, head of the group)
struct RowTile {
  int first_c, g;
  const int* list;
  __device__ __forceinline__ bool locate(int r, int N, bool masked, int& n, int& gi) const {
    const int c = r / g;
    gi = r - c * g;
    n = masked ? list[c - first_c] : (c < N ? c : -1);
    return n >= 0;
  }
};

// kept slots of a mask (or all), one wave; returns their number
__device__ __forceinline__ int keep_list(const float* __restrict__ maskf, int N, int* list) {
  if (maskf == nullptr) {
    for (int i = threadIdx.x & 63; i < N; i += 64) list[i] = i;
    return N;
  }
  int c = 0;
  for (int lo = 0; lo < N; lo += kChunk) c += compact_chunk(maskf, lo, N, list + c);
  return c;
}

struct Shape {
  int B, Nq, Nk, nh, nkv, D, g;                   // g = nh / nkv query heads share one key head
};

// small clouds (cross_attention_resident.hip)
bool resident_fits(const Shape& s, int dtype, bool bwd);
int resident_fwd(const Shape& s, int dtype, bool vec, const void* q, int64_t q_ld, const void* k, int64_t k_ld, const void* v,
                 int64_t v_ld, const float* mq, const float* mk, float scale, void* out, int64_t out_ld, float* lse, hipStream_t st);
int resident_bwd(const Shape& s, int dtype, bool vec, const void* q, int64_t q_ld, const void* k, int64_t k_ld, const void* v,
                 int64_t v_ld, const float* mq, const float* mk, float scale, const void* out, int64_t out_ld, const void* dout,
                 int64_t dout_ld, const float* lse, void* dq, int64_t dq_ld, void* dk, int64_t dk_ld, void* dv, int64_t dv_ld, hipStream_t st);

// the same in floats with narrow heads (cross_attention_jets.hip)
bool jets_fit(const Shape& s, int dtype, bool bwd);
int jets_fwd(const Shape& s, bool vec, const float* q, int64_t q_ld, const float* k, int64_t k_ld, const float* v, int64_t v_ld,
             const float* mq, const float* mk, float scale, float* out, int64_t out_ld, float* lse, hipStream_t st);
int jets_bwd(const Shape& s, bool vec, const float* q, int64_t q_ld, const float* k, int64_t k_ld, const float* v, int64_t v_ld,
             const float* mq, const float* mk, float scale, const float* out, int64_t out_ld, const float* dout, int64_t dout_ld,
             const float* lse, float* dq, int64_t dq_ld, float* dk, int64_t dk_ld, float* dv, int64_t dv_ld, hipStream_t st);

inline int pad_width(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : 128; }
int check_shape(const char* who, int B, int Nq, int Nk, int nh, int nkv, int D, int dtype, float scale);
inline bool chunk_aligned(const void* p, int64_t ld, int es) { return ((uintptr_t)p & 15) == 0 && ld * es % 16 == 0; }

}  // namespace xattn
}  // namespace mmb
