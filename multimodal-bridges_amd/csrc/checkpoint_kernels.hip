// Activations kept for the reverse pass in 8 bits, and the weight gradient read from them.
//
// 32 consecutive features of a row share a step 2^e: e is the smallest exponent (>= -127) with 127 * 2^e >= max |x|, the
// codes are round(x / 2^e) in [-127, 127], ties to even.  Both divisions are by powers of two, so a code depends on no
// rounding but its own, and a value stands for at most half a step off: |xhat - x| <= 2^(e-1), which is below max|x| / 127
// but for blocks of subnormals (e = -127 is the smallest).  At the other end, e = 122, 64 steps would be 2^128: codes end at
// 63 there and the values next to the largest float are up to a step off.  An integer
// grid over a shared step holds a block of like-sized activations about four times closer than an 8-bit float would (whose
// three mantissa bits spend the range on small values).
// With keep_nonzero a value that would round to code 0 takes code +-1 (a step off at most, not half): what is told from the
// sign of an activation -- whether a ReLU passes the gradient -- is then told the same from its checkpoint.
// step byte = e + 127; 255 marks a block that held an infinity or a NaN: it comes back as NaN, never as a finite value.
//
// A code is an integer of 7 bits: code * 2^e is EXACT in bf16.  The weight gradient dW = dZ^T Xhat therefore needs ONE bf16
// plane for Xhat and three for a float dZ (exact split, truncated 8 + 8 + 8 bits; two for fp16, one for bf16): three matrix
// products where float activations need six, and a quarter of the bytes.
#include "regions.h"

namespace mmb {
namespace ckpt {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <typename T> __device__ __forceinline__ float max_of();
template <> __device__ __forceinline__ float max_of<float>() { return 3.4028234663852886e38f; }
template <> __device__ __forceinline__ float max_of<__bf16>() { return 3.3895313892515355e38f; }
template <> __device__ __forceinline__ float max_of<_Float16>() { return 65504.0f; }

__device__ __forceinline__ float step_of(uint32_t s) {      // 2^(s - 127); s == 0: the subnormal 2^-127; 255: NaN
  return __uint_as_float(s == 255u ? 0x7fc00000u : s == 0u ? 0x00400000u : s << 23);
}

template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* __restrict__ p, int k, int K, float v[8]) {
  if constexpr (VEC) {
    if (k >= K) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    } else if constexpr (sizeof(T) == 4) {
      const float4 a = *reinterpret_cast<const float4*>(p + k), b = *reinterpret_cast<const float4*>(p + k + 4);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
      T t[8];
      const uint4 a = *reinterpret_cast<const uint4*>(p + k);
      __builtin_memcpy(t, &a, 16);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = (float)t[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = k + i < K ? (float)p[k + i] : 0.0f;
  }
}

// a thread owns 8 features, four neighbouring lanes one block of 32
template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
encode_kernel(int64_t M, int K, int nb, int keep_nonzero, const T* __restrict__ x, int64_t x_ld, int8_t* __restrict__ codes,
              uint8_t* __restrict__ steps) {
  const int64_t n = M * nb * 4;
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < n; t += (int64_t)gridDim.x * 256) {
    const int64_t blk = t >> 2, row = blk / nb;
    const int k = (int)(blk - row * nb) * 32 + (int)(t & 3) * 8;
    float v[8];
    load8<T, VEC>(x + row * x_ld, k, K, v);
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
    top = max(top, (uint32_t)__shfl_xor((int)top, 1, 64));
    top = max(top, (uint32_t)__shfl_xor((int)top, 2, 64));
    uint32_t s = 255u;
    uint2 packed = make_uint2(0u, 0u);
    if (top < 0x7f800000u) {
      // max = 1.m 2^(E-127); 127 = 1.984375 2^6 (mantissa 0x7e0000)
      const int e = (int)(top >> 23) - 6 + ((top & 0x7fffffu) > 0x7e0000u ? 1 : 0);
      s = (uint32_t)max(e, 0);
      const float inv = __uint_as_float((254u - s) << 23);              // 2^-(s - 127), s <= 249
      const float lim = s >= 249u ? 63.0f : 127.0f;                     // (64 * 2^122 would leave the range of a float)
      int q[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        q[i] = (int)fminf(fmaxf(rintf(v[i] * inv), -lim), lim);
        if (keep_nonzero && q[i] == 0 && v[i] != 0.0f) q[i] = v[i] > 0.0f ? 1 : -1;
      }
      packed.x = (q[0] & 255) | (q[1] & 255) << 8 | (q[2] & 255) << 16 | (uint32_t)q[3] << 24;
      packed.y = (q[4] & 255) | (q[5] & 255) << 8 | (q[6] & 255) << 16 | (uint32_t)q[7] << 24;
    }
    *reinterpret_cast<uint2*>(codes + t * 8) = packed;
    if ((t & 3) == 0) steps[blk] = (uint8_t)s;
  }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
decode_kernel(int64_t M, int K, int nb, const int8_t* __restrict__ codes, const uint8_t* __restrict__ steps, T* __restrict__ y, int64_t y_ld) {
  const int64_t n = M * nb * 4;
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < n; t += (int64_t)gridDim.x * 256) {
    const int64_t blk = t >> 2, row = blk / nb;
    const int k = (int)(blk - row * nb) * 32 + (int)(t & 3) * 8;
    const uint2 c = *reinterpret_cast<const uint2*>(codes + t * 8);
    const uint32_t s = steps[blk];
    const float st = step_of(s), big = max_of<T>();
    T o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t w = i < 4 ? c.x : c.y;
      float f = (float)(int8_t)(w >> (8 * (i & 3))) * st;
      if (s != 255u) f = fminf(fmaxf(f, -big), big);      // (a code next to the type's largest value may round past it)
      o[i] = (T)f;
    }
    T* p = y + row * y_ld + k;
    if constexpr (VEC) {
      if (k < K) {
        if constexpr (sizeof(T) == 4) {
          *reinterpret_cast<float4*>(p) = make_float4(o[0], o[1], o[2], o[3]);
          *reinterpret_cast<float4*>(p + 4) = make_float4(o[4], o[5], o[6], o[7]);
        } else {
          uint4 a;
          __builtin_memcpy(&a, o, 16);
          *reinterpret_cast<uint4*>(p) = a;
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (k + i < K) p[i] = o[i];
    }
  }
}

// ---- dW (N, K) = dZ^T (N, M) . Xhat (M, K), db (N) = column sums of dZ -------------------------------------------
// A workgroup owns a BN x BK tile of dW (128 x 128, 128 x 256 with four waves, 256 x 256 with eight) over a range of rows and
// walks the range 32 rows at a time; a wave computes 64 x BK/2.  What a wave has to decode and move beside its products falls
// with the tile's size.  dZ (in bf16 planes) and Xhat lie in LDS as they come, row by row; the matrix operands want
// eight consecutive ROWS of one column, which the transposing LDS read supplies (four rows of 16 columns per 16 lanes), so
// nothing is transposed in registers.  Row pitch 16 banks past a multiple of 64: the four rows of such a read do not meet.
// Two buffers, one barrier a step; the rows of the two steps behind are on their way to registers meanwhile.
// The rows are split over workgroups to fill the chip; partial tiles are summed by a second launch in a fixed order (no
// atomics: equal inputs give equal bits).
constexpr int MS = 32;                            // rows of a step
constexpr int pitch_of(int cols) { return cols + 32; }

template <typename T> struct Planes;
template <> struct Planes<float> { static constexpr int n = 3; };
template <> struct Planes<_Float16> { static constexpr int n = 2; };
template <> struct Planes<__bf16> { static constexpr int n = 1; };

struct GwArgs {
  int64_t M;
  int N, K, nb, nt, kt, splits;
  int64_t rows;                                   // rows a split walks, a multiple of MS
  const int8_t* codes;
  const uint8_t* steps;
  const void* dz;
  int64_t dz_ld;
  float *pw, *pb;                                 // partial sums (splits, N, K), (splits, N)
};

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// rows 8h .. 8h+7 (h: lane half) of column (lane & 31) of a row-major LDS block: two transposing reads of four rows
__device__ __forceinline__ u32x4 read_cols(const uint16_t* p, int pitch) {
  union { s16x4 h[2]; u32x4 v; } r;
  r.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
  r.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 4 * pitch));
  return r.v;
}

template <typename T, int BN, int BK>
constexpr int gw_lds() { return 2 * MS * (Planes<T>::n * pitch_of(BN) + pitch_of(BK)) * 2; }

// (No instance may spill registers: the compiler has stored one under a narrowed exec mask and read it back for all lanes.  One
// wave a SIMD for 128 x 256 tiles of float -- their LDS admits no more -- and of half precision element by element.)
template <typename T, int BN, int BK, bool VEC>
__global__ void __launch_bounds__(2 * BN, BN < BK && (Planes<T>::n == 3 || (Planes<T>::n == 2 && !VEC)) ? 1 : 2) gw_kernel(GwArgs a) {
  constexpr int NT = 2 * BN, NWN = BN / 64;
  constexpr int PL = Planes<T>::n, PA = pitch_of(BN), PB = pitch_of(BK), NJ = BK / 64, XC = MS * BK / 16 / NT;
  extern __shared__ __attribute__((aligned(16))) uint16_t gw_sm[];
  constexpr int BUF = MS * (PL * PA + PB);
  const int tiles = a.nt * a.kt;
  // all tiles of one row range on one XCD (workgroup ids go round the eight): they read the same rows
  const int64_t y = blockIdx.x >> 3;
  const int split = (int)(y / tiles) * 8 + (int)(blockIdx.x & 7), tile = (int)(y % tiles);
  if (split >= a.splits) return;
  const int n0 = (tile % a.nt) * BN, k0 = (tile / a.nt) * BK;
  const bool sums = tile / a.nt == 0;              // the tiles of the first K window also sum dZ's columns
  const int64_t m0 = (int64_t)split * a.rows, m1 = min(a.M, m0 + a.rows);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, col = lane & 31, h = lane >> 5;
  const int wn = wave % NWN * 64, wk = wave / NWN * (BK / 2);
  // transposing reads: lane j of 16 addresses row j >> 2, four columns from 4 (j & 3)
  const int tr_row = 8 * h + ((lane & 15) >> 2), tr_col = ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
  // loads: dZ rows zr, zr + 16 .., eight columns; Xhat 16 codes a chunk
  const int zr = threadIdx.x / (BN / 8), zc = threadIdx.x % (BN / 8) * 8;
  f32x16 acc[2][NJ];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
  float db[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  constexpr int ZW = sizeof(T) == 4 ? 8 : 4;       // words of eight elements
  struct Step {                                    // one step's rows on their way from memory to LDS
    uint32_t zw[MS / 16][ZW];
    u32x4 cw[XC];
    uint32_t sw[XC];
  } steps[2];
  // addresses: a uniform part that moves with the rows, and 32-bit offsets that stay.  Columns past the matrix read column 0
  // instead: what they multiply into is not stored.
  const int zcol = n0 + zc < a.N ? zc : 0;
  const uint32_t zoff = (uint32_t)(zr * a.dz_ld + zcol) * (uint32_t)sizeof(T);
  uint32_t coff[XC], soff[XC];
  int crow_[XC];
#pragma unroll
  for (int j = 0; j < XC; ++j) {
    const int it = threadIdx.x + NT * j, c = (it % (BK / 16)) * 16, cc = k0 + c < a.nb * 32 ? k0 + c : 0;
    crow_[j] = it / (BK / 16);
    coff[j] = (uint32_t)crow_[j] * (uint32_t)(a.nb * 32) + cc;
    soff[j] = (uint32_t)crow_[j] * (uint32_t)a.nb + cc / 32;
  }
  auto fetch = [&](Step& st, int64_t m) {
    auto &zw = st.zw;
    auto &cw = st.cw;
    auto &sw = st.sw;
    const int left = (int)min((int64_t)MS, m1 - m);                         // rows of this step: fewer than MS in the last only
    const char* zb = reinterpret_cast<const char*>((const T*)a.dz + m * a.dz_ld + n0);
    const int8_t* cb = a.codes + m * (a.nb * 32);
    const uint8_t* sb = a.steps + m * a.nb;
#pragma unroll
    for (int j = 0; j < MS / 16; ++j) {
      const bool in = left == MS || zr + 16 * j < left;
      if constexpr (VEC) {
        const char* p = zb + (int64_t)j * 16 * a.dz_ld * (int64_t)sizeof(T);
#pragma unroll
        for (int w = 0; w < ZW / 4; ++w) {
          const u32x4 t = in ? *reinterpret_cast<const u32x4*>(p + zoff + 16 * w) : u32x4{0u, 0u, 0u, 0u};
#pragma unroll
          for (int i = 0; i < 4; ++i) zw[j][4 * w + i] = t[i];
        }
      } else {
        const T* p = (const T*)a.dz + (m + zr + 16 * j) * a.dz_ld + n0 + zc;
        T t[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = in && n0 + zc + i < a.N ? p[i] : (T)0.0f;
        __builtin_memcpy(zw[j], t, sizeof(t));
      }
    }
#pragma unroll
    for (int j = 0; j < XC; ++j) {
      const bool in = left == MS || crow_[j] < left;
      cw[j] = in ? *reinterpret_cast<const u32x4*>(cb + coff[j]) : u32x4{0u, 0u, 0u, 0u};
      sw[j] = in ? sb[soff[j]] : 0u;
    }
  };
  auto put = [&](const Step& step, uint16_t* buf) {
    const auto &zw = step.zw;
    const auto &cw = step.cw;
    const auto &sw = step.sw;
#pragma unroll
    for (int j = 0; j < MS / 16; ++j) {
      uint16_t* dst = buf + (zr + 16 * j) * PA + zc;
      float f[8];
      if (PL > 1 || sums) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(zw[j][i]);
        } else if constexpr (PL > 1) {
          T t[8];
          __builtin_memcpy(t, zw[j], 16);
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] = (float)t[i];
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            f[2 * i] = __uint_as_float(zw[j][i] << 16);
            f[2 * i + 1] = __uint_as_float(zw[j][i] & 0xffff0000u);
          }
        }
        if (sums) {
#pragma unroll
          for (int i = 0; i < 8; ++i) db[i] += f[i];
        }
      }
      if constexpr (PL == 1) {
        *reinterpret_cast<u32x4*>(dst) = u32x4{zw[j][0], zw[j][1], zw[j][2], zw[j][3]};
      } else {                                     // truncated planes: x = hi + mid (+ lo) exactly
#pragma unroll
        for (int p = 0; p < PL; ++p) {
          u32x4 w;
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = __builtin_amdgcn_perm(__float_as_uint(f[2 * i + 1]), __float_as_uint(f[2 * i]), 0x07060302u);
          *reinterpret_cast<u32x4*>(dst + p * MS * PA) = w;
          if (p + 1 < PL) {
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] -= __uint_as_float(__float_as_uint(f[i]) & 0xffff0000u);
          }
        }
      }
    }
#pragma unroll
    for (int j = 0; j < XC; ++j) {
      const int it = threadIdx.x + NT * j;
      uint16_t* dst = buf + MS * PL * PA + (it / (BK / 16)) * PB + (it % (BK / 16)) * 16;
      const float st = step_of(sw[j]);
      // code * step with the code as an unsigned byte, offset by 128: (u - 128) step, exact in one fused step -- unless
      // 128 step leaves the range of a float
      const bool huge = __any(sw[j] >= 248u);
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t u = cw[j][2 * q + i] ^ 0x80808080u;
#pragma unroll
          for (int k = 0; k < 4; ++k) x[4 * i + k] = fmaf((float)((u >> (8 * k)) & 255u), st, -128.0f * st);
        }
        if (huge) {
          asm volatile("");                        // (a branch: not computed beside the above)
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = (float)(int8_t)(cw[j][2 * q + (i >> 2)] >> (8 * (i & 3))) * st;
        }
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __builtin_amdgcn_perm(__float_as_uint(x[2 * i + 1]), __float_as_uint(x[2 * i]), 0x07060302u);
        *reinterpret_cast<u32x4*>(dst + 8 * q) = w;
      }
    }
  };
  auto products = [&](const uint16_t* buf) {
    const uint16_t* As = buf + tr_row * PA + wn + tr_col;
    const uint16_t* Bs = buf + MS * PL * PA + tr_row * PB + wk + tr_col;
#pragma unroll
    for (int s = 0; s < MS / 16; ++s) {
      u32x4 bf[NJ];
#pragma unroll
      for (int j = 0; j < NJ; ++j) bf[j] = read_cols(Bs + 16 * s * PB + 32 * j, PB);
#pragma unroll
      for (int q = PL - 1; q >= 0; --q)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const bf16x8 af = __builtin_bit_cast(bf16x8, read_cols(As + q * MS * PA + 16 * s * PA + 32 * i, PA));
#pragma unroll
          for (int j = 0; j < NJ; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(af, __builtin_bit_cast(bf16x8, bf[j]), acc[i][j], 0, 0, 0);
        }
    }
  };
  // two steps' rows are on their way while one is worked on; of the two LDS buffers one is written while the other is read
  fetch(steps[0], m0);
  if (m0 + MS < m1) fetch(steps[1], m0 + MS);
  for (int64_t m = m0; m < m1; m += 2 * MS) {
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int64_t at = m + p * MS;
      if (at >= m1) break;
      put(steps[p], gw_sm + p * BUF);
      if (at + 2 * MS < m1) fetch(steps[p], at + 2 * MS);
      __syncthreads();                             // (the other buffer's readers passed here after their products)
      products(gw_sm + p * BUF);
    }
  }
  float* pw = a.pw + (int64_t)split * a.N * a.K;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int n = n0 + wn + 32 * i + (r >> 2) * 8 + h * 4 + (r & 3), k = k0 + wk + 32 * j + col;
        if (n < a.N && k < a.K) pw[(int64_t)n * a.K + k] = acc[i][j][r];
      }
  if (sums) {
    float* red = reinterpret_cast<float*>(gw_sm);  // 16 row groups x BN columns
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) red[zr * BN + zc + i] = db[i];
    __syncthreads();
    if (threadIdx.x < BN && n0 + threadIdx.x < a.N) {
      float s = 0.0f;
#pragma unroll
      for (int q = 0; q < 16; ++q) s += red[q * BN + threadIdx.x];
      a.pb[(int64_t)split * a.N + n0 + threadIdx.x] = s;
    }
  }
}

// dW, db from the partial sums of the row ranges: eight threads share the ranges of one element, joined in LDS
__global__ void __launch_bounds__(256)
gw_fold_kernel(int64_t first, int splits, int64_t nw, int N, int K, const float* __restrict__ pw, const float* __restrict__ pb,
               float* __restrict__ dW, int64_t dw_ld, float* __restrict__ db, int accumulate) {
  __shared__ float red[8][33];
  const int c = threadIdx.x & 31, g = threadIdx.x >> 5;
  const int64_t i = first + (int64_t)blockIdx.x * 32 + c;
  float s = 0.0f;
  if (i < nw) {
#pragma unroll 4
    for (int p = g; p < splits; p += 8) s += pw[(int64_t)p * nw + i];
  } else if (i < nw + N) {
    for (int p = g; p < splits; p += 8) s += pb[(int64_t)p * N + (i - nw)];
  }
  red[g][c] = s;
  __syncthreads();
  if (g != 0 || i >= nw + N) return;
#pragma unroll
  for (int q = 1; q < 8; ++q) s += red[q][c];
  if (i < nw) {
    float* d = dW + i / K * dw_ld + i % K;
    *d = accumulate ? *d + s : s;
  } else if (db) {
    db[i - nw] = accumulate ? db[i - nw] + s : s;
  }
}

// Tile: 256 x 256 where both sides have more than 128 columns and it wastes little more than 128-wide tiles would.
// Row ranges: enough workgroups for eight waves on every CU, no range shorter than 8 steps, and no more partial sums than a
// quarter of what the operands themselves hold (they are written and read once more).
struct GwPlan {
  int bn, bk, nt, kt, splits;
  int64_t rows;
};
static GwPlan gw_plan(int64_t M, int N, int K) {
  GwPlan p;
  p.bk = K > 128 ? 256 : 128;
  p.bn = p.bk == 256 && N > 128 && (int64_t)(N + 255) / 256 * 256 * 4 <= (int64_t)(N + 127) / 128 * 128 * 5 ? 256 : 128;
  p.nt = (N + p.bn - 1) / p.bn;
  p.kt = (K + p.bk - 1) / p.bk;
  const int64_t tiles = (int64_t)p.nt * p.kt, groups = p.bn == 256 ? 256 : 512;
  int64_t s = (groups + tiles - 1) / tiles;
  const int64_t most = (M + 8 * MS - 1) / (8 * MS), fit = M * ((int64_t)K + 4 * N) / (32 * (int64_t)N * K) + 1;
  if (s > most) s = most;
  if (s > fit) s = fit;
  if (s < 1) s = 1;
  p.rows = (M + s * MS - 1) / (s * MS) * MS;
  p.splits = (int)((M + p.rows - 1) / p.rows);
  return p;
}

static int check_q8(const char* who, int64_t M, int K, const void* codes, const void* steps) {
  MMB_REQUIRE(M > 0 && K > 0 && K <= (1 << 20), "%s: M must be positive, K in 1..2^20 (got %lld, %d)", who, (long long)M, K);
  MMB_REQUIRE(codes && steps, "%s: codes or steps is NULL", who);
  MMB_REQUIRE(((uintptr_t)codes & 15) == 0, "%s: codes must be 16-byte aligned", who);
  return MMB_OK;
}
static int elem_bytes(int dtype) { return dtype == MMB_DT_F32 ? 4 : dtype == MMB_DT_BF16 || dtype == MMB_DT_F16 ? 2 : 0; }
static Region code_region(const void* codes, int64_t M, int K) { return flat_region(codes, M * ((K + 31) / 32 * 32)); }
static Region step_region(const void* steps, int64_t M, int K) { return flat_region(steps, M * ((K + 31) / 32)); }

template <typename T>
static int encode(int64_t M, int K, int keep_nonzero, const void* x, int64_t x_ld, void* codes, void* steps, hipStream_t st) {
  const int nb = (K + 31) / 32, grid = stream_grid(M * nb * 4, 256);
  const bool vec = K % 8 == 0 && ((uintptr_t)x & 15) == 0 && x_ld * (int64_t)sizeof(T) % 16 == 0;
  if (vec) encode_kernel<T, true><<<grid, 256, 0, st>>>(M, K, nb, keep_nonzero, (const T*)x, x_ld, (int8_t*)codes, (uint8_t*)steps);
  else encode_kernel<T, false><<<grid, 256, 0, st>>>(M, K, nb, keep_nonzero, (const T*)x, x_ld, (int8_t*)codes, (uint8_t*)steps);
  return check_launch("mmb_checkpoint_rows");
}
template <typename T>
static int decode(int64_t M, int K, const void* codes, const void* steps, void* y, int64_t y_ld, hipStream_t st) {
  const int nb = (K + 31) / 32, grid = stream_grid(M * nb * 4, 256);
  const bool vec = K % 8 == 0 && ((uintptr_t)y & 15) == 0 && y_ld * (int64_t)sizeof(T) % 16 == 0;
  if (vec) decode_kernel<T, true><<<grid, 256, 0, st>>>(M, K, nb, (const int8_t*)codes, (const uint8_t*)steps, (T*)y, y_ld);
  else decode_kernel<T, false><<<grid, 256, 0, st>>>(M, K, nb, (const int8_t*)codes, (const uint8_t*)steps, (T*)y, y_ld);
  return check_launch("mmb_restore_rows");
}
template <typename T, int BN, int BK, bool VEC>
static int launch_gw(const GwArgs& a, hipStream_t st) {
  constexpr int bytes = gw_lds<T, BN, BK>();
  static_assert(bytes <= 160 * 1024, "LDS");
  const int64_t blocks = (int64_t)(a.splits + 7) / 8 * 8 * a.nt * a.kt;
  MMB_REQUIRE(grid_fits(blocks, 2 * BN), "mmb_grad_weight_rows_q8: %lld workgroups are more than a launch takes", (long long)blocks);
  auto kern = gw_kernel<T, BN, BK, VEC>;
  static PerDeviceOnce once;
  if (bytes > 64 * 1024 &&
      !once.run([&] { return hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) == hipSuccess; })) {
    set_error("mmb_grad_weight_rows_q8: the runtime refuses %d bytes of LDS", bytes);
    return MMB_ERR_LAUNCH;
  }
  kern<<<(unsigned)blocks, 2 * BN, bytes, st>>>(a);
  return check_launch("mmb_grad_weight_rows_q8");
}
template <typename T, bool VEC>
static int pick_tile(const GwArgs& a, const GwPlan& p, hipStream_t st) {
  if (p.bn == 256) return launch_gw<T, 256, 256, VEC>(a, st);
  return p.bk == 256 ? launch_gw<T, 128, 256, VEC>(a, st) : launch_gw<T, 128, 128, VEC>(a, st);
}
template <typename T>
static int grad_weight(GwArgs& a, const GwPlan& p, float* dW, int64_t dw_ld, float* db, int accumulate, hipStream_t st) {
  const bool vec = a.N % 8 == 0 && ((uintptr_t)a.dz & 15) == 0 && a.dz_ld * (int64_t)sizeof(T) % 16 == 0 && a.dz_ld < (1 << 24);
  const int64_t nw = (int64_t)a.N * a.K, fold = (nw + a.N + 31) / 32, most = 1 << 23;      // (blocks of one launch)
  int rc = vec ? pick_tile<T, true>(a, p, st) : pick_tile<T, false>(a, p, st);
  if (rc != MMB_OK) return rc;
  for (int64_t at = 0; at < fold && rc == MMB_OK; at += most) {
    gw_fold_kernel<<<(unsigned)(fold - at < most ? fold - at : most), 256, 0, st>>>(at * 32, a.splits, nw, a.N, a.K, a.pw, a.pb, dW, dw_ld, db,
                                                                                    accumulate);
    rc = check_launch("mmb_grad_weight_rows_q8 (fold)");
  }
  return rc;
}

}  // namespace ckpt
}  // namespace mmb

using namespace mmb;
using namespace mmb::ckpt;

extern "C" int mmb_checkpoint_rows(int64_t M, int K, int dtype, int keep_nonzero, const void* x, int64_t x_ld, void* codes, void* steps,
                                   void* stream) {
  if (int rc = check_q8("mmb_checkpoint_rows", M, K, codes, steps)) return rc;
  MMB_REQUIRE(x && x_ld >= K, "mmb_checkpoint_rows: x is NULL or its leading dimension smaller than its row");
  const int es = elem_bytes(dtype);
  MMB_REQUIRE(es, "mmb_checkpoint_rows: unknown dtype %d", dtype);
  const Region outs[] = {code_region(codes, M, K), step_region(steps, M, K)}, in = row_region(x, M, K, x_ld, es);
  if (int rc = check_apart("mmb_checkpoint_rows", outs, 2, &in, 1)) return rc;
  hipStream_t st = as_stream(stream);
  if (dtype == MMB_DT_F32) return encode<float>(M, K, keep_nonzero != 0, x, x_ld, codes, steps, st);
  if (dtype == MMB_DT_BF16) return encode<__bf16>(M, K, keep_nonzero != 0, x, x_ld, codes, steps, st);
  return encode<_Float16>(M, K, keep_nonzero != 0, x, x_ld, codes, steps, st);
}

extern "C" int mmb_restore_rows(int64_t M, int K, int dtype, const void* codes, const void* steps, void* y, int64_t y_ld, void* stream) {
  if (int rc = check_q8("mmb_restore_rows", M, K, codes, steps)) return rc;
  MMB_REQUIRE(y && y_ld >= K, "mmb_restore_rows: y is NULL or its leading dimension smaller than its row");
  const int es = elem_bytes(dtype);
  MMB_REQUIRE(es, "mmb_restore_rows: unknown dtype %d", dtype);
  const Region out = row_region(y, M, K, y_ld, es), ins[] = {code_region(codes, M, K), step_region(steps, M, K)};
  if (int rc = check_apart("mmb_restore_rows", &out, 1, ins, 2)) return rc;
  hipStream_t st = as_stream(stream);
  if (dtype == MMB_DT_F32) return decode<float>(M, K, codes, steps, y, y_ld, st);
  if (dtype == MMB_DT_BF16) return decode<__bf16>(M, K, codes, steps, y, y_ld, st);
  return decode<_Float16>(M, K, codes, steps, y, y_ld, st);
}

extern "C" int mmb_grad_weight_rows_q8_workspace(int64_t M, int N, int K, int64_t* bytes_host) {
  MMB_REQUIRE(M > 0 && N > 0 && K > 0 && N <= (1 << 20) && K <= (1 << 20) && bytes_host,
              "mmb_grad_weight_rows_q8_workspace: sizes must be positive, N and K at most 2^20, bytes_host not NULL");
  *bytes_host = (int64_t)gw_plan(M, N, K).splits * ((int64_t)N * K + N) * 4;
  return MMB_OK;
}

extern "C" int mmb_grad_weight_rows_q8(int64_t M, int K, int N, int dtype, const void* codes, const void* steps, const void* dZ,
                                       int64_t dz_ld, float* dW, int64_t dw_ld, float* db, int accumulate, void* workspace,
                                       int64_t workspace_bytes, void* stream) {
  if (int rc = check_q8("mmb_grad_weight_rows_q8", M, K, codes, steps)) return rc;
  MMB_REQUIRE(N > 0 && N <= (1 << 20) && dZ && dz_ld >= N && dW && dw_ld >= K,
              "mmb_grad_weight_rows_q8: N in 1..2^20, dZ, dW not NULL, leading dimensions no smaller than their rows");
  const GwPlan p = gw_plan(M, N, K);
  GwArgs a = {M, N, K, (K + 31) / 32, p.nt, p.kt, p.splits, p.rows, (const int8_t*)codes, (const uint8_t*)steps, dZ, dz_ld, nullptr, nullptr};
  const int64_t need = (int64_t)a.splits * ((int64_t)N * K + N) * 4;
  MMB_REQUIRE(workspace && workspace_bytes >= need, "mmb_grad_weight_rows_q8: workspace of %lld bytes needed, got %lld", (long long)need,
              (long long)(workspace ? workspace_bytes : 0));
  const int es = elem_bytes(dtype);
  MMB_REQUIRE(es, "mmb_grad_weight_rows_q8: unknown dtype %d", dtype);
  const Region outs[] = {row_region(dW, N, K, dw_ld, 4), flat_region(db, 4 * (int64_t)N), flat_region(workspace, need)};
  const Region ins[] = {code_region(codes, M, K), step_region(steps, M, K), row_region(dZ, M, N, dz_ld, es)};
  if (int rc = check_apart("mmb_grad_weight_rows_q8", outs, 3, ins, 3)) return rc;
  a.pw = (float*)workspace;
  a.pb = a.pw + (int64_t)a.splits * N * K;
  hipStream_t st = as_stream(stream);
  if (dtype == MMB_DT_F32) return grad_weight<float>(a, p, dW, dw_ld, db, accumulate, st);
  if (dtype == MMB_DT_BF16) return grad_weight<__bf16>(a, p, dW, dw_ld, db, accumulate, st);
  return grad_weight<_Float16>(a, p, dW, dw_ld, db, accumulate, st);
}
