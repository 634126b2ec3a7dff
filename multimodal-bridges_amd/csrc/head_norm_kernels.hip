// Norm of every query and key head, and the rotation by the rows' positions, in one pass (forward and reverse).
//
//   r = 1 / sqrt(mean_d x^2 + eps);   u = x r w;   pair p = (a, b):  (a cos t - b sin t, a sin t + b cos t),
//   t = pos[row][axis of p] freq[p]
// Reverse, with g = the rotation's transpose applied to dy:
//   dw_d = sum over rows and heads of g_d x_d r;      dx = r (g w - x r^2 mean_d (g w x))
//
// Memory bound: x is read once, y written once.  A thread owns eight consecutive features of ONE row and walks the heads of
// that row, so its angles -- the same for every head -- are computed once.  The angle is formed in 64 bits (the product of
// two floats is exact there) and reduced to a fraction of a turn before the 32-bit sine: positions far down a list keep
// full accuracy.  Statistics and products are in 32 bits, one rounding when a value is stored.
#include "regions.h"

namespace mmb {
namespace headnorm {

constexpr int kMaxBlocks = MMB_HEAD_NORM_MAX_BLOCKS;

struct Args {
  int64_t M;
  int nh1, nh2, D, P, per_axis, interleaved;       // P rotated pairs, per_axis of them on each coordinate
  const void *x, *dy;
  const float *w1, *w2, *pos, *freq;
  int64_t x_ld, dy_ld, pos_ld, y_ld;
  float eps;
  void* y;                                         // forward: y; reverse: dx
  float* part;                                     // reverse: (blocks, 2, D) partial dw
  int hb, nhb;                                     // heads a thread walks, groups of them
};

__device__ __forceinline__ void turn(float pos, float freq, float& c, float& s) {
  const double rev = (double)pos * (double)freq * 0.15915494309189533577;
  const float f = (float)(rev - rint(rev));
  sincospif(2.0f * f, &s, &c);
}

template <typename T>
__device__ __forceinline__ void load8(const T* __restrict__ p, float v[8]) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    T t[8];
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    __builtin_memcpy(t, &a, 16);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)t[i];
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float v[8]) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    T t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = (T)v[i];
    uint4 a;
    __builtin_memcpy(&a, t, 16);
    *reinterpret_cast<uint4*>(p) = a;
  }
}

// rotation of a thread's eight features (sgn +1: forward, -1: transpose); LP lanes hold one head
struct Rot {
  float c[8], s[8];                                // half layout: one pair member each; interleaved: pairs in [0, 4)
  int src;                                         // lane that holds the other members (half layout), -1: no rotation here
  __device__ __forceinline__ void init(const Args& a, int64_t row, int ch, int lane, int lp) {
    src = -1;
    if (a.P == 0) return;
    const float* pos = a.pos + row * a.pos_ld;
    const int d = ch * 8;
    if (a.interleaved) {
      if (d >= 2 * a.P) return;
      src = lane;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int p = d / 2 + i;
        turn(pos[p / a.per_axis], a.freq[p], c[i], s[i]);
      }
    } else {
      const bool first = d < a.P;
      if (d >= 2 * a.P) return;
      src = first ? lane + a.P / 8 : lane - a.P / 8;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int p = (first ? d : d - a.P) + i;
        turn(pos[p / a.per_axis], a.freq[p], c[i], s[i]);
        if (first) s[i] = -s[i];                   // a cos - b sin  |  b cos + a sin
      }
    }
  }
  __device__ __forceinline__ void apply(const Args& a, float v[8], float sgn, int lane) const {
    if (a.P == 0) return;
    if (a.interleaved) {
      if (src >= 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x = v[2 * i], y = v[2 * i + 1], sn = sgn * s[i];
          v[2 * i] = x * c[i] - y * sn;
          v[2 * i + 1] = x * sn + y * c[i];
        }
      }
    } else {
      float o[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = __shfl(v[i], src < 0 ? lane : src, 64);
      if (src >= 0) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = v[i] * c[i] + sgn * s[i] * o[i];
      }
    }
  }
};

template <int LP>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = LP / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// D a multiple of 8, LP = lanes of a head (a power of two >= D / 8), rows 16-byte aligned
template <typename T, int LP, bool BWD>
__global__ void __launch_bounds__(256) rows_kernel(Args a) {
  constexpr int GROUPS = 256 / LP;
  __shared__ float red[BWD ? 256 * 8 : 1];
  const int lane = threadIdx.x & 63, ch = threadIdx.x % LP, grp = threadIdx.x / LP, nh = a.nh1 + a.nh2;
  const bool on = ch * 8 < a.D;
  const float inv_d = 1.0f / (float)a.D;
  float w[2][8], dw[2][8];
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float* p = j ? a.w2 : a.w1;
      w[j][i] = on ? (p ? p[ch * 8 + i] : 1.0f) : 0.0f;
      dw[j][i] = 0.0f;
    }
  const int64_t items = a.M * a.nhb;
  for (int64_t it = (int64_t)blockIdx.x * GROUPS + grp; it < (items + GROUPS - 1) / GROUPS * GROUPS; it += (int64_t)gridDim.x * GROUPS) {
    // the whole workgroup leaves the loop together: groups past the end idle through their last turn
    const bool live = it < items && on;
    const int64_t row = it < items ? it / a.nhb : 0;
    const int h0 = it < items ? (int)(it - row * a.nhb) * a.hb : 0, h1 = min(nh, h0 + a.hb);
    Rot rot;
    rot.init(a, row, ch, lane, LP);
    const T* xp = (const T*)a.x + row * a.x_ld + ch * 8;
    const T* gp = BWD ? (const T*)a.dy + row * a.dy_ld + ch * 8 : nullptr;
    T* yp = (T*)a.y + row * a.y_ld + ch * 8;
    for (int h = h0; h < h1; ++h) {
      const int j = h >= a.nh1;
      float x[8] = {0, 0, 0, 0, 0, 0, 0, 0}, g[8] = {0, 0, 0, 0, 0, 0, 0, 0};
      if (live) {
        load8<T>(xp + (int64_t)h * a.D, x);
        if constexpr (BWD) load8<T>(gp + (int64_t)h * a.D, g);
      }
      float ss = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
      ss = group_sum<LP>(ss);
      const float r = 1.0f / sqrtf(fmaf(ss, inv_d, a.eps));
      if constexpr (!BWD) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = x[i] * r * (j ? w[1][i] : w[0][i]);
        rot.apply(a, x, 1.0f, lane);
        if (live) store8<T>(yp + (int64_t)h * a.D, x);
      } else {
        rot.apply(a, g, -1.0f, lane);
        float dot = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float xr = x[i] * r, t = g[i] * xr;
          dw[0][i] += j ? 0.0f : t;
          dw[1][i] += j ? t : 0.0f;
          g[i] *= j ? w[1][i] : w[0][i];
          x[i] = xr;
          dot = fmaf(g[i], xr, dot);
        }
        dot = group_sum<LP>(dot) * inv_d;
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] = r * (g[i] - x[i] * dot);
        if (live) store8<T>(yp + (int64_t)h * a.D, g);
      }
    }
  }
  if constexpr (BWD) {                             // groups of the workgroup -> one partial sum a feature, in a fixed order
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 8; ++i) red[grp * (LP * 8) + ch * 8 + i] = dw[j][i];
      __syncthreads();
      for (int d = threadIdx.x; d < a.D; d += 256) {
        float s = 0.0f;
        for (int q = 0; q < GROUPS; ++q) s += red[q * (LP * 8) + d];
        a.part[((int64_t)blockIdx.x * 2 + j) * a.D + d] = s;
      }
    }
  }
}

// any D <= 256, any alignment: one wave per (row, head), the rotation through LDS
template <typename T, bool BWD>
__global__ void __launch_bounds__(256) any_kernel(Args a) {
  __shared__ float buf[4][256];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, nh = a.nh1 + a.nh2;
  const float inv_d = 1.0f / (float)a.D;
  float dw[2][4] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
  const int64_t items = a.M * nh;
  for (int64_t it = (int64_t)blockIdx.x * 4 + wave; it < (items + 3) / 4 * 4; it += (int64_t)gridDim.x * 4) {
    const bool live = it < items;
    const int64_t row = live ? it / nh : 0;
    const int h = live ? (int)(it - row * nh) : 0, j = h >= a.nh1;
    const T* xp = (const T*)a.x + row * a.x_ld + (int64_t)h * a.D;
    const T* gp = BWD ? (const T*)a.dy + row * a.dy_ld + (int64_t)h * a.D : nullptr;
    const float* w = j ? a.w2 : a.w1;
    float x[4], v[4], wv[4], ss = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = lane + 64 * i;
      const bool in = live && d < a.D;
      x[i] = in ? (float)xp[d] : 0.0f;
      wv[i] = in ? (w ? w[d] : 1.0f) : 0.0f;
      v[i] = BWD ? (in ? (float)gp[d] : 0.0f) : 0.0f;
      ss = fmaf(x[i], x[i], ss);
    }
    ss = wave_sum(ss);
    const float r = 1.0f / sqrtf(fmaf(ss, inv_d, a.eps));
    if constexpr (!BWD) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = x[i] * r * wv[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (lane + 64 * i < a.D) buf[wave][lane + 64 * i] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = lane + 64 * i;
      if (d < 2 * a.P) {
        const int p = a.interleaved ? d >> 1 : (d < a.P ? d : d - a.P);
        const bool second = a.interleaved ? (d & 1) : d >= a.P;
        const int o = a.interleaved ? d ^ 1 : (second ? d - a.P : d + a.P);
        float c, s;
        turn(a.pos[row * a.pos_ld + p / a.per_axis], a.freq[p], c, s);
        if (!second) s = -s;
        if (BWD) s = -s;
        v[i] = v[i] * c + s * buf[wave][o];
      }
    }
    if constexpr (BWD) {
      float dot = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float xr = x[i] * r, t = v[i] * xr;
        dw[0][i] += j ? 0.0f : t;
        dw[1][i] += j ? t : 0.0f;
        v[i] *= wv[i];
        x[i] = xr;
        dot = fmaf(v[i], xr, dot);
      }
      dot = wave_sum(dot) * inv_d;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = r * (v[i] - x[i] * dot);
    }
    T* yp = (T*)a.y + row * a.y_ld + (int64_t)h * a.D;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (live && lane + 64 * i < a.D) yp[lane + 64 * i] = (T)v[i];
  }
  if constexpr (BWD) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 4; ++i) buf[wave][lane + 64 * i] = dw[j][i];
      __syncthreads();
      if (threadIdx.x < a.D)
        a.part[((int64_t)blockIdx.x * 2 + j) * a.D + threadIdx.x] =
            buf[0][threadIdx.x] + buf[1][threadIdx.x] + buf[2][threadIdx.x] + buf[3][threadIdx.x];
    }
  }
}

// dw[j][d] = sum over blocks of part[block][j][d]; a wave per (j, d) column
__global__ void __launch_bounds__(256) fold_kernel(int blocks, int D, const float* __restrict__ part, float* __restrict__ dw1,
                                                   float* __restrict__ dw2) {
  const int col = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (col >= 2 * D) return;
  float s = 0.0f;
  for (int b = lane; b < blocks; b += 64) s += part[(int64_t)b * 2 * D + col];
  s = wave_sum(s);
  float* dst = col < D ? dw1 : dw2;
  if (lane == 0 && dst) dst[col < D ? col : col - D] = s;
}

static bool aligned16(const void* p, int64_t ld, int es) { return ((uintptr_t)p & 15) == 0 && ld * es % 16 == 0; }

template <typename T, bool BWD>
static int launch(Args& a, float* dw1, float* dw2, hipStream_t st, const char* who) {
  const int es = sizeof(T), nh = a.nh1 + a.nh2;
  const bool rot_ok = a.P == 0 || (a.interleaved ? a.P % 4 == 0 : a.P % 8 == 0);
  const bool vec = a.D % 8 == 0 && rot_ok && aligned16(a.x, a.x_ld, es) && aligned16(a.y, a.y_ld, es) &&
                   (!BWD || aligned16(a.dy, a.dy_ld, es));
  int blocks;
  if (vec) {
    const int l = a.D / 8, lp = l <= 1 ? 1 : l <= 2 ? 2 : l <= 4 ? 4 : l <= 8 ? 8 : l <= 16 ? 16 : 32;
    // heads a thread walks: all of a row when the rows alone give every CU four workgroups (the angles are then computed
    // once a row), fewer when there are few rows
    const int64_t row_threads = a.M * lp, want = 256 * 4 * 256;
    a.nhb = 1;
    if (row_threads < want) a.nhb = (int)((want + row_threads - 1) / row_threads);
    if (a.nhb > nh) a.nhb = nh;
    a.hb = (nh + a.nhb - 1) / a.nhb;
    a.nhb = (nh + a.hb - 1) / a.hb;
    const int64_t groups = 256 / lp, need = (a.M * a.nhb + groups - 1) / groups;
    const int cap = BWD ? kMaxBlocks : 256 * 16;
    blocks = (int)(need < cap ? need : cap);
    switch (lp) {
      case 1: rows_kernel<T, 1, BWD><<<blocks, 256, 0, st>>>(a); break;
      case 2: rows_kernel<T, 2, BWD><<<blocks, 256, 0, st>>>(a); break;
      case 4: rows_kernel<T, 4, BWD><<<blocks, 256, 0, st>>>(a); break;
      case 8: rows_kernel<T, 8, BWD><<<blocks, 256, 0, st>>>(a); break;
      case 16: rows_kernel<T, 16, BWD><<<blocks, 256, 0, st>>>(a); break;
      default: rows_kernel<T, 32, BWD><<<blocks, 256, 0, st>>>(a); break;
    }
  } else {
    const int64_t need = (a.M * nh + 3) / 4;
    blocks = (int)(need < kMaxBlocks ? need : kMaxBlocks);
    any_kernel<T, BWD><<<blocks, 256, 0, st>>>(a);
  }
  int rc = check_launch(who);
  if (rc == MMB_OK && BWD) {
    fold_kernel<<<(2 * a.D + 3) / 4, 256, 0, st>>>(blocks, a.D, a.part, dw1, dw2);
    rc = check_launch(who);
  }
  return rc;
}

static int check(const char* who, int64_t M, int nh1, int nh2, int D, int dtype, const void* x, int64_t x_ld, const void* y, int64_t y_ld,
                 float eps, const float* pos, int64_t pos_ld, int n_axes, const float* freq, int P, int interleaved) {
  MMB_REQUIRE(M > 0 && nh1 > 0 && nh2 >= 0, "%s: M and nheads must be positive, nheads2 >= 0 (got %lld, %d, %d)", who, (long long)M, nh1, nh2);
  MMB_REQUIRE(D > 0 && D <= 256, "%s: head width must be 1..256 (got %d)", who, D);
  MMB_REQUIRE(dtype == MMB_DT_F32 || dtype == MMB_DT_BF16 || dtype == MMB_DT_F16, "%s: unknown dtype %d", who, dtype);
  MMB_REQUIRE(x && y, "%s: NULL rows", who);
  MMB_REQUIRE((int64_t)nh1 + nh2 <= (1 << 20) && x_ld >= (int64_t)(nh1 + nh2) * D && y_ld >= (int64_t)(nh1 + nh2) * D,
              "%s: a leading dimension is smaller than its row", who);
  MMB_REQUIRE(eps > 0.0f, "%s: eps must be positive", who);
  MMB_REQUIRE(P >= 0 && 2 * P <= D, "%s: %d rotated pairs do not fit a head of %d", who, P, D);
  MMB_REQUIRE(P == 0 || (pos && freq && n_axes > 0 && P % n_axes == 0 && pos_ld >= n_axes),
              "%s: %d pairs need pos, freq and a number of coordinates that divides them (got %d)", who, P, n_axes);
  MMB_REQUIRE(interleaved == 0 || interleaved == 1, "%s: unknown layout %d", who, interleaved);
  return MMB_OK;
}

// y over x (dx over x or dy) row by row is fine: a head is read whole before it is written.  Shifted by anything it is not.
static Region other_than(const Region& r, const Region& y) {
  return r.at == y.at && (r.ld == y.ld || r.rows == 1) ? Region{} : r;
}

}  // namespace headnorm
}  // namespace mmb

using namespace mmb;
using namespace mmb::headnorm;

extern "C" int mmb_head_norm_rotate_fwd(int64_t M, int nheads, int nheads2, int D, int dtype, const void* x, int64_t x_ld,
                                        const float* weight, const float* weight2, float eps, const float* pos, int64_t pos_ld,
                                        int n_axes, const float* freq, int n_pairs, int interleaved, void* y, int64_t y_ld,
                                        void* stream) {
  if (int rc = check("mmb_head_norm_rotate_fwd", M, nheads, nheads2, D, dtype, x, x_ld, y, y_ld, eps, pos, pos_ld, n_axes, freq,
                     n_pairs, interleaved))
    return rc;
  Args a = {M, nheads, nheads2, D, n_pairs, n_pairs ? n_pairs / n_axes : 1, interleaved, x, nullptr, weight, weight2, pos, freq,
            x_ld, 0, pos_ld, y_ld, eps, y, nullptr, 0, 0};
  hipStream_t st = as_stream(stream);
  const char* who = "mmb_head_norm_rotate_fwd";
  const int es = dtype == MMB_DT_F32 ? 4 : 2;
  const int64_t w = (int64_t)(nheads + nheads2) * D;
  const Region ry = row_region(y, M, w, y_ld, es);
  const Region ins[] = {other_than(row_region(x, M, w, x_ld, es), ry), flat_region(weight, 4 * D), flat_region(weight2, 4 * D),
                        row_region(n_pairs ? pos : nullptr, M, n_axes, pos_ld, 4), flat_region(n_pairs ? freq : nullptr, 4 * n_pairs)};
  if (int rc = check_apart(who, &ry, 1, ins, 5)) return rc;
  if (dtype == MMB_DT_F32) return launch<float, false>(a, nullptr, nullptr, st, who);
  if (dtype == MMB_DT_BF16) return launch<__bf16, false>(a, nullptr, nullptr, st, who);
  return launch<_Float16, false>(a, nullptr, nullptr, st, who);
}

extern "C" int mmb_head_norm_rotate_bwd(int64_t M, int nheads, int nheads2, int D, int dtype, const void* x, int64_t x_ld,
                                        const void* dy, int64_t dy_ld, const float* weight, const float* weight2, float eps,
                                        const float* pos, int64_t pos_ld, int n_axes, const float* freq, int n_pairs,
                                        int interleaved, void* dx, int64_t dx_ld, float* dweight, float* dweight2, float* partials,
                                        void* stream) {
  const char* who = "mmb_head_norm_rotate_bwd";
  if (int rc = check(who, M, nheads, nheads2, D, dtype, x, x_ld, dx, dx_ld, eps, pos, pos_ld, n_axes, freq, n_pairs, interleaved)) return rc;
  MMB_REQUIRE(dy && dy_ld >= (int64_t)(nheads + nheads2) * D, "%s: dy is NULL or its leading dimension smaller than its row", who);
  MMB_REQUIRE(partials, "%s: partials is NULL (2 * D * MMB_HEAD_NORM_MAX_BLOCKS floats)", who);
  Args a = {M, nheads, nheads2, D, n_pairs, n_pairs ? n_pairs / n_axes : 1, interleaved, x, dy, weight, weight2, pos, freq,
            x_ld, dy_ld, pos_ld, dx_ld, eps, dx, partials, 0, 0};
  hipStream_t st = as_stream(stream);
  const int es = dtype == MMB_DT_F32 ? 4 : 2;
  const int64_t w = (int64_t)(nheads + nheads2) * D;
  const Region outs[] = {row_region(dx, M, w, dx_ld, es), flat_region(dweight, 4 * D), flat_region(dweight2, 4 * D),
                         flat_region(partials, (int64_t)2 * D * kMaxBlocks * 4)};
  const Region rx = row_region(x, M, w, x_ld, es), rdy = row_region(dy, M, w, dy_ld, es);
  const Region fixed[] = {flat_region(weight, 4 * D), flat_region(weight2, 4 * D), row_region(n_pairs ? pos : nullptr, M, n_axes, pos_ld, 4),
                          flat_region(n_pairs ? freq : nullptr, 4 * n_pairs)};
  const Region of_dx[] = {other_than(rx, outs[0]), other_than(rdy, outs[0])}, of_sums[] = {rx, rdy};
  if (int rc = check_apart(who, outs, 4, fixed, 4)) return rc;
  if (int rc = check_apart(who, outs, 1, of_dx, 2)) return rc;
  if (int rc = check_apart(who, outs + 1, 3, of_sums, 2)) return rc;
  if (dtype == MMB_DT_F32) return launch<float, true>(a, dweight, dweight2, st, who);
  if (dtype == MMB_DT_BF16) return launch<__bf16, true>(a, dweight, dweight2, st, who);
  return launch<_Float16, true>(a, dweight, dweight2, st, who);
}
