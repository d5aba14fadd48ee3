// Rotary positions with several axes (time, height, width of image and video tokens).
//
// Pair p of a head belongs to axis(p) and turns by  angle(row, p) = pos[row][axis(p)] * f(p)  -- f(p) = theta^(-j / n) with (j, n) = the
// pair's place in its axis's section and that section's size (every axis its own ladder), or (p, all pairs) (joint: one ladder
// shared by the axes).  (a, b) -> (a cos - b sin, a sin + b cos); the inverse (= the gradient) turns by -angle.
// HBM-bound: a row is read and written once.  The angles of a row are formed once per block and used by all of its heads.  25088 rows of 24 heads of 64, bf16
// (154 MB): 33 us, 4.6 TB/s; 4111 rows of 12 heads of 80, fp32 (32 MB, in cache): 10.5 us; 32 rows of 20 heads of 128: 3.9 us, a launch and one chain of
// loads.  A far position
// times a frequency does not fit 32 bits (position 10^6: an angle off by 0.03), so the product is formed in 64 bits, in
// TURNS, its whole part dropped, and only the fraction goes on in 32 bits.
#include "dh_common.h"
#include <math.h>

namespace {

constexpr int MAX_PAIRS = DH_ROPE_MAX_PAIRS;
struct RopeP {
  const void* x;
  void* y;
  const void* pos;
  long ldx, ldy;
  int rows, pos_rows, axes, heads, hd, pairs, interleaved, frac;
  float sign;
  double f[MAX_PAIRS];                 // turns per unit of position
  unsigned char axis[MAX_PAIRS];
};

// V elements as floats
template <typename T, int V> __device__ __forceinline__ void ldv(const T* p, float* o) {
  if constexpr (V == 8) ld8(p, o);
  else if constexpr (V == 4 && sizeof(T) == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    o[0] = __uint_as_float(v.x << 16); o[1] = __uint_as_float(v.x & 0xffff0000u); o[2] = __uint_as_float(v.y << 16); o[3] = __uint_as_float(v.y & 0xffff0000u);
  } else if constexpr (V == 4) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    o[0] = v.x; o[1] = v.y; o[2] = v.z; o[3] = v.w;
  } else o[0] = ld<T>(p);
}
template <typename T, int V> __device__ __forceinline__ void stv(T* p, const float* o) {
  if constexpr (V == 8) st8_fast(p, o);
  else if constexpr (V == 4 && sizeof(T) == 2) {
    uint2 w;
    w.x = pack2bf_hw(o[0], o[1]); w.y = pack2bf_hw(o[2], o[3]);
    *reinterpret_cast<uint2*>(p) = w;
  } else if constexpr (V == 4) *reinterpret_cast<float4*>(p) = make_float4(o[0], o[1], o[2], o[3]);
  else st<T>(p, o[0]);
}

// R rows per block and round; V pairs per task (V divides the pairs and what is left of a head)
template <typename T, int V>
__global__ __launch_bounds__(256) void rope_kernel(RopeP p, int R) {
  DH_DYN_LDS_A16(float2, cs);                          // [R][pairs] (cos, sin)
  const int tid = threadIdx.x;
  const int rot = p.pairs / V, rest = (p.hd - 2 * p.pairs) / V, per_head = rot + rest, per_row = p.heads * per_head;
  for (long r0 = (long)blockIdx.x * R; r0 < p.rows; r0 += (long)gridDim.x * R) {
    const int n = (int)min((long)R, p.rows - r0);
    __syncthreads();                                   // the round before is done with the table
    for (int i = tid; i < n * p.pairs; i += 256) {
      const int r = i / p.pairs, k = i - r * p.pairs;
      const long at = (long)((int)(r0 + r) % p.pos_rows) * p.axes + p.axis[k];
      const double pos = p.frac ? (double)((const float*)p.pos)[at] : (double)((const int*)p.pos)[at];
      const double turns = pos * p.f[k];
      const float u = 2.f * (float)(turns - rint(turns));
      cs[i] = make_float2(cospif(u), p.sign * sinpif(u));
    }
    __syncthreads();
    for (int i = tid; i < n * per_row; i += 256) {
      const int r = i / per_row, j = i - r * per_row, head = j / per_head, c = j - head * per_head;
      const T* x = (const T*)p.x + (r0 + r) * p.ldx + (long)head * p.hd;
      T* y = (T*)p.y + (r0 + r) * p.ldy + (long)head * p.hd;
      float a[V], b[V], oa[V], ob[V];
      if (c >= rot) {                                  // behind the rotary part
        const int e = 2 * p.pairs + (c - rot) * V;
        ldv<T, V>(x + e, a);
        stv<T, V>(y + e, a);
        continue;
      }
      const float2* t = cs + r * p.pairs + c * V;
      if (p.interleaved) {
        float z[2 * V], o[2 * V];
        ldv<T, V>(x + 2 * c * V, z);
        ldv<T, V>(x + 2 * c * V + V, z + V);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          o[2 * e] = z[2 * e] * t[e].x - z[2 * e + 1] * t[e].y;
          o[2 * e + 1] = z[2 * e] * t[e].y + z[2 * e + 1] * t[e].x;
        }
        stv<T, V>(y + 2 * c * V, o);
        stv<T, V>(y + 2 * c * V + V, o + V);
      } else {
        ldv<T, V>(x + c * V, a);
        ldv<T, V>(x + p.pairs + c * V, b);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          oa[e] = a[e] * t[e].x - b[e] * t[e].y;
          ob[e] = a[e] * t[e].y + b[e] * t[e].x;
        }
        stv<T, V>(y + c * V, oa);
        stv<T, V>(y + p.pairs + c * V, ob);
      }
    }
  }
}

template <typename T>
int rope_launch(const RopeP& p, hipStream_t st) {
  // elements per access: what the pairs, the rest of a head, the row strides and the addresses allow
  auto fits = [&](int v) {
    const int bytes = v * (int)sizeof(T) > 16 ? 16 : v * (int)sizeof(T);
    return p.pairs % v == 0 && (p.hd - 2 * p.pairs) % v == 0 && p.hd % v == 0 && p.ldx % v == 0 && p.ldy % v == 0 && ((uintptr_t)p.x % bytes) == 0 &&
           ((uintptr_t)p.y % bytes) == 0;
  };
  const int v = fits(8) ? 8 : fits(4) ? 4 : 1;
  // rows per round: as many as give every thread one angle to form (the table of a round costs two barriers)
  int R = 256 / p.pairs < 1 ? 1 : 256 / p.pairs;
  if (R > 8) R = 8;
  while (R > 1 && dh_cdiv(p.rows, R) < 512) R /= 2;       // few rows: one each, spread over the chip
  int grid = dh_cdiv(p.rows, R);
  if (grid > 2048) grid = 2048;
  const size_t lds = (size_t)R * p.pairs * sizeof(float2);
  if (v == 8) hipLaunchKernelGGL((rope_kernel<T, 8>), dim3(grid), dim3(256), lds, st, p, R);
  else if (v == 4) hipLaunchKernelGGL((rope_kernel<T, 4>), dim3(grid), dim3(256), lds, st, p, R);
  else hipLaunchKernelGGL((rope_kernel<T, 1>), dim3(grid), dim3(256), lds, st, p, R);
  DH_CHECK_LAUNCH();
  return DH_OK;
}

}  // namespace

extern "C" int dh_rope_plan_init(dh_rope_plan* plan, int hd, const int* sections, const double* theta, int axes, int joint, int interleaved) {
  DH_REQUIRE(plan && sections && theta, "dh_rope_plan_init: null pointer");
  DH_REQUIRE(hd > 0 && axes > 0 && axes <= 8, "dh_rope_plan_init: head size %d, %d axes (up to 8)", hd, axes);
  int64_t pairs = 0;
  for (int a = 0; a < axes; ++a) {
    DH_REQUIRE(sections[a] > 0 && sections[a] <= MAX_PAIRS, "dh_rope_plan_init: section %d of axis %d", sections[a], a);
    DH_REQUIRE(theta[a] > 0. && theta[a] < INFINITY, "dh_rope_plan_init: theta of axis %d must be positive and finite", a);
    DH_REQUIRE(!joint || theta[a] == theta[0], "dh_rope_plan_init: a joint ladder has one theta");
    pairs += sections[a];
  }
  DH_REQUIRE(pairs <= MAX_PAIRS && 2 * pairs <= hd, "dh_rope_plan_init: %lld pairs in a head of %d", (long long)pairs, hd);
  plan->axes = axes; plan->pairs = (int)pairs; plan->hd = hd; plan->interleaved = interleaved != 0;
  int k = 0;
  for (int a = 0; a < axes; ++a)
    for (int j = 0; j < sections[a]; ++j, ++k) {
      const double e = joint ? (double)k / (double)pairs : (double)j / (double)sections[a];
      plan->turns[k] = pow(theta[a], -e) / 6.283185307179586476925286766559;
      plan->axis[k] = (unsigned char)a;
    }
  return DH_OK;
}

extern "C" int dh_rope_axes(const dh_rope_plan* plan, int dtype, const void* x, int64_t ldx, void* y, int64_t ldy, int rows, int heads, const void* pos,
                            int pos_float, int pos_rows, int inverse, dh_stream_t stream) {
  DH_REQUIRE(plan && plan->axes > 0 && plan->axes <= 8 && plan->pairs > 0 && plan->pairs <= MAX_PAIRS && plan->hd >= 2 * plan->pairs, "dh_rope_axes: plan not initialised");
  DH_REQUIRE(dtype == DH_F32 || dtype == DH_BF16, "dh_rope_axes: dtype %d", dtype);
  DH_REQUIRE(rows >= 0 && rows < (1 << 30) && heads > 0, "dh_rope_axes: rows %d (below 2^30), heads %d", rows, heads);
  const int64_t width = (int64_t)heads * plan->hd;
  DH_REQUIRE(width < (1 << 27) && (rows <= 1 || (ldx >= width && ldy >= width)), "dh_rope_axes: row strides %lld, %lld for %d heads of %d", (long long)ldx, (long long)ldy, heads, plan->hd);
  if (rows == 0) return DH_OK;
  DH_REQUIRE(x && y && pos && pos_rows > 0 && rows % pos_rows == 0, "dh_rope_axes: %d rows, %d positions", rows, pos_rows);
  RopeP p;
  p.x = x; p.y = y; p.pos = pos; p.ldx = ldx; p.ldy = ldy;
  p.rows = rows; p.pos_rows = pos_rows; p.axes = plan->axes; p.heads = heads; p.hd = plan->hd; p.pairs = plan->pairs; p.interleaved = plan->interleaved; p.frac = pos_float;
  p.sign = inverse ? -1.f : 1.f;
  for (int k = 0; k < p.pairs; ++k) {
    DH_REQUIRE(plan->axis[k] < plan->axes, "dh_rope_axes: plan not initialised");
    p.f[k] = plan->turns[k];
    p.axis[k] = plan->axis[k];
  }
  return dtype == DH_BF16 ? rope_launch<bf16_t>(p, (hipStream_t)stream) : rope_launch<float>(p, (hipStream_t)stream);
}
