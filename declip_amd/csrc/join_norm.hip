// The boundary of a residual block in one pass: the norm behind the block, its gate and residual scale, the residual sum and the
// norm in front of the next block.
//
//   p = N_post(y) (or y);   t = scale[c] * g * p;   x' = alpha x + t;   n = N_pre(x')
//   N(z) = (z - mean) rstd w + b, or without mean and b (rms);   g = gate or tanh(gate): per group of rows, or per group and channel
//
//   G = dx' + N_pre'(dn);   dx = alpha G;   dp = G scale g;   dy = N_post'(dp)
//   with A[c] = sum_rows G g yhat, B[c] = sum_rows G g:   dpost_w = scale A, dpost_b = scale B, dscale = w A + b B;
//   C[c] = sum dn xhat = dpre_w, E[c] = sum dn = dpre_b;   dgate = the same sums per group (channel gate) or sum_c G scale p (row gate)
//
// HBM-bound: the forward reads x, y and writes x', n; the backward reads x, y, dx', dn, recomputes p, x', xhat from the rows' saved statistics
// (in fp32, the forward's own values) and writes dx, dy.  A row lives in the registers of one wave (d <= 1024) or of one block, statistics
// are fp32 and two-pass (mean first).  The column sums stay in registers over a block's rows, go to a partial row per block, and are
// added in a fixed order by a second small kernel: no atomics, the same result on every run.
#include "dh_common.h"
#include <initializer_list>

namespace {

struct JP {
  const void *x, *y, *dxo, *dn;
  void *x_out, *n, *dx, *dy;
  const float *post_w, *post_b, *gate, *scale, *pre_w, *pre_b;
  float* stats;                                  // [4][rows]: mean, rstd behind the block; mean, rstd in front of the next
  float *part, *rowdot;                          // backward: [blocks][4][d]; [rows]
  float *d_post_w, *d_post_b, *d_gate, *d_scale, *d_pre_w, *d_pre_b;
  float alpha, eps;
  int rows, d, groups, channel, rms, gate_tanh, pre;   // rows / groups rows share a gate value (row gate) or vector (channel gate)
  int per_group;                                 // blocks per group (channel gate): a block's rows lie in one group
};

__device__ __forceinline__ float act(const JP& p, float g) { return p.gate_tanh ? tanhf(g) : g; }

// sum over the waves that hold a row (W waves; block = 4 waves = 4 / W rows at a time)
template <int W> __device__ __forceinline__ void row_sum2(float& a, float& b, float* red) {
  a = wave_sum_fast(a);
  b = wave_sum_fast(b);
  if (W > 1) {
    const int wave = threadIdx.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) { red[2 * wave] = a; red[2 * wave + 1] = b; }
    __syncthreads();
    a = red[0] + red[2] + red[4] + red[6];
    b = red[1] + red[3] + red[5] + red[7];
  }
}

// V elements per lane and chunk (8: 16-byte accesses of bf16; 1: any d and alignment), NC chunks in registers
template <typename T, int V> __device__ __forceinline__ void ldn(const T* p, float* o) {
  if constexpr (V == 8) ld8(p, o); else o[0] = ld<T>(p);
}
template <typename T, int V> __device__ __forceinline__ void stn(T* p, const float* o) {
  if constexpr (V == 8) st8_fast(p, o); else st<T>(p, o[0]);
}

// column of chunk k of this lane
template <int W, int V> __device__ __forceinline__ int col_of(int k) {
  const int w = W == 1 ? 0 : (threadIdx.x >> 6);
  return ((threadIdx.x & 63) + 64 * (w + W * k)) * V;
}

// ------------------------------------------------------------------------------------------ forward
template <typename T, int W, int NC, int V>
__global__ __launch_bounds__(256) void join_fwd_kernel(JP p) {
  __shared__ float red[8];
  constexpr int RB = 4 / W;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, d = p.d;
  const T *x = (const T*)p.x, *y = (const T*)p.y;
  const int rows_per_gate = p.rows / p.groups;
  const float inv_d = 1.f / d;
  for (int row0 = blockIdx.x * RB; row0 < p.rows; row0 += gridDim.x * RB) {
    const int row = row0 + (W == 1 ? wave : 0);
    const bool live = row < p.rows;
    const long at = (long)(live ? row : 0) * d;
    float yv[NC][V], xv[NC][V];
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int c = col_of<W, V>(k);
#pragma unroll
      for (int e = 0; e < V; ++e) xv[k][e] = yv[k][e] = 0.f;
      if (live && c < d) { ldn<T, V>(y + at + c, yv[k]); ldn<T, V>(x + at + c, xv[k]); }
    }
    float g = 1.f;
    const int grp = live ? row / rows_per_gate : 0;
    if (p.gate && !p.channel) g = act(p, p.gate[grp]);
    float mu = 0.f, rs = 1.f;
    if (p.post_w) {
      float s = 0.f, zero = 0.f;
      if (!p.rms) {
#pragma unroll
        for (int k = 0; k < NC; ++k)
#pragma unroll
          for (int e = 0; e < V; ++e) s += yv[k][e];
        row_sum2<W>(s, zero, red);
        mu = s * inv_d;
      }
      float q = 0.f;
#pragma unroll
      for (int k = 0; k < NC; ++k)
        if (col_of<W, V>(k) < d)
#pragma unroll
          for (int e = 0; e < V; ++e) { const float u = yv[k][e] - mu; q = fmaf(u, u, q); }
      row_sum2<W>(q, zero, red);
      rs = 1.f / sqrtf(q * inv_d + p.eps);
      if (live && lane == 0 && (W == 1 || wave == 0)) { p.stats[row] = mu; p.stats[p.rows + row] = rs; }
    }
    float s = 0.f, zero = 0.f;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int c = col_of<W, V>(k);
      if (c < d) {
        float w[V], b[V], sc[V], gc[V];
#pragma unroll
        for (int e = 0; e < V; ++e) { w[e] = sc[e] = 1.f; b[e] = 0.f; gc[e] = g; }
        if (p.post_w) ldn<float, V>(p.post_w + c, w);
        if (p.post_b) ldn<float, V>(p.post_b + c, b);
        if (p.scale) ldn<float, V>(p.scale + c, sc);
        if (p.gate && p.channel) {
          ldn<float, V>(p.gate + (long)grp * d + c, gc);
#pragma unroll
          for (int e = 0; e < V; ++e) gc[e] = act(p, gc[e]);
        }
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float pv = fmaf((yv[k][e] - mu) * rs, w[e], b[e]);
          xv[k][e] = fmaf(p.alpha, xv[k][e], sc[e] * gc[e] * pv);
          s += xv[k][e];
        }
        if (live) stn<T, V>((T*)p.x_out + at + c, xv[k]);
      }
    }
    if (!p.pre) continue;
    float mu2 = 0.f;
    if (!p.rms) {
      row_sum2<W>(s, zero, red);
      mu2 = s * inv_d;
    }
    float q = 0.f;
#pragma unroll
    for (int k = 0; k < NC; ++k)
      if (col_of<W, V>(k) < d)
#pragma unroll
        for (int e = 0; e < V; ++e) { const float u = xv[k][e] - mu2; q = fmaf(u, u, q); }
    row_sum2<W>(q, zero, red);
    const float rs2 = 1.f / sqrtf(q * inv_d + p.eps);
    if (live && lane == 0 && (W == 1 || wave == 0)) { p.stats[2 * (long)p.rows + row] = mu2; p.stats[3 * (long)p.rows + row] = rs2; }
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int c = col_of<W, V>(k);
      if (c < d && live) {
        float w[V], b[V], o[V];
        ldn<float, V>(p.pre_w + c, w);
#pragma unroll
        for (int e = 0; e < V; ++e) b[e] = 0.f;
        if (p.pre_b) ldn<float, V>(p.pre_b + c, b);
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = fmaf((xv[k][e] - mu2) * rs2, w[e], b[e]);
        stn<T, V>((T*)p.n + at + c, o);
      }
    }
  }
}

// ------------------------------------------------------------------------------------------ backward
template <typename T, int W, int NC, int V>
__global__ __launch_bounds__(256) void join_bwd_kernel(JP p) {
  DH_DYN_LDS_A16(float, sm);                      // W == 1: [4][d] for the waves' column sums
  __shared__ float red[8];
  constexpr int RB = 4 / W;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, d = p.d;
  const T *x = (const T*)p.x, *y = (const T*)p.y, *dxo = (const T*)p.dxo, *dn = (const T*)p.dn;
  const int rows_per_gate = p.rows / p.groups;
  const float inv_d = 1.f / d;
  int first, last, step;
  if (p.channel) {                                // blocks of group blockIdx / per_group
    const int g = blockIdx.x / p.per_group;
    first = g * rows_per_gate + (blockIdx.x % p.per_group) * RB;
    last = (g + 1) * rows_per_gate;
    step = p.per_group * RB;
  } else {
    first = blockIdx.x * RB; last = p.rows; step = gridDim.x * RB;
  }
  float A[NC][V], B[NC][V], C[NC][V], E[NC][V];
#pragma unroll
  for (int k = 0; k < NC; ++k)
#pragma unroll
    for (int e = 0; e < V; ++e) A[k][e] = B[k][e] = C[k][e] = E[k][e] = 0.f;
  for (int row0 = first; row0 < last; row0 += step) {
    const int row = row0 + (W == 1 ? wave : 0);
    const bool live = row < last;
    const long at = (long)(live ? row : first) * d;
    const int grp = (live ? row : first) / rows_per_gate;
    float g = 1.f, mu = 0.f, rs = 1.f, mu2 = 0.f, rs2 = 1.f;
    if (p.gate && !p.channel) g = act(p, p.gate[grp]);
    const int srow = live ? row : first;
    if (p.post_w) { mu = p.stats[srow]; rs = p.stats[p.rows + srow]; }
    if (p.dn) { mu2 = p.stats[2 * (long)p.rows + srow]; rs2 = p.stats[3 * (long)p.rows + srow]; }
    float yh[NC][V], G[NC][V], xh[NC][V], wn[NC][V];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int c = col_of<W, V>(k);
#pragma unroll
      for (int e = 0; e < V; ++e) yh[k][e] = G[k][e] = xh[k][e] = wn[k][e] = 0.f;
      if (!live || c >= d) continue;
      float w[V], b[V], sc[V], gc[V], xv[V];
#pragma unroll
      for (int e = 0; e < V; ++e) { w[e] = sc[e] = 1.f; b[e] = 0.f; gc[e] = g; }
      ldn<T, V>(y + at + c, yh[k]);
      if (p.dxo) ldn<T, V>(dxo + at + c, G[k]);
#pragma unroll
      for (int e = 0; e < V; ++e) yh[k][e] = (yh[k][e] - mu) * rs;
      if (!p.dn) continue;
      if (p.post_w) ldn<float, V>(p.post_w + c, w);
      if (p.post_b) ldn<float, V>(p.post_b + c, b);
      if (p.scale) ldn<float, V>(p.scale + c, sc);
      if (p.gate && p.channel) {
        ldn<float, V>(p.gate + (long)grp * d + c, gc);
#pragma unroll
        for (int e = 0; e < V; ++e) gc[e] = act(p, gc[e]);
      }
      ldn<T, V>(x + at + c, xv);
      float dnv[V], w2[V];
      ldn<T, V>(dn + at + c, dnv);
      ldn<float, V>(p.pre_w + c, w2);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float xo = fmaf(p.alpha, xv[e], sc[e] * gc[e] * fmaf(yh[k][e], w[e], b[e]));
        xh[k][e] = (xo - mu2) * rs2;
        wn[k][e] = dnv[e] * w2[e];
        s1 += wn[k][e];
        s2 = fmaf(wn[k][e], xh[k][e], s2);
        C[k][e] = fmaf(dnv[e], xh[k][e], C[k][e]);
        E[k][e] += dnv[e];
      }
    }
    if (p.dn) {
      row_sum2<W>(s1, s2, red);
      const float c1 = p.rms ? 0.f : s1 * inv_d, c2 = s2 * inv_d;
#pragma unroll
      for (int k = 0; k < NC; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e) G[k][e] += rs2 * (wn[k][e] - c1 - xh[k][e] * c2);
    }
    float s3 = 0.f, s4 = 0.f, dot = 0.f, zero = 0.f;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int c = col_of<W, V>(k);
      if (!live || c >= d) {
#pragma unroll
        for (int e = 0; e < V; ++e) wn[k][e] = 0.f;
        continue;
      }
      float w[V], b[V], sc[V], gc[V], o[V];
#pragma unroll
      for (int e = 0; e < V; ++e) { w[e] = sc[e] = 1.f; b[e] = 0.f; gc[e] = g; }
      if (p.post_w) ldn<float, V>(p.post_w + c, w);
      if (p.post_b) ldn<float, V>(p.post_b + c, b);
      if (p.scale) ldn<float, V>(p.scale + c, sc);
      if (p.gate && p.channel) {
        ldn<float, V>(p.gate + (long)grp * d + c, gc);
#pragma unroll
        for (int e = 0; e < V; ++e) gc[e] = act(p, gc[e]);
      }
#pragma unroll
      for (int e = 0; e < V; ++e) {
        o[e] = p.alpha * G[k][e];
        const float q = G[k][e] * sc[e];
        dot = fmaf(q, fmaf(yh[k][e], w[e], b[e]), dot);
        const float Gg = p.channel ? G[k][e] : G[k][e] * g;
        A[k][e] = fmaf(Gg, yh[k][e], A[k][e]);
        B[k][e] += Gg;
        wn[k][e] = q * gc[e] * w[e];                // dp w (w = 1 without a norm behind the block)
        s3 += wn[k][e];
        s4 = fmaf(wn[k][e], yh[k][e], s4);
      }
      stn<T, V>((T*)p.dx + at + c, o);
    }
    float c3 = 0.f, c4 = 0.f;
    if (p.post_w) {
      row_sum2<W>(s3, s4, red);
      c3 = p.rms ? 0.f : s3 * inv_d;
      c4 = s4 * inv_d;
    }
    if (p.rowdot) {
      row_sum2<W>(dot, zero, red);
      if (live && lane == 0 && (W == 1 || wave == 0)) p.rowdot[row] = dot;
    }
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int c = col_of<W, V>(k);
      if (!live || c >= d) continue;
      float o[V];
#pragma unroll
      for (int e = 0; e < V; ++e) o[e] = rs * (wn[k][e] - c3 - yh[k][e] * c4);
      stn<T, V>((T*)p.dy + at + c, o);
    }
  }
  if (!p.part) return;
  float* out = p.part + (long)blockIdx.x * 4 * d;
  auto put = [&](float (&v)[NC][V], int which) {
    if (W > 1) {
#pragma unroll
      for (int k = 0; k < NC; ++k) {
        const int c = col_of<W, V>(k);
        if (c < d)
#pragma unroll
          for (int e = 0; e < V; ++e) out[(long)which * d + c + e] = v[k][e];
      }
      return;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int c = col_of<W, V>(k);
      if (c < d)
#pragma unroll
        for (int e = 0; e < V; ++e) sm[wave * d + c + e] = v[k][e];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < d; i += 256) out[(long)which * d + i] = sm[i] + sm[d + i] + sm[2 * d + i] + sm[3 * d + i];
  };
  put(A, 0); put(B, 1); put(C, 2); put(E, 3);
}

// the column sums over the blocks' partial rows, in a fixed order: a block owns 16 columns, 16 strands of partial rows each
__global__ __launch_bounds__(256) void join_reduce_kernel(JP p, int blocks) {
  __shared__ float sm[16][17];
  const int cl = threadIdx.x & 15, strand = threadIdx.x >> 4, c = blockIdx.x * 16 + cl, d = p.d;
  const bool in = c < d;
  auto total = [&](float v) {                       // over the strands; every thread gets its column's
    __syncthreads();
    sm[strand][cl] = v;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) s += sm[i][cl];
    return s;
  };
  const float sc = in && p.scale ? p.scale[c] : 1.f, w = in && p.post_w ? p.post_w[c] : 1.f, b = in && p.post_b ? p.post_b[c] : 0.f;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  if (p.channel) {
    for (int g = strand; g < p.groups; g += 16) {
      float a = 0.f, bb = 0.f;
      for (int i = 0; i < p.per_group && in; ++i) {
        const float* part = p.part + ((long)g * p.per_group + i) * 4 * d + c;
        a += part[0]; bb += part[d]; s[2] += part[2 * (long)d]; s[3] += part[3 * (long)d];
      }
      if (in) {
        const float gv = act(p, p.gate[(long)g * d + c]);
        s[0] = fmaf(gv, a, s[0]); s[1] = fmaf(gv, bb, s[1]);
        if (p.d_gate) {
          const float v = sc * (w * a + b * bb);
          p.d_gate[(long)g * d + c] = p.gate_tanh ? v * (1.f - gv * gv) : v;
        }
      }
    }
  } else {
    for (int i = strand; i < blocks && in; i += 16) {
      const float* part = p.part + (long)i * 4 * d + c;
      s[0] += part[0]; s[1] += part[d]; s[2] += part[2 * (long)d]; s[3] += part[3 * (long)d];
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) s[i] = total(s[i]);
  if (!in || strand) return;
  if (p.d_post_w) p.d_post_w[c] = sc * s[0];
  if (p.d_post_b) p.d_post_b[c] = sc * s[1];
  if (p.d_scale) p.d_scale[c] = w * s[0] + b * s[1];
  if (p.d_pre_w) p.d_pre_w[c] = s[2];
  if (p.d_pre_b) p.d_pre_b[c] = s[3];
}

// row gate: the rows of a group
__global__ __launch_bounds__(256) void join_gate_kernel(JP p) {
  __shared__ float red[8];
  const int n = p.rows / p.groups;
  for (int g = blockIdx.x; g < p.groups; g += gridDim.x) {
    float s = 0.f;
    for (int i = threadIdx.x; i < n; i += 256) s += p.rowdot[(long)g * n + i];
    s = block_sum256(s, red);
    if (threadIdx.x == 0) {
      const float gv = act(p, p.gate[g]);
      p.d_gate[g] = p.gate_tanh ? s * (1.f - gv * gv) : s;
    }
  }
}

// ------------------------------------------------------------------------------------------ host side
struct Shape { int w, nc, v; };
// one wave per row up to 1024 columns (2 chunks of 8 per lane: the backward's four column sums and three row operands fit its registers),
// a block per row up to 8192; single elements where d or an address rules 16-byte accesses out
bool shape_of(int d, bool vec, Shape& s) {
  if (vec) {
    if (d <= 512) s = {1, 1, 8};
    else if (d <= 1024) s = {1, 2, 8};
    else if (d <= 2048) s = {4, 1, 8};
    else if (d <= 4096) s = {4, 2, 8};
    else if (d <= 8192) s = {4, 4, 8};
    else return false;
  } else {
    if (d <= 256) s = {1, 4, 1};
    else if (d <= 2048) s = {4, 8, 1};
    else if (d <= 8192) s = {4, 32, 1};
    else return false;
  }
  return true;
}
#define JOIN_SHAPES(CASE) CASE(1, 1, 8) CASE(1, 2, 8) CASE(4, 1, 8) CASE(4, 2, 8) CASE(4, 4, 8) CASE(1, 4, 1) CASE(4, 8, 1) CASE(4, 32, 1)

bool aligned16(std::initializer_list<const void*> ps) {
  for (const void* q : ps) if ((uintptr_t)q & 15) return false;
  return true;
}
int blocks_of(const dh_join_norm_args* a, int w, int& per_group) {
  const int rb = 4 / w;
  per_group = 1;
  if (a->gate && a->gate_channel) {
    const int per = a->rows / a->gate_rows, most = dh_cdiv(per, rb);
    int want = 512 / a->gate_rows;
    per_group = want < 1 ? 1 : want > most ? most : want;
    return a->gate_rows * per_group;
  }
  const int n = dh_cdiv(a->rows, rb);
  return n > 512 ? 512 : n;
}

int check(const dh_join_norm_args* a, const char* who) {
  DH_REQUIRE(a, "%s: null args", who);
  DH_REQUIRE(a->dtype == DH_F32 || a->dtype == DH_BF16, "%s: dtype %d", who, a->dtype);
  DH_REQUIRE(a->rows >= 0 && a->d > 0 && a->d <= 8192, "%s: rows %d, width %d (up to 8192)", who, a->rows, a->d);
  DH_REQUIRE(!a->post_b || (a->post_w && !a->rms), "%s: a bias needs its weight and a LayerNorm", who);
  DH_REQUIRE(!a->pre_b || (a->pre_w && !a->rms), "%s: a bias needs its weight and a LayerNorm", who);
  DH_REQUIRE(!a->gate || (a->gate_rows > 0 && a->rows % a->gate_rows == 0), "%s: %d gate rows for %d rows", who, a->gate_rows, a->rows);
  DH_REQUIRE(a->eps >= 0.f && a->eps < INFINITY, "%s: eps", who);
  DH_REQUIRE(a->rows == 0 || (a->x && a->y && a->stats), "%s: x, y and stats are needed", who);
  return DH_OK;
}
JP jparams(const dh_join_norm_args* a) {
  JP p = {};
  p.x = a->x; p.y = a->y; p.x_out = a->x_out; p.n = a->n; p.dxo = a->dx_out; p.dn = a->dn; p.dx = a->dx; p.dy = a->dy;
  p.post_w = a->post_w; p.post_b = a->post_b; p.gate = a->gate; p.scale = a->scale; p.pre_w = a->pre_w; p.pre_b = a->pre_b;
  p.stats = a->stats;
  p.alpha = a->alpha; p.eps = a->eps; p.rows = a->rows; p.d = a->d; p.rms = a->rms; p.gate_tanh = a->gate_tanh; p.pre = a->pre_w != nullptr;
  p.groups = a->gate ? a->gate_rows : 1;
  p.channel = a->gate && a->gate_channel;
  p.per_group = 1;
  return p;
}
bool vec_ok(const dh_join_norm_args* a, bool bwd) {
  bool ok = a->d % 8 == 0 && aligned16({a->x, a->y, a->post_w, a->post_b, a->scale, a->pre_w, a->pre_b}) && (!a->gate || !a->gate_channel || aligned16({a->gate}));
  if (bwd) return ok && aligned16({a->dx_out, a->dn, a->dx, a->dy});
  return ok && aligned16({a->x_out, a->n});
}

}  // namespace

extern "C" int dh_join_norm_fwd(const dh_join_norm_args* a, dh_stream_t stream) {
  if (int e = check(a, "dh_join_norm_fwd")) return e;
  if (a->rows == 0) return DH_OK;
  DH_REQUIRE(a->x_out && (!a->pre_w || a->n), "dh_join_norm_fwd: null output");
  const JP p = jparams(a);
  Shape s;
  DH_REQUIRE(shape_of(a->d, vec_ok(a, false), s), "dh_join_norm_fwd: width %d", a->d);
  int grid = dh_cdiv(a->rows, 4 / s.w);
  if (grid > 2048) grid = 2048;
#define CASE(W_, N_, V_)                                                                                                               \
  if (s.w == W_ && s.nc == N_ && s.v == V_) {                                                                                          \
    if (a->dtype == DH_BF16) hipLaunchKernelGGL((join_fwd_kernel<bf16_t, W_, N_, V_>), dim3(grid), dim3(256), 0, (hipStream_t)stream, p); \
    else hipLaunchKernelGGL((join_fwd_kernel<float, W_, N_, V_>), dim3(grid), dim3(256), 0, (hipStream_t)stream, p);                    \
  }
  JOIN_SHAPES(CASE)
#undef CASE
  DH_CHECK_LAUNCH();
  return DH_OK;
}

extern "C" int64_t dh_join_norm_bwd_ws_bytes(const dh_join_norm_args* a) {
  if (check(a, "dh_join_norm_bwd_ws_bytes")) return -1;
  if (a->rows == 0) return 0;
  int per;
  const int b1 = blocks_of(a, 1, per), b4 = blocks_of(a, 4, per);
  return ((int64_t)(b1 > b4 ? b1 : b4) * 4 * a->d + a->rows) * 4;
}

extern "C" int dh_join_norm_bwd(const dh_join_norm_args* a, dh_stream_t stream) {
  if (int e = check(a, "dh_join_norm_bwd")) return e;
  DH_REQUIRE(a->rows > 0, "dh_join_norm_bwd: no rows");
  DH_REQUIRE(a->dx && a->dy, "dh_join_norm_bwd: null output");
  DH_REQUIRE(a->dx_out || a->dn, "dh_join_norm_bwd: no gradient given");
  DH_REQUIRE(!a->dn || a->pre_w, "dh_join_norm_bwd: dn without the norm it belongs to");
  DH_REQUIRE(a->ws && a->ws_bytes >= dh_join_norm_bwd_ws_bytes(a), "dh_join_norm_bwd: workspace of %lld bytes needed", (long long)dh_join_norm_bwd_ws_bytes(a));
  JP p = jparams(a);
  p.pre = a->dn != nullptr;
  Shape s;
  DH_REQUIRE(shape_of(a->d, vec_ok(a, true), s), "dh_join_norm_bwd: width %d", a->d);
  const int grid = blocks_of(a, s.w, p.per_group);
  const bool gate_rows = a->gate && !p.channel && a->d_gate;
  const bool cols = a->d_post_w || a->d_post_b || a->d_scale || a->d_pre_w || a->d_pre_b || (p.channel && a->d_gate);
  p.part = cols ? (float*)a->ws : nullptr;
  p.rowdot = gate_rows ? (float*)a->ws + (int64_t)grid * 4 * a->d : nullptr;
  p.d_post_w = a->d_post_w; p.d_post_b = a->d_post_b; p.d_gate = a->d_gate; p.d_scale = a->d_scale; p.d_pre_w = a->d_pre_w; p.d_pre_b = a->d_pre_b;
  const size_t lds = s.w == 1 ? (size_t)16 * a->d : 0;
#define CASE(W_, N_, V_)                                                                                                                  \
  if (s.w == W_ && s.nc == N_ && s.v == V_) {                                                                                             \
    if (a->dtype == DH_BF16) hipLaunchKernelGGL((join_bwd_kernel<bf16_t, W_, N_, V_>), dim3(grid), dim3(256), lds, (hipStream_t)stream, p); \
    else hipLaunchKernelGGL((join_bwd_kernel<float, W_, N_, V_>), dim3(grid), dim3(256), lds, (hipStream_t)stream, p);                     \
  }
  JOIN_SHAPES(CASE)
#undef CASE
  DH_CHECK_LAUNCH();
  if (cols) {
    hipLaunchKernelGGL(join_reduce_kernel, dim3(dh_cdiv(a->d, 16)), dim3(256), 0, (hipStream_t)stream, p, grid);
    DH_CHECK_LAUNCH();
  }
  if (gate_rows) {
    hipLaunchKernelGGL(join_gate_kernel, dim3(a->gate_rows > 1024 ? 1024 : a->gate_rows), dim3(256), 0, (hipStream_t)stream, p);
    DH_CHECK_LAUNCH();
  }
  return DH_OK;
}
