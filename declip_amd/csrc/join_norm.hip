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
// (in fp32, the forward's own values) and writes dx, dy.  A row lives in the registers of 1 to 8 waves, statistics
// are fp32 and two-pass (mean first).  The column sums stay in registers over a block's rows, go to a partial row per block, and are
// added in a fixed order by a second small kernel: no atomics, the same result on every run.
// Measured, bf16: 25600 rows of 768, a gate vector per 50 rows: forward 33 us (157 MB: 4.8 TB/s), backward 55 + 8 us (236 MB: 4.2 TB/s); 8191 rows of 4096,
// one gate: 51 us (268 MB: 5.3 TB/s), 97 + 8 us (403 MB: 4.2 TB/s).  fp32: 61 and 110 + 10 us (314, 472 MB), 100 and 177 + 9 us (537, 805 MB).  What holds the backward below the
// forward's rate: a block of 512 threads and 168 registers leaves room for no second one (two waves per SIMD, where 256 threads would allow three).
// A gate vector per ROW is the slow case: a block and a partial row of 16 bytes per element for each, more than the call's own traffic (25600 x 768, bf16: 244, 702 + 352 us).
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
  int per_group;                                 // channel gate: blocks per group (a block's rows lie in one group); else: rows per block
};

__device__ __forceinline__ float act(const JP& p, float g) { return p.gate_tanh ? tanhf(g) : g; }

// V consecutive elements as they come from memory: the next row is on its way in this form
template <typename T, int V> struct Raw;
template <> struct Raw<bf16_t, 8> {
  uint4 v;
  __device__ __forceinline__ void load(const bf16_t* p) { v = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void zero() { v = make_uint4(0u, 0u, 0u, 0u); }
  __device__ __forceinline__ void get(float* o) const {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { o[2 * i] = __uint_as_float(w[i] << 16); o[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
  }
};
template <> struct Raw<bf16_t, 4> {
  uint2 v;
  __device__ __forceinline__ void load(const bf16_t* p) { v = *reinterpret_cast<const uint2*>(p); }
  __device__ __forceinline__ void zero() { v = make_uint2(0u, 0u); }
  __device__ __forceinline__ void get(float* o) const {
    o[0] = __uint_as_float(v.x << 16); o[1] = __uint_as_float(v.x & 0xffff0000u); o[2] = __uint_as_float(v.y << 16); o[3] = __uint_as_float(v.y & 0xffff0000u);
  }
};
template <> struct Raw<bf16_t, 1> {
  bf16_t v;
  __device__ __forceinline__ void load(const bf16_t* p) { v = *p; }
  __device__ __forceinline__ void zero() { v = 0; }
  __device__ __forceinline__ void get(float* o) const { o[0] = bf2f(v); }
};
template <int V> struct Raw<float, V> {
  float v[V];
  __device__ __forceinline__ void load(const float* p) {
    if constexpr (V == 1) v[0] = *p;
    else
#pragma unroll
      for (int i = 0; i < V; i += 4) {
        const float4 a = *reinterpret_cast<const float4*>(p + i);
        v[i] = a.x; v[i + 1] = a.y; v[i + 2] = a.z; v[i + 3] = a.w;
      }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = 0.f;
  }
  __device__ __forceinline__ void get(float* o) const {
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = v[i];
  }
};
template <int V> __device__ __forceinline__ void put(float* p, const float* o) {
  if constexpr (V == 1) *p = o[0];
  else
#pragma unroll
    for (int i = 0; i < V; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
}
template <int V> __device__ __forceinline__ void put(bf16_t* p, const float* o) {
  if constexpr (V == 1) *p = f2bf(o[0]);
  else if constexpr (V == 4) {
    uint2 w;
    w.x = pack2bf_hw(o[0], o[1]); w.y = pack2bf_hw(o[2], o[3]);
    *reinterpret_cast<uint2*>(p) = w;
  } else st8_hw(p, o);
}

// Block of 8 waves = G groups of W waves; a group holds a row, V elements per lane and chunk, NC chunks.
constexpr int NT = 512;
template <int W> struct Lanes {
  static constexpr int G = 8 / W;
  int lane, wave, group, lid;                      // lid: place in the group
  int turn = 0;
  __device__ __forceinline__ Lanes() {
    lane = threadIdx.x & 63;
    wave = threadIdx.x >> 6;
    group = wave / W;
    lid = (wave % W) * 64 + lane;
  }
  template <int V> __device__ __forceinline__ int col(int k) const { return (lid + 64 * W * k) * V; }
  // sums over the group's lanes; every thread of the block comes here (W > 1: one barrier -- two buffers in turn, so the next sum does not write what
  // the last one still reads)
  __device__ __forceinline__ void sum2(float& a, float& b, float* red) {
    a = wave_sum_fast(a);
    b = wave_sum_fast(b);
    if (W > 1) {
      float* r = red + turn * 16;
      turn ^= 1;
      if (lane == 0) { r[2 * wave] = a; r[2 * wave + 1] = b; }
      __syncthreads();
      a = b = 0.f;
#pragma unroll
      for (int i = 0; i < W; ++i) { a += r[2 * (group * W + i)]; b += r[2 * (group * W + i) + 1]; }
    }
  }
  __device__ __forceinline__ float sum(float a, float* red) {
    float zero = 0.f;
    sum2(a, zero, red);
    return a;
  }
};

// rows of a block: a run of consecutive ones, inside one group of rows where the gate is a vector per group
__device__ __forceinline__ void rows_of(const JP& p, int& first, int& last) {
  if (p.channel) {
    const int n = p.rows / p.groups, g = blockIdx.x / p.per_group, part = blockIdx.x % p.per_group, run = (n + p.per_group - 1) / p.per_group;
    first = g * n + min(part * run, n);
    last = g * n + min((part + 1) * run, n);
  } else {
    first = min((long)blockIdx.x * p.per_group, (long)p.rows);
    last = min((long)first + p.per_group, (long)p.rows);
  }
}

// a column vector of the parameters in the lane's columns; `none` where there is no such vector or no such column
template <int W, int NC, int V>
__device__ __forceinline__ void columns(const Lanes<W>& ln, const float* v, int d, float none, float (&o)[NC][V]) {
#pragma unroll
  for (int k = 0; k < NC; ++k) {
    const int c = ln.template col<V>(k);
#pragma unroll
    for (int e = 0; e < V; ++e) o[k][e] = none;
    if (v && c < d) {
      Raw<float, V> r;
      r.load(v + c);
      r.get(o[k]);
    }
  }
}
// what multiplies yhat and what is added, per column: scale (times the group's gate vector) times the norm's weight and bias
template <int W, int NC, int V>
__device__ __forceinline__ void branch_vectors(const JP& p, const Lanes<W>& ln, int first, float (&sw)[NC][V], float (&sb)[NC][V]) {
  float s[NC][V], g[NC][V];
  const int grp = p.channel ? first / (p.rows / p.groups) : 0;
  columns<W, NC, V>(ln, p.scale, p.d, 1.f, s);
  columns<W, NC, V>(ln, p.channel ? p.gate + (long)grp * p.d : nullptr, p.d, 1.f, g);
  columns<W, NC, V>(ln, p.post_w, p.d, 1.f, sw);
  columns<W, NC, V>(ln, p.post_b, p.d, 0.f, sb);
#pragma unroll
  for (int k = 0; k < NC; ++k)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      float m = s[k][e] * (p.channel ? act(p, g[k][e]) : 1.f);
      if (ln.template col<V>(k) >= p.d) m = 0.f;     // lanes behind the last column add nothing to any sum
      sw[k][e] *= m;
      sb[k][e] *= m;
    }
}

// ------------------------------------------------------------------------------------------ forward
template <typename T, int W, int NC, int V>
__global__ __launch_bounds__(NT, NC * V <= 12 ? 4 : 2) void join_fwd_kernel(JP p) {
  __shared__ float red[32];
  Lanes<W> ln;
  constexpr int G = Lanes<W>::G;
  const int d = p.d, rows_per_gate = p.rows / p.groups;
  const float inv_d = 1.f / d;
  int first, last;
  rows_of(p, first, last);
  if (first >= last) return;
  float sw[NC][V], sb[NC][V], pw[NC][V], pb[NC][V];
  Raw<T, V> nx[NC], ny[NC];
  float ng = 1.f;
  auto fetch = [&](int row) {
    row = min(row, last - 1);
    const long at = (long)row * d;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int c = ln.template col<V>(k);
      if (c < d) { nx[k].load((const T*)p.x + at + c); ny[k].load((const T*)p.y + at + c); }
      else { nx[k].zero(); ny[k].zero(); }
    }
    if (p.gate && !p.channel) ng = p.gate[row / rows_per_gate];
  };
  fetch(first + ln.group);
  branch_vectors<W, NC, V>(p, ln, first, sw, sb);
  columns<W, NC, V>(ln, p.pre_w, d, 0.f, pw);
  columns<W, NC, V>(ln, p.pre_b, d, 0.f, pb);
  for (int row0 = first; row0 < last; row0 += G) {
    const int row = row0 + ln.group;
    const bool live = row < last, head = live && ln.lid == 0;
    float xv[NC][V], yv[NC][V];
#pragma unroll
    for (int k = 0; k < NC; ++k) { nx[k].get(xv[k]); ny[k].get(yv[k]); }
    const float g = p.gate && !p.channel ? act(p, ng) : 1.f;
    if (row0 + G < last) fetch(row + G);
    float mu = 0.f, rs = 1.f;
    if (p.post_w) {
      if (!p.rms) {
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < NC; ++k)
#pragma unroll
          for (int e = 0; e < V; ++e) s += yv[k][e];
        mu = ln.sum(s, red) * inv_d;
      }
      float q = 0.f;
#pragma unroll
      for (int k = 0; k < NC; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e) { const float u = ln.template col<V>(k) < d ? yv[k][e] - mu : 0.f; q = fmaf(u, u, q); }
      rs = 1.f / sqrtf(ln.sum(q, red) * inv_d + p.eps);
      if (head) { p.stats[row] = mu; p.stats[p.rows + row] = rs; }
    }
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int c = ln.template col<V>(k);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        xv[k][e] = c < d ? fmaf(p.alpha, xv[k][e], g * fmaf((yv[k][e] - mu) * rs, sw[k][e], sb[k][e])) : 0.f;
        s += xv[k][e];
      }
      if (live && c < d) put<V>((T*)p.x_out + (long)row * d + c, xv[k]);
    }
    if (!p.pre) continue;
    const float mu2 = p.rms ? 0.f : ln.sum(s, red) * inv_d;
    float q = 0.f;
#pragma unroll
    for (int k = 0; k < NC; ++k)
#pragma unroll
      for (int e = 0; e < V; ++e) { const float u = ln.template col<V>(k) < d ? xv[k][e] - mu2 : 0.f; q = fmaf(u, u, q); }
    const float rs2 = 1.f / sqrtf(ln.sum(q, red) * inv_d + p.eps);
    if (head) { p.stats[2 * (long)p.rows + row] = mu2; p.stats[3 * (long)p.rows + row] = rs2; }
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int c = ln.template col<V>(k);
      float o[V];
#pragma unroll
      for (int e = 0; e < V; ++e) o[e] = fmaf((xv[k][e] - mu2) * rs2, pw[k][e], pb[k][e]);
      if (live && c < d) put<V>((T*)p.n + (long)row * d + c, o);
    }
  }
}

// channel gate: gradient of element i of the gate (column c) from the group's sums A and B, and its share of the totals into out[c], out[d + c]
__device__ __forceinline__ void gate_columns(const JP& p, long i, int c, float a, float b, float* out) {
  const float gv = act(p, p.gate[i]);
  if (p.d_gate) {
    const float v = (p.scale ? p.scale[c] : 1.f) * ((p.post_w ? p.post_w[c] : 1.f) * a + (p.post_b ? p.post_b[c] : 0.f) * b);
    p.d_gate[i] = p.gate_tanh ? v * (1.f - gv * gv) : v;
  }
  out[c] = gv * a;
  out[p.d + c] = gv * b;
}

// ------------------------------------------------------------------------------------------ backward
template <typename T, int W, int NC, int V, bool ROWGATE>
__global__ __launch_bounds__(NT, 2) void join_bwd_kernel(JP p) {
  DH_DYN_LDS_A16(float, sm);                      // three parameter vectors over the lanes' columns; behind the loop [G][d] for the groups' column sums
  constexpr int WIDE = 64 * W * NC * V;
  // The next row on its way beside the current one, but for the shape of single elements (odd widths above 4096), whose 16 addresses and 16 columns of each of
  // four operands and sums would spill up to 1513 registers: 2048 rows of 8191 1710 -> 323 us (fp32, one gate), 508 -> 296 (bf16); spills 130 and 113.
  constexpr bool AHEAD = NC < 16;
  __shared__ float red[32];
  Lanes<W> ln;
  constexpr int G = Lanes<W>::G;
  const int d = p.d, rows_per_gate = p.rows / p.groups;
  const float inv_d = 1.f / d;
  int first, last;
  rows_of(p, first, last);
  float A[NC][V], B[NC][V], C[NC][V], E[NC][V];
#pragma unroll
  for (int k = 0; k < NC; ++k)
#pragma unroll
    for (int e = 0; e < V; ++e) A[k][e] = B[k][e] = C[k][e] = E[k][e] = 0.f;
  Raw<T, V> nx[NC], ny[NC], no[NC], nn[NC];
  float nst[4] = {0.f, 1.f, 0.f, 1.f}, ng = 1.f;
  auto fetch = [&](int row) {                      // (a row behind the last one comes as zeros: it adds nothing to the column sums)
    const bool live = row < last;
    row = min(row, last - 1);
    const long at = (long)row * d;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int c = ln.template col<V>(k);
      const bool in = c < d && live;
      if (in) ny[k].load((const T*)p.y + at + c); else ny[k].zero();
      if (in && p.dxo) no[k].load((const T*)p.dxo + at + c); else no[k].zero();
      if (in && p.dn) { nx[k].load((const T*)p.x + at + c); nn[k].load((const T*)p.dn + at + c); } else { nx[k].zero(); nn[k].zero(); }
    }
    if (ROWGATE) ng = p.gate[row / rows_per_gate];
    if (p.post_w) { nst[0] = p.stats[row]; nst[1] = p.stats[p.rows + row]; }
    if (p.dn) { nst[2] = p.stats[2 * (long)p.rows + row]; nst[3] = p.stats[3 * (long)p.rows + row]; }
  };
  if (AHEAD && first < last) fetch(first + ln.group);
  // read by every row from LDS: held in registers they would leave room for half of the waves
  for (int c = threadIdx.x; c < WIDE; c += NT) {
    float s = 0.f, w = 1.f, b = 0.f;               // (columns behind d add nothing to any sum)
    if (c < d) {
      s = p.scale ? p.scale[c] : 1.f;
      if (p.channel) s *= act(p, p.gate[(long)(first < p.rows ? first / rows_per_gate : 0) * d + c]);
      if (p.post_w) w = p.post_w[c];
      if (p.post_b) b = p.post_b[c];
    }
    sm[c] = s * w;
    sm[WIDE + c] = s * b;
    sm[2 * WIDE + c] = c < d && p.dn ? p.pre_w[c] : 0.f;
  }
  __syncthreads();
  auto param = [&](int which, int k, float* o) {
    asm volatile("" ::: "memory");                 // (not moved out of the loop into registers)
    Raw<float, V> r;
    r.load(sm + which * WIDE + ln.template col<V>(k));
    r.get(o);
  };
  for (int row0 = first; row0 < last; row0 += G) {
    const int row = row0 + ln.group;
    const bool live = row < last;
    if (!AHEAD) fetch(row);
    const float mu = nst[0], rs = nst[1], mu2 = nst[2], rs2 = nst[3], g = ROWGATE ? act(p, ng) : 1.f;
    float yh[NC][V], Gr[NC][V], xh[NC][V], wn[NC][V];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      float xv[V], dnv[V], sw[V], sb[V], pw[V];
      param(0, k, sw); param(1, k, sb); param(2, k, pw);
      ny[k].get(yh[k]);
      no[k].get(Gr[k]);
      nx[k].get(xv);
      nn[k].get(dnv);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        yh[k][e] = (yh[k][e] - mu) * rs;
        const float t = fmaf(yh[k][e], sw[e], sb[e]);
        xh[k][e] = (fmaf(p.alpha, xv[e], ROWGATE ? g * t : t) - mu2) * rs2;
        wn[k][e] = dnv[e] * pw[e];              // (0 behind column d and without dn)
        s1 += wn[k][e];
        s2 = fmaf(wn[k][e], xh[k][e], s2);
        C[k][e] = fmaf(dnv[e], xh[k][e], C[k][e]);
        E[k][e] += dnv[e];
      }
    }
    if (AHEAD && row0 + G < last) fetch(row + G);
    if (p.dn) {
      ln.sum2(s1, s2, red);
      const float c1 = p.rms ? 0.f : -rs2 * s1 * inv_d, c2 = -rs2 * s2 * inv_d;
      if (live)                                    // (c1 and c2 are 0 for a row of zeros but for its mean: 0 times what it holds, kept out all the same)
#pragma unroll
        for (int k = 0; k < NC; ++k)
#pragma unroll
          for (int e = 0; e < V; ++e) Gr[k][e] += fmaf(rs2, wn[k][e], fmaf(xh[k][e], c2, c1));
    }
    float s3 = 0.f, s4 = 0.f, dot = 0.f;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int c = ln.template col<V>(k);
      float o[V], sw[V], sb[V];
      param(0, k, sw);
      if (ROWGATE) param(1, k, sb);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        o[e] = p.alpha * Gr[k][e];
        if (ROWGATE) dot = fmaf(Gr[k][e], fmaf(yh[k][e], sw[e], sb[e]), dot);
        const float Gg = ROWGATE ? Gr[k][e] * g : Gr[k][e];     // (channel gate: the vector sits in sw)
        A[k][e] = fmaf(Gg, yh[k][e], A[k][e]);
        B[k][e] += Gg;
        wn[k][e] = Gg * sw[e];
        s3 += wn[k][e];
        s4 = fmaf(wn[k][e], yh[k][e], s4);
      }
      if (live && c < d) put<V>((T*)p.dx + (long)row * d + c, o);
    }
    float c3 = 0.f, c4 = 0.f;
    if (p.post_w) {
      ln.sum2(s3, s4, red);
      c3 = p.rms ? 0.f : -rs * s3 * inv_d;
      c4 = -rs * s4 * inv_d;
    }
    if (ROWGATE && p.rowdot) {
      dot = ln.sum(dot, red);
      if (live && ln.lid == 0) p.rowdot[row] = rows_per_gate == 1 && p.gate_tanh ? dot * (1.f - g * g) : dot;    // (a value per row: this is its gradient)
    }
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int c = ln.template col<V>(k);
      float o[V];
#pragma unroll
      for (int e = 0; e < V; ++e) o[e] = fmaf(rs, wn[k][e], fmaf(yh[k][e], c4, c3));
      if (live && c < d) put<V>((T*)p.dy + (long)row * d + c, o);
    }
  }
  if (!p.part) return;
  float* out = p.part + (long)blockIdx.x * 4 * d;
  auto gather = [&](float (&v)[NC][V], int which) {
    __syncthreads();
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int c = ln.template col<V>(k);
      if (c < d)
#pragma unroll
        for (int e = 0; e < V; ++e) sm[ln.group * d + c + e] = v[k][e];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < d; i += NT) {
      float s = sm[i];
#pragma unroll
      for (int r = 1; r < G; ++r) s += sm[r * d + i];
      out[(long)which * d + i] = s;
    }
  };
  gather(A, 0); gather(B, 1); gather(C, 2); gather(E, 3);
  if (p.channel && p.per_group == 1)               // the whole group is here: the gradient of its gate vector, and A and B with the gate in them
    for (int c = threadIdx.x; c < d; c += NT) gate_columns(p, (long)blockIdx.x * d + c, c, out[c], out[d + c], out);
}

// channel gate, several blocks per group: added up into the group's first partial row; a thread per (group, column)
__global__ __launch_bounds__(256) void join_channel_kernel(JP p) {
  const int d = p.d;
  const long n = (long)p.groups * d;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) {
    const long g = i / d;
    const int c = (int)(i - g * d);
    float* part = p.part + g * p.per_group * 4 * d;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    for (int b = 0; b < p.per_group; ++b)
#pragma unroll
      for (int k = 0; k < 4; ++k) s[k] += part[((long)b * 4 + k) * d + c];
    part[2 * (long)d + c] = s[2];
    part[3 * (long)d + c] = s[3];
    gate_columns(p, i, c, s[0], s[1], part);
  }
}

// sum of a value per thread over the 64 strands of 16 columns
__device__ __forceinline__ float strands(float v, float (&sm)[64][17], int strand, int cl) {
  __syncthreads();
  sm[strand][cl] = v;
  __syncthreads();
  if (strand < 8) {
    v = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) v += sm[strand * 8 + i][cl];
  }
  __syncthreads();
  if (strand < 8) sm[strand][cl] = v;
  __syncthreads();
  v = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) v += sm[i][cl];
  return v;
}
// The sums over rows, in a fixed order.  The first `cols` blocks: 16 columns each, 64 strands over the partial rows (every `step`-th).  The blocks
// behind them: a row gate's groups.
__global__ __launch_bounds__(1024) void join_reduce_kernel(JP p, int blocks, int step, int cols) {
  __shared__ float sm[64][17];
  const int cl = threadIdx.x & 15, strand = threadIdx.x >> 4, d = p.d;
  if ((int)blockIdx.x >= cols) {
    const int n = p.rows / p.groups;
    for (int g = blockIdx.x - cols; g < p.groups; g += gridDim.x - cols) {
      float s = 0.f;
#pragma unroll 4
      for (int i = threadIdx.x; i < n; i += 1024) s += p.rowdot[(long)g * n + i];
      s = strands(s, sm, strand, cl);
#pragma unroll
      for (int m = 8; m; m >>= 1) s += __shfl_xor(s, m, 64);
      if (threadIdx.x == 0) {
        const float gv = act(p, p.gate[g]);
        p.d_gate[g] = p.gate_tanh ? s * (1.f - gv * gv) : s;
      }
    }
    return;
  }
  const int c = blockIdx.x * 16 + cl;
  const bool in = c < d;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  if (in) {
#pragma unroll 4
    for (int i = strand; i < blocks; i += 64) {
      const float* part = p.part + (long)i * step * 4 * d + c;
      s[0] += part[0]; s[1] += part[d]; s[2] += part[2 * (long)d]; s[3] += part[3 * (long)d];
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) s[k] = strands(s[k], sm, strand, cl);
  if (!in || strand) return;
  const float sc = p.scale ? p.scale[c] : 1.f, w = p.post_w ? p.post_w[c] : 1.f, b = p.post_b ? p.post_b[c] : 0.f;
  if (p.d_post_w) p.d_post_w[c] = sc * s[0];
  if (p.d_post_b) p.d_post_b[c] = sc * s[1];
  if (p.d_scale) p.d_scale[c] = w * s[0] + b * s[1];
  if (p.d_pre_w) p.d_pre_w[c] = s[2];
  if (p.d_pre_b) p.d_pre_b[c] = s[3];
}

// ------------------------------------------------------------------------------------------ host side
struct Shape { int w, nc, v; };
// 1, 2, 4 or 8 waves per row, so that a lane holds 8 or 12 columns (the backward's four column sums, three parameter vectors, four operands and the
// next row's fit its registers).  8 elements per access, or 4 where that leaves no lane idle (768 columns: three full accesses instead of one and a
// half); single elements where the width or an address rules vectors out.  One wave up to 1024 columns and a block above, no row
// fetched ahead: forward 44 us, backward 86 (25600 x 768), 61 and 130 (8191 x 4096).
bool shape_of(int d, int vec, Shape& s) {
  const int w = d <= 768 ? 1 : d <= 1536 ? 2 : d <= 2048 ? 4 : 8;
  if (vec == 1) s = d <= 256 ? Shape{1, 4, 1} : d <= 4096 ? Shape{8, 8, 1} : Shape{8, 16, 1};
  else if (d <= 256) s = {1, 1, 4};
  else if (d <= 512 * w && d <= 4096) s = vec == 8 ? Shape{w, 1, 8} : Shape{w, 2, 4};
  else if (d <= 1536) s = {w, 3, 4};
  else s = vec == 8 ? Shape{8, 2, 8} : Shape{8, 4, 4};
  return d <= 8192;
}
#define JOIN_SHAPES(CASE)                                                                                                                \
  CASE(1, 1, 4) CASE(1, 1, 8) CASE(1, 2, 4) CASE(1, 3, 4) CASE(2, 1, 8) CASE(2, 2, 4) CASE(2, 3, 4) CASE(4, 1, 8) CASE(4, 2, 4) CASE(8, 1, 8) \
  CASE(8, 2, 4) CASE(8, 2, 8) CASE(8, 4, 4) CASE(1, 4, 1) CASE(8, 8, 1) CASE(8, 16, 1)

int j_cus() {
  static int n = 0;
  if (!n) {
    int dev = 0;
    hipDeviceProp_t pr;
    n = (hipGetDevice(&dev) == hipSuccess && hipGetDeviceProperties(&pr, dev) == hipSuccess && pr.multiProcessorCount > 0) ? pr.multiProcessorCount : 256;
  }
  return n;
}
// blocks of a launch with at most `most` of them (channel gate: at least one per group), and JP::per_group
int blocks_of(const dh_join_norm_args* a, int w, int most, int& per_group) {
  const int g = 8 / w;
  if (a->gate && a->gate_channel) {
    const int per = a->rows / a->gate_rows, fit = dh_cdiv(per, g);
    per_group = most / a->gate_rows < 1 ? 1 : most / a->gate_rows > fit ? fit : most / a->gate_rows;
    return a->gate_rows * per_group;
  }
  int n = dh_cdiv(a->rows, g);
  if (n > most) n = most;
  per_group = dh_cdiv(dh_cdiv(a->rows, n), g) * g;
  return dh_cdiv(a->rows, per_group);
}
// one block per compute unit, whose column sums leave once (two rounds of blocks at 25600 x 768: 109 us against 55) -- but with a gate vector per group of rows a block
// per group at least (512 groups of 50 rows: two rounds)
int bwd_blocks(const dh_join_norm_args* a, int w, int& per_group) { return blocks_of(a, w, j_cus(), per_group); }

int check(const dh_join_norm_args* a, const char* who) {
  DH_REQUIRE(a, "%s: null args", who);
  DH_REQUIRE(a->dtype == DH_F32 || a->dtype == DH_BF16, "%s: dtype %d", who, a->dtype);
  DH_REQUIRE(a->rows >= 0 && a->rows < (1 << 30) && a->d > 0 && a->d <= 8192, "%s: rows %d (below 2^30), width %d (up to 8192)", who, a->rows, a->d);
  DH_REQUIRE(!a->post_b || (a->post_w && !a->rms), "%s: a bias needs its weight and a LayerNorm", who);
  DH_REQUIRE(!a->pre_b || (a->pre_w && !a->rms), "%s: a bias needs its weight and a LayerNorm", who);
  DH_REQUIRE(!a->gate || (a->gate_rows > 0 && a->rows % a->gate_rows == 0), "%s: %d gate rows for %d rows", who, a->gate_rows, a->rows);
  DH_REQUIRE(!a->gate || !a->gate_channel || a->gate_rows < (1 << 22), "%s: %d gate vectors (below 2^22)", who, a->gate_rows);
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
// elements per access that the width and the addresses allow: 8, 4 or 1
int vec_of(const dh_join_norm_args* a, bool bwd) {
  const void* act[] = {a->x, a->y, bwd ? a->dx_out : a->x_out, bwd ? a->dn : a->n, bwd ? a->dx : nullptr, bwd ? a->dy : nullptr};
  for (const void* q : {a->post_w, a->post_b, a->scale, a->pre_w, a->pre_b, a->gate && a->gate_channel ? a->gate : nullptr})
    if ((uintptr_t)q & 15) return 1;
  const int size = a->dtype == DH_BF16 ? 2 : 4;
  for (int v = 8; v >= 4; v -= 4) {
    bool ok = a->d % v == 0;
    for (const void* q : act) ok = ok && (uintptr_t)q % (v * size > 16 ? 16 : v * size) == 0;
    if (ok) return v;
  }
  return 1;
}

}  // namespace

extern "C" int dh_join_norm_fwd(const dh_join_norm_args* a, dh_stream_t stream) {
  if (int e = check(a, "dh_join_norm_fwd")) return e;
  if (a->rows == 0) return DH_OK;
  DH_REQUIRE(a->x_out && (!a->pre_w || a->n), "dh_join_norm_fwd: null output");
  JP p = jparams(a);
  Shape s;
  DH_REQUIRE(shape_of(a->d, vec_of(a, false), s), "dh_join_norm_fwd: width %d", a->d);
  const int grid = blocks_of(a, s.w, 4 * j_cus(), p.per_group);
#define CASE(W_, N_, V_)                                                                                                               \
  if (s.w == W_ && s.nc == N_ && s.v == V_) {                                                                                          \
    if (a->dtype == DH_BF16) hipLaunchKernelGGL((join_fwd_kernel<bf16_t, W_, N_, V_>), dim3(grid), dim3(NT), 0, (hipStream_t)stream, p); \
    else hipLaunchKernelGGL((join_fwd_kernel<float, W_, N_, V_>), dim3(grid), dim3(NT), 0, (hipStream_t)stream, p);                    \
  }
  JOIN_SHAPES(CASE)
#undef CASE
  DH_CHECK_LAUNCH();
  return DH_OK;
}

extern "C" int64_t dh_join_norm_bwd_ws_bytes(const dh_join_norm_args* a) {
  if (check(a, "dh_join_norm_bwd_ws_bytes")) return -1;
  if (a->rows == 0) return 0;
  int per, most = 0;
  for (int w = 1; w <= 8; w *= 2) { const int b = bwd_blocks(a, w, per); most = b > most ? b : most; }    // (which one runs depends on the addresses)
  return ((int64_t)most * 4 * a->d + a->rows) * 4;
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
  DH_REQUIRE(shape_of(a->d, vec_of(a, true), s), "dh_join_norm_bwd: width %d", a->d);
  const int grid = bwd_blocks(a, s.w, p.per_group);
  const bool row_gate = a->gate && !p.channel, gate_rows = row_gate && a->d_gate;
  const bool cols = a->d_post_w || a->d_post_b || a->d_scale || a->d_pre_w || a->d_pre_b || (p.channel && a->d_gate);
  p.part = cols ? (float*)a->ws : nullptr;
  const bool per_row = gate_rows && a->gate_rows == a->rows;           // the rows' sums are the gate's gradient
  p.rowdot = per_row ? a->d_gate : gate_rows ? (float*)a->ws + (int64_t)grid * 4 * a->d : nullptr;
  p.d_post_w = a->d_post_w; p.d_post_b = a->d_post_b; p.d_gate = a->d_gate; p.d_scale = a->d_scale; p.d_pre_w = a->d_pre_w; p.d_pre_b = a->d_pre_b;
  const size_t vectors = (size_t)3 * 64 * s.w * s.nc * s.v * 4, sums = (size_t)(8 / s.w) * a->d * 4, lds = vectors > sums ? vectors : sums;
#define CASE(W_, N_, V_)                                                                                                                  \
  if (s.w == W_ && s.nc == N_ && s.v == V_) {                                                                                             \
    if (a->dtype == DH_BF16 && row_gate) hipLaunchKernelGGL((join_bwd_kernel<bf16_t, W_, N_, V_, true>), dim3(grid), dim3(NT), lds, (hipStream_t)stream, p); \
    else if (a->dtype == DH_BF16) hipLaunchKernelGGL((join_bwd_kernel<bf16_t, W_, N_, V_, false>), dim3(grid), dim3(NT), lds, (hipStream_t)stream, p); \
    else if (row_gate) hipLaunchKernelGGL((join_bwd_kernel<float, W_, N_, V_, true>), dim3(grid), dim3(NT), lds, (hipStream_t)stream, p);   \
    else hipLaunchKernelGGL((join_bwd_kernel<float, W_, N_, V_, false>), dim3(grid), dim3(NT), lds, (hipStream_t)stream, p);              \
  }
  JOIN_SHAPES(CASE)
#undef CASE
  DH_CHECK_LAUNCH();
  if (p.channel && cols && p.per_group > 1) {
    const int64_t n = ((int64_t)p.groups * a->d + 255) / 256;
    hipLaunchKernelGGL(join_channel_kernel, dim3(n > 2048 ? 2048 : (unsigned)n), dim3(256), 0, (hipStream_t)stream, p);
    DH_CHECK_LAUNCH();
  }
  const int nc = cols ? dh_cdiv(a->d, 16) : 0, ng = !gate_rows || per_row ? 0 : a->gate_rows > 1024 ? 1024 : a->gate_rows;
  if (nc + ng) {
    hipLaunchKernelGGL(join_reduce_kernel, dim3(nc + ng), dim3(1024), 0, (hipStream_t)stream, p, p.channel ? p.groups : grid, p.channel ? p.per_group : 1, nc);
    DH_CHECK_LAUNCH();
  }
  return DH_OK;
}
