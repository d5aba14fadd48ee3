// Cross attention: queries of one packed batch against keys / values of another length (an encoder's states).
//
//   s = scale q k^T over the valid keys, p = softmax(s), o = p v;   lse = log sum exp s
//   D = sum(do o), dv = p^T do, ds = p (do v^T - D), dq = scale ds k, dk = scale ds^T q
//
// Rows of one kv head: the `rep` query heads that share it are packed into the query axis, row m = (query m / rep, head m % rep), so
// shared heads cost no extra pass over k / v and their dk / dv are sums inside one accumulator (a fixed order, no atomics).
//
// One pass with running maximum and sum.  The scores are formed TRANSPOSED, S^T = K Q^T (v_mfma 32x32): a lane then owns one query
// (column), the softmax is in-lane plus one exchange between the half-waves, and the accumulator registers 8t .. 8t+7 of a 32-key block are
// at once the B operand of the next product O^T = V^T P^T: its contraction index is numbered as the accumulator has it
// (key 8i + 4h + r <-> slot (h, 4i' + r)), V^T's fragment is read from the row-major tile by the transpose read with the same numbering.
// P never leaves the registers.
//   fwd   a wave owns 32 rows m, Q in registers, K / V tiles in LDS
//   dq    the same with dO in registers too: dP^T = V dO^T, D = sum p dp, then dS^T, dQ^T += K^T dS^T;  writes D for dkv
//   dkv   a wave owns 32 keys, K / V in registers, Q / dO tiles in LDS: S = Q K^T, dP = dO V^T, dV^T += dO^T P, dK^T += Q^T dS
// bf16: v_mfma_f32_32x32x16_bf16.  P and dS are rounded to bf16 as its operands, the one rounding between inputs and results: independent element by element,
// it costs the results about as much as their own rounding (1.7e-3 of the norm each), and kept in two bf16 parts P and dS would double half of the
// products.  Their sums (l, D) are formed before, in fp32.  fp32: v_mfma_f32_32x32x2_f32, nothing rounded.
//
// What bounds it, measured (bf16):
//   256 captions of 5 .. 77 tokens on 197 keys, 8 heads of 64: 32 / 54 / 60 us (fwd / dq / dkv), memory: 125 / 241 / 229 MB at 3.9 .. 4.5 TB/s.  Each tensor once would
//   be 249 MB, 48 us for all three; k and v are read four times, q and do three.
//   16 pairs of 4096 rows on 1568 .. 3136 keys, hd 128: 142 / 305 / 272 us = 740 / 860 / 770 TFLOP/s of matrix instructions at full lengths (dq's five
//   products, two of them for D).  They hold the matrix units for 31 / 38 / 33 % of the cycles, vector instructions 42 / 39 / 27 %: one after
//   the other in a wave, and two waves per SIMD cover part of it.  dkv has blocks for 208 of 256 compute units.
//   24 pairs of 2047 rows on 6272 keys, hd 64: 104 + 9 us.  147 tiles of 32 rows and 64 keys per SIMD, each 512 cycles of matrix instructions and about 900 of vector
//   ones (512 of them the 32 exponentials): 34 + 59 us at the 2.2 GHz it ran at, so the two hardly overlap.
//   64 sequences of one token, 4 kv heads, up to 3136 keys: 27 + 7 us, 129 MB = 4.8 TB/s.
//   fp32, 16 sequences of up to 77 on 257, 12 heads of 80: 40 / 50 / 44 us.  The 64-cycle matrix instructions of a block in a chain are 13 .. 19 of it (twice that where
//   two blocks share a compute unit); half of the waves of 128-row blocks have no rows, a head of 80 is computed as 96, and the forward spills.
//
// Keys outside the sequence or masked: their rows are staged as ZEROS (whatever the memory holds, NaN included) and their scores are
// -inf.  A row without a valid key: o = 0, lse = -inf, no gradient.  Rows that no sequence owns are written as zeros (lse -inf).
#include "dh_common.h"
#include <math.h>

namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct XP {
  const void *q, *k, *v, *o, *dout;
  void *out, *dq, *dk, *dv;
  float *lse, *delta, *part_o, *part_ml, *part_d;
  const int *cu_q, *cu_kv, *kv_len;
  const uint8_t* key_mask;
  long ldq, ldk, ldv, ldo, lddo, lddq, lddk, lddv;
  int rows_q, rows_kv, batch, heads, kv_heads, rep, hd;
  unsigned magic;     // ceil(2^32 / rep)
  float scale;
  int tiles;          // tiles per (sequence, kv head) in the grid; a block walks t, t + tiles, ... (longer sequences than announced are still whole)
  int nsplit;         // key ranges per tile (forward)
  int main_blocks;    // blocks behind these clear the rows no sequence owns
  int by_pair;        // block order: 1 = the blocks of one (sequence, kv head) on one XCD
};

// Tiles in LDS: row-major, rows padded so that 16 consecutive rows at one 16-byte chunk (the row operand) start in 16 different groups of 4 banks and 4
// consecutive rows (the transpose read, 64 bytes of each) overlap as little as such a stride allows.  (Conflict-free for both would be an exclusive-or of the
// chunk with the row; its address registers spill: hd 128 dq 191 -> 213 us, dkv 382 -> 453.  128 columns padded by 8 instead of 24: fwd 159 us against 150,
// dkv 384 against 350.)
template <typename T, int HDP> struct Lay {
  static constexpr int EPC = 16 / sizeof(T), LD = HDP + (sizeof(T) == 2 && HDP == 128 ? 24 : EPC);
};

template <typename T> struct Op;
template <> struct Op<bf16_t> {
  static constexpr int EPC = 8;                      // elements of a 16-byte chunk
  typedef bf16x8_t Frag;
  struct PF { bf16x8_t f[2]; };
  static __device__ __forceinline__ void mma(f32x16_t& c, Frag a, Frag b) { c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ PF pack(const f32x16_t& s) {
    PF p;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      union { uint32_t u[4]; bf16x8_t v; } x;
#pragma unroll
      for (int e = 0; e < 4; ++e) x.u[e] = pack2bf_hw(s[8 * t + 2 * e], s[8 * t + 2 * e + 1]);
      p.f[t] = x.v;
    }
    return p;
  }
  // c[32 columns col0.. of the tile] += tile rows row0 .. row0 + 31, transposed, times p
  template <int HDP>
  static __device__ __forceinline__ void mma_t(f32x16_t& c, const bf16_t* tile, int row0, int col0, const PF& p, int lane) {
    typedef __attribute__((ext_vector_type(4))) short s16x4;
    constexpr int ld = Lay<bf16_t, HDP>::LD;
    const int t16 = lane & 15;
    const bf16_t* b = tile + (row0 + 4 * (lane >> 5) + (t16 >> 2)) * ld + col0 + 16 * ((lane >> 4) & 1) + 4 * (t16 & 3);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      union { struct { s16x4 a, b; } s; bf16x8_t v; } u;
      u.s.a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(b + (16 * t) * ld));
      u.s.b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(b + (16 * t + 8) * ld));
      c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(u.v, p.f[t], c, 0, 0, 0);
    }
  }
  static __device__ __forceinline__ void store4(bf16_t* p, float a, float b, float c, float d) {
    uint2 w;
    w.x = pack2bf_hw(a, b); w.y = pack2bf_hw(c, d);
    *reinterpret_cast<uint2*>(p) = w;
  }
  static __device__ __forceinline__ float dot(Frag a, Frag b) {
    union { Frag f; uint32_t u[4]; } x, y;
    x.f = a; y.f = b;
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      s = fmaf(__uint_as_float(x.u[e] << 16), __uint_as_float(y.u[e] << 16), s);
      s = fmaf(__uint_as_float(x.u[e] & 0xffff0000u), __uint_as_float(y.u[e] & 0xffff0000u), s);
    }
    return s;
  }
};
template <> struct Op<float> {
  static constexpr int EPC = 4;
  typedef f32x4_t Frag;
  typedef f32x16_t PF;
  static __device__ __forceinline__ void mma(f32x16_t& c, Frag a, Frag b) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
  }
  static __device__ __forceinline__ PF pack(const f32x16_t& s) { return s; }
  template <int HDP>
  static __device__ __forceinline__ void mma_t(f32x16_t& c, const float* tile, int row0, int col0, const PF& p, int lane) {
    constexpr int ld = Lay<float, HDP>::LD;
    const float* b = tile + (row0 + 4 * (lane >> 5)) * ld + col0 + (lane & 31);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) c = __builtin_amdgcn_mfma_f32_32x32x2f32(b[(8 * i + r) * ld], p[4 * i + r], c, 0, 0, 0);
  }
  static __device__ __forceinline__ void store4(float* p, float a, float b, float c, float d) { *reinterpret_cast<float4*>(p) = make_float4(a, b, c, d); }
  static __device__ __forceinline__ float dot(Frag a, Frag b) { return fmaf(a[0], b[0], fmaf(a[1], b[1], fmaf(a[2], b[2], a[3] * b[3]))); }
};

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// ------------------------------------------------------------------------------------------ geometry
struct Seq { int q0, nq, k0, nk, nseg; };      // query rows, valid keys, key rows of the segment
__device__ __forceinline__ int clampi(int v, int lo, int hi) { return v < lo ? lo : (v > hi ? hi : v); }
__device__ __forceinline__ Seq seq_of(const XP& p, int b) {
  Seq s;
  if (p.cu_q) {
    s.q0 = clampi(p.cu_q[b], 0, p.rows_q);
    s.nq = clampi(p.cu_q[b + 1], s.q0, p.rows_q) - s.q0;
  } else {
    s.nq = p.rows_q / p.batch;
    s.q0 = b * s.nq;
  }
  if (p.cu_kv) {
    s.k0 = clampi(p.cu_kv[b], 0, p.rows_kv);
    s.nseg = clampi(p.cu_kv[b + 1], s.k0, p.rows_kv) - s.k0;
  } else {
    s.nseg = p.rows_kv / p.batch;
    s.k0 = b * s.nseg;
  }
  s.nk = p.kv_len ? clampi(p.kv_len[b], 0, s.nseg) : s.nseg;
  return s;
}

// block -> (sequence, kv head, tile, split).  by_pair: consecutive blocks go to the 8 XCDs in turn, so the pairs are dealt to the XCDs and all
// blocks of a pair land on one of them (its L2 then holds that pair's k / v or q / do once).
struct Work { int b, g, t, split; bool live; };
__device__ __forceinline__ Work work_of(const XP& p, int bid) {
  const int inner = p.tiles * p.nsplit, pairs = p.batch * p.kv_heads;
  int pair, in;
  if (p.by_pair) {
    const int slot = bid >> 3;
    pair = (slot / inner) * 8 + (bid & 7);
    in = slot % inner;
  } else {
    pair = bid / inner;
    in = bid % inner;
  }
  Work w;
  w.live = pair < pairs;
  w.g = pair % p.kv_heads;
  w.b = pair / p.kv_heads;
  w.split = in % p.nsplit;
  w.t = in / p.nsplit;
  return w;
}

// rows [0, first) and [last, rows) of a [rows][width] matrix are cleared by the blocks behind the main ones
template <typename T>
__device__ void clear_rows(T* x, long ld, int width, int first, int last, int rows, int blk, int nblk, int tid, int nthr) {
  const int nch = width / Op<T>::EPC, n0 = first, n = first + (rows - last);
  for (long i = (long)blk * nthr + tid; i < (long)n * nch; i += (long)nblk * nthr) {
    const int r = (int)(i / nch), c = (int)(i % nch);
    const long row = r < n0 ? r : last + (r - n0);
    *reinterpret_cast<uint4*>(x + row * ld + (long)c * Op<T>::EPC) = make_uint4(0u, 0u, 0u, 0u);
  }
}
__device__ __forceinline__ void owned(const int* cu, int batch, int rows, int& first, int& last) {
  first = clampi(cu[0], 0, rows);
  last = clampi(cu[batch], first, rows);
}

// row m of the packed query axis -> (query, head of the group): the quotient by rep from one high product with magic = ceil(2^32 / rep), which is too
// large by one at most
__device__ __forceinline__ void m_split(const XP& p, int m, int& q, int& r) {
  q = p.rep == 1 ? m : (int)__umulhi((unsigned)m, p.magic);
  r = m - q * p.rep;
  if (r < 0) { --q; r += p.rep; }
}
__device__ __forceinline__ long m_offset(const XP& p, const Seq& s, int g, int m, long ld) {
  int q, r;
  m_split(p, m, q, r);
  return (long)(s.q0 + q) * ld + (g * p.rep + r) * p.hd;
}
__device__ __forceinline__ long m_stat(const XP& p, const Seq& s, int g, int m) {
  int q, r;
  m_split(p, m, q, r);
  return (long)(g * p.rep + r) * p.rows_q + s.q0 + q;
}

// this lane's operand chunks of one row (lane half h: elements ks * 2 EPC + h EPC ..), zero where dead
template <typename T, int HDP>
__device__ __forceinline__ void load_row(typename Op<T>::Frag* f, const T* row, bool live, int hd, int h) {
  constexpr int EPC = Op<T>::EPC, KS = HDP / (2 * EPC);
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    union { uint4 u; typename Op<T>::Frag f; } x;
    x.u = make_uint4(0u, 0u, 0u, 0u);
    const int c = ks * 2 * EPC + h * EPC;
    if (live && c < hd) x.u = *reinterpret_cast<const uint4*>(row + c);
    f[ks] = x.f;
  }
}
// The operand rows are here: a use in front of the tile loop, on every path to it.  Without it the compiler places their wait at the loop's first
// product, where it waits on every turn for ALL loads under way, the next tile's too.
template <typename F, int KS>
__device__ __forceinline__ void arrived(F (&f)[KS]) {
#ifndef DH_HOST_EMU
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(f[ks]));
#endif
}
template <typename T, int HDP>
__device__ __forceinline__ f32x16_t mma_row(const T* tile, int row0, const typename Op<T>::Frag* f, int lane) {
  constexpr int EPC = Op<T>::EPC, KS = HDP / (2 * EPC);
  f32x16_t c;
#pragma unroll
  for (int i = 0; i < 16; ++i) c[i] = 0.f;
  const T* row = tile + (row0 + (lane & 31)) * Lay<T, HDP>::LD + (lane >> 5) * EPC;
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) Op<T>::mma(c, *reinterpret_cast<const typename Op<T>::Frag*>(row + ks * 2 * EPC), f[ks]);
  return c;
}

// the value of the lane 32 further (the other half of the same row / key column)
__device__ __forceinline__ float other_half(float v) {
#ifndef DH_HOST_EMU
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float((threadIdx.x & 32) ? r[0] : r[1]);
#else
  return __shfl_xor(v, 32, 64);
#endif
}
__device__ __forceinline__ float half_max(float v) {
#ifndef DH_HOST_EMU
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
#else
  return fmaxf(v, __shfl_xor(v, 32, 64));
#endif
}

// Two tiles of ROWS rows on their way from memory to LDS.  fetch() asks for the next tile while the current one is multiplied (16-byte loads, no
// branch: rows behind the last one read that one again), store() puts it into the other LDS buffer one iteration later.
template <typename T, int HDP, int ROWS, int NT>
struct Pair2 {
  static constexpr int EPC = Op<T>::EPC, NCH = HDP / EPC, N = (ROWS * NCH + NT - 1) / NT, LD = Lay<T, HDP>::LD;
  static constexpr bool RAGGED = ROWS * NCH % NT != 0;      // fewer tasks than threads, or a last round of fewer
  uint4 a[N], b[N];
  uint8_t keep[N];
  // pa / pb: the tile's bases (uniform); off_a / off_b(row): element offsets of its rows from there, 32 bits (scalar base + vector offset, no 64-bit
  // address per thread); last: the last of its rows that exists; mask: the tile's byte per row, or NULL
  template <typename FA, typename FB>
  __device__ __forceinline__ void fetch(const T* pa, const T* pb, FA off_a, FB off_b, int last, const uint8_t* mask, int hd, int tid) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      if (RAGGED && tid + k * NT >= ROWS * NCH) continue;
      const int task = tid + k * NT, row = min(task / NCH, last), c = (task % NCH) * EPC, col = HDP == hd || c < hd ? c : 0;
      a[k] = *reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(pa) + (uint32_t)((off_a(row) + col) * (int)sizeof(T)));
      b[k] = *reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(pb) + (uint32_t)((off_b(row) + col) * (int)sizeof(T)));
      if (mask) keep[k] = mask[row];
    }
  }
  // edge: rows or columns of this tile may have to be zeros (first .. last and mask as fetched)
  __device__ __forceinline__ void store(T* ta, T* tb, bool edge, int first, int last, bool masked, int hd, int tid) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int task = tid + k * NT, row = task / NCH, c = (task % NCH) * EPC;
      if (RAGGED && task >= ROWS * NCH) continue;
      if (edge && (first + row > last || c >= hd || (masked && !keep[k]))) a[k] = b[k] = make_uint4(0u, 0u, 0u, 0u);
      *reinterpret_cast<uint4*>(ta + row * LD + c) = a[k];
      *reinterpret_cast<uint4*>(tb + row * LD + c) = b[k];
    }
  }
};

// The key tiles of a sequence: K and V rows in two LDS buffers, the validity of their keys beside them.
template <typename T, int HDP, int BN, int NT>
struct Tiles {
  static constexpr int LD = Lay<T, HDP>::LD;
  const T *kb, *vb;
  const uint8_t* km;
  T* buf;
  float* bias;
  long ldk, ldv;
  int nk, hd;
  uint8_t own;                                         // validity of key `tid` of the tile on its way
  Pair2<T, HDP, BN, NT> st;
  __device__ __forceinline__ Tiles(const XP& p, const Seq& s, int g, unsigned char* smem) {
    kb = (const T*)p.k + (long)s.k0 * p.ldk + (long)g * p.hd;
    vb = (const T*)p.v + (long)s.k0 * p.ldv + (long)g * p.hd;
    km = p.key_mask ? p.key_mask + s.k0 : nullptr;
    buf = reinterpret_cast<T*>(smem);
    bias = reinterpret_cast<float*>(buf + 4 * BN * LD);
    ldk = p.ldk; ldv = p.ldv; nk = s.nk; hd = p.hd;
  }
  __device__ __forceinline__ void fetch(int kt, int tid) {
    const int first = kt * BN, last = nk - 1 - first;
    const uint8_t* m = km ? km + first : nullptr;
    st.fetch(kb + (long)first * ldk, vb + (long)first * ldv, [&](int r) { return r * (int)ldk; }, [&](int r) { return r * (int)ldv; }, last, m, hd, tid);
    if (m && tid < BN) own = m[min(tid, last)];
  }
  __device__ __forceinline__ bool edge(int kt) const { return km != nullptr || (kt + 1) * BN > nk; }
  __device__ __forceinline__ void store(int kt, int tid) {
    T* b = buf + (kt & 1) * 2 * BN * LD;
    const bool e = edge(kt);
    st.store(b, b + BN * LD, e || hd < HDP, kt * BN, nk - 1, km != nullptr, hd, tid);
    if (e && tid < BN) bias[(kt & 1) * BN + tid] = kt * BN + tid < nk && (!km || own) ? 0.f : -INFINITY;
  }
  __device__ __forceinline__ void begin(int lo, int hi, int tid) {
    if (lo >= hi) return;
    fetch(lo, tid);
    store(lo, tid);
    if (lo + 1 < hi) fetch(lo + 1, tid);
    __syncthreads();
  }
  // tile kt for reading (true: with keys that are none, see bias); the one after it goes to the other buffer, the next but one on its way
  __device__ __forceinline__ bool next(int kt, int hi, int tid, const T*& ks, const T*& vs, const float*& bi) {
    if (kt + 1 < hi) {
      store(kt + 1, tid);
      if (kt + 2 < hi) fetch(kt + 2, tid);
    }
    ks = buf + (kt & 1) * 2 * BN * LD;
    vs = ks + BN * LD;
    bi = bias + (kt & 1) * BN;
    return edge(kt);
  }
};
// scores of keys that are none become -inf (a select, not a sum: such a score may be anything)
__device__ __forceinline__ void mask_keys(f32x16_t& sc, const float* bias, int h) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float4 bi = *reinterpret_cast<const float4*>(bias + 8 * i + 4 * h);
    sc[4 * i] = bi.x < 0.f ? -INFINITY : sc[4 * i]; sc[4 * i + 1] = bi.y < 0.f ? -INFINITY : sc[4 * i + 1];
    sc[4 * i + 2] = bi.z < 0.f ? -INFINITY : sc[4 * i + 2]; sc[4 * i + 3] = bi.w < 0.f ? -INFINITY : sc[4 * i + 3];
  }
}

// The result rows of a wave leave through LDS as whole rows, 16 bytes per lane (the accumulators hold 4 columns of a row per lane and register group:
// stored from there a row would be written in 8-byte pieces).  acc[d][4 i + r] = row (lane & 31), column 32 d + 8 i + 4 h + r, times f; row_ptr(r): where
// row r of the block goes, or nullptr.  U: element type of the result.  Every thread of the block comes here; the LDS is free before and after.
template <typename U, int HDP, typename F>
__device__ __forceinline__ void rows_out(unsigned char* smem, const f32x16_t* acc, float f, int hd, int tid, F row_ptr) {
  constexpr int EPC = Op<U>::EPC, LD = HDP + EPC, DB = HDP / 32, NCH = HDP / EPC;
  const int lane = tid & 63, wave = tid >> 6, h = lane >> 5;
  U* mine = reinterpret_cast<U*>(smem) + wave * 32 * LD;
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      Op<U>::store4(mine + (lane & 31) * LD + d * 32 + 8 * i + 4 * h, acc[d][4 * i] * f, acc[d][4 * i + 1] * f, acc[d][4 * i + 2] * f, acc[d][4 * i + 3] * f);
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 32 * NCH / 64; ++k) {
    const int task = lane + 64 * k, r = task / NCH, c = (task % NCH) * EPC;
    U* to = row_ptr(wave * 32 + r);
    if (to && c < hd) *reinterpret_cast<uint4*>(to + c) = *reinterpret_cast<const uint4*>(mine + r * LD + c);
  }
  __syncthreads();
}

// Waves per SIMD a shape is compiled for.  Two (a budget of 256 registers keeps the accumulators out of the accumulation registers, whose moves cost the
// rescaled forward 192 instructions a tile) unless that spills more than it hides.  Measured in us, 256 captions of 5 .. 77 tokens on 197 keys, 8 heads:
// hd 128 dq 1 wave per block 87 for one wave per SIMD against 262 for two, dkv of 2 waves per block 180 / 370, of 4 waves 194 / 276; hd 96 (128 sequences
// of 77) dkv of 4 waves 97 / 79; fp32 hd 64 (16 sequences of 77) dkv 23 / 29, fwd of one wave 17.6 / 23.  RW: waves per block.
template <typename T, int HDP, int RW, bool SPLIT> constexpr int waves_fwd() {
  constexpr int row = HDP * sizeof(T);
  return SPLIT && RW == 4 && row <= 128 && sizeof(T) == 2 ? 3 : RW == 1 ? (row <= 64 ? 3 : sizeof(T) == 2 && row <= 128 ? 2 : 1) : row <= 384 ? 2 : 1;
}
template <typename T, int HDP, int RW> constexpr int waves_dq() {
  constexpr int row = HDP * sizeof(T);
  return RW == 1 && row <= 64 ? 3 : row <= 128 || RW == 8 || (RW == 4 && row <= 256) ? 2 : 1;
}
template <typename T, int HDP, int RW> constexpr int waves_dkv() {
  constexpr int row = HDP * sizeof(T);
  return RW == 1 && row <= 64 ? 3 : row <= 128 || RW == 8 || (RW == 4 && row == 192) ? 2 : 1;
}

// ------------------------------------------------------------------------------------------ forward
template <typename T, int HDP, int RW, int BN, bool SPLIT>
__global__ __launch_bounds__(64 * RW, (waves_fwd<T, HDP, RW, SPLIT>())) void xattn_fwd_kernel(XP p) {
  constexpr int EPC = Op<T>::EPC, KS = HDP / (2 * EPC), DB = HDP / 32, NB = BN / 32, BM = 32 * RW, NT = 64 * RW;
  DH_DYN_LDS_A16(unsigned char, smem);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;
  if ((int)blockIdx.x >= p.main_blocks) {
    int first, last;
    owned(p.cu_q, p.batch, p.rows_q, first, last);
    const int blk = blockIdx.x - p.main_blocks, nblk = gridDim.x - p.main_blocks;
    clear_rows<T>((T*)p.out, p.ldo, p.heads * p.hd, first, last, p.rows_q, blk, nblk, tid, NT);
    const int n = first + p.rows_q - last;
    for (long i = (long)blk * NT + tid; i < (long)n * p.heads; i += (long)nblk * NT) {
      const int r = (int)(i % n);
      p.lse[(i / n) * p.rows_q + (r < first ? r : last + r - first)] = -INFINITY;
    }
    return;
  }
  const Work w = work_of(p, blockIdx.x);
  if (!w.live) return;
  const Seq s = seq_of(p, w.b);
  const int M = s.nq * p.rep;
  const int nt = (s.nk + BN - 1) / BN;
  int lo = 0, hi = nt;
  if (SPLIT) {
    const int per = (nt + p.nsplit - 1) / p.nsplit;
    lo = min(w.split * per, nt);
    hi = min(lo + per, nt);
  }
  const float c = p.scale * kLog2e;

  for (int t = w.t; (long)t * BM < M; t += p.tiles) {
    const int m = t * BM + wave * 32 + (lane & 31);
    const bool live = m < M, wave_live = t * BM + wave * 32 < M;
    typename Op<T>::Frag qf[KS];
    load_row<T, HDP>(qf, (const T*)p.q + (live ? m_offset(p, s, w.g, m, p.ldq) : 0), live, p.hd, h);
    f32x16_t o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
    float mrun = -INFINITY, l = 0.f;
    Tiles<T, HDP, BN, NT> kt_(p, s, w.g, smem);
    kt_.begin(lo, hi, tid);
    for (int kt = lo; kt < hi; ++kt) {
      const T *Ks, *Vs;
      const float* bias;
      const bool masked = kt_.next(kt, hi, tid, Ks, Vs, bias);
      if (wave_live) {
        f32x16_t sc[NB];
        __builtin_amdgcn_s_setprio(1);                 // (the wave at its products goes before the one at its softmax: 162 -> 158 us for 16 pairs of 4096 on 3136, hd 128)
#pragma unroll
        for (int b = 0; b < NB; ++b) sc[b] = mma_row<T, HDP>(Ks, b * 32, qf, lane);
        __builtin_amdgcn_s_setprio(0);
        if (masked) {
#pragma unroll
          for (int b = 0; b < NB; ++b) mask_keys(sc[b], bias + b * 32, h);
        }
        float mx = sc[0][0];
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int i = 0; i < 16; ++i) mx = fmaxf(mx, sc[b][i]);
        mx = half_max(mx) * c;
        // the running maximum follows only when a score passes it by 2^8: p stays below 2^8, and most tiles leave the sums as they are
        const bool up = mx > mrun + 8.f;
        if (__any(up)) {
          const float mnew = up ? mx : mrun, alpha = mrun == -INFINITY ? 0.f : exp2_fast(mrun - mnew);
          mrun = mnew;
          l *= alpha;
#pragma unroll
          for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[d][i] *= alpha;
        }
        const float ms = mrun == -INFINITY ? 0.f : mrun;
        float sum = 0.f;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float e = exp2_fast(fmaf(sc[b][i], c, -ms));
            sc[b][i] = e;
            sum += e;
          }
        l += sum;                                      // this half-wave's keys; joined behind the loop
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const typename Op<T>::PF pf = Op<T>::pack(sc[b]);
#pragma unroll
          for (int d = 0; d < DB; ++d) Op<T>::template mma_t<HDP>(o[d], Vs, b * 32, d * 32, pf, lane);
        }
        __builtin_amdgcn_s_setprio(0);
      }
      __syncthreads();                                 // this buffer is read, the other one written
    }
    l += other_half(l);
    const long stat = live ? m_stat(p, s, w.g, m) : 0;
    if (SPLIT) {
      const long base = (long)w.split * p.heads * p.rows_q;
      if (live && h == 0) { p.part_ml[2 * (base + stat)] = mrun; p.part_ml[2 * (base + stat) + 1] = l; }
      if (lo < hi)
        rows_out<float, HDP>(smem, o, 1.f, p.hd, tid, [&](int r) -> float* { return t * BM + r < M ? p.part_o + (base + m_stat(p, s, w.g, t * BM + r)) * p.hd : nullptr; });
    } else {
      if (live && h == 0) p.lse[stat] = l == 0.f ? -INFINITY : (mrun + __log2f(l)) * kLn2;
      rows_out<T, HDP>(smem, o, l == 0.f ? 0.f : 1.f / l, p.hd, tid,
                       [&](int r) -> T* { return t * BM + r < M ? (T*)p.out + m_offset(p, s, w.g, t * BM + r, p.ldo) : nullptr; });
    }
  }
}

// Joins the key ranges of a (query row, head): o = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s, in a fixed order.
// Few ranges: a thread per 4 columns, all of its loads independent.
template <typename T>
__global__ __launch_bounds__(256) void xattn_join_kernel(XP p) {
  int first = 0, last = p.rows_q;
  if (p.cu_q) owned(p.cu_q, p.batch, p.rows_q, first, last);
  const int nch = p.hd / 4;
  const long n = (long)(last - first) * p.heads * nch, stride = (long)p.heads * p.rows_q;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) {
    const long pair = i / nch;
    const int c = (int)(i - pair * nch) * 4, row = first + (int)(pair / p.heads), head = (int)(pair % p.heads);
    const long stat = (long)head * p.rows_q + row;
    float m = -INFINITY;
#pragma unroll 4
    for (int s = 0; s < p.nsplit; ++s) m = fmaxf(m, p.part_ml[2 * (s * stride + stat)]);
    const float ms = m == -INFINITY ? 0.f : m;
    float l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int s = 0; s < p.nsplit; ++s) {
      const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + 2 * (s * stride + stat));
      const float4 v = *reinterpret_cast<const float4*>(p.part_o + (s * stride + stat) * p.hd + c);
      const float f = exp2_fast(ml.x - ms);
      l = fmaf(f, ml.y, l);
      if (ml.y != 0.f) { o.x = fmaf(f, v.x, o.x); o.y = fmaf(f, v.y, o.y); o.z = fmaf(f, v.z, o.z); o.w = fmaf(f, v.w, o.w); }   // (an empty range wrote no sums)
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    Op<T>::store4((T*)p.out + (long)row * p.ldo + (long)head * p.hd + c, o.x * inv, o.y * inv, o.z * inv, o.w * inv);
    if (c == 0) p.lse[stat] = l == 0.f ? -INFINITY : (m + __log2f(l)) * kLn2;
  }
}
// Many ranges of few pairs: a block per pair, its waves take every fourth range, eight loads of a lane at a time.
template <typename T>
__global__ __launch_bounds__(256) void xattn_join_many_kernel(XP p) {
  __shared__ float2 part_sum[4][64];
  int first = 0, last = p.rows_q;
  if (p.cu_q) owned(p.cu_q, p.batch, p.rows_q, first, last);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c0 = 2 * lane;
  const long n = (long)(last - first) * p.heads, stride = (long)p.heads * p.rows_q;
  for (long i = blockIdx.x; i < n; i += gridDim.x) {
    const int row = first + (int)(i / p.heads), head = (int)(i % p.heads);
    const long stat = (long)head * p.rows_q + row;
    float2 ml = make_float2(-INFINITY, 0.f);
    if (lane < p.nsplit) ml = *reinterpret_cast<const float2*>(p.part_ml + 2 * (lane * stride + stat));
    const float m = wave_max(ml.x), f = ml.y == 0.f ? 0.f : exp2_fast(ml.x - m), l = wave_sum(f * ml.y);
    float2 acc = make_float2(0.f, 0.f);
    const float* part = p.part_o + stat * p.hd + (c0 < p.hd ? c0 : 0);
    for (int s0 = wave; s0 < p.nsplit; s0 += 32) {
      float2 v[8];
      float fs[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int s = min(s0 + 4 * k, p.nsplit - 1);
        v[k] = *reinterpret_cast<const float2*>(part + s * stride * p.hd);
        fs[k] = s0 + 4 * k < p.nsplit ? __shfl(f, s, 64) : 0.f;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (fs[k] != 0.f) {
          acc.x = fmaf(fs[k], v[k].x, acc.x);
          acc.y = fmaf(fs[k], v[k].y, acc.y);
        }
    }
    __syncthreads();
    part_sum[wave][lane] = acc;
    __syncthreads();
    if (wave) continue;
    acc = part_sum[0][lane];
#pragma unroll
    for (int k = 1; k < 4; ++k) { acc.x += part_sum[k][lane].x; acc.y += part_sum[k][lane].y; }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T* o = (T*)p.out + (long)row * p.ldo + (long)head * p.hd + c0;
    if (c0 < p.hd) { st<T>(o, acc.x * inv); st<T>(o + 1, acc.y * inv); }
    if (lane == 0) p.lse[stat] = l == 0.f ? -INFINITY : (m + __log2f(l)) * kLn2;
  }
}

// gradients whose other axis was split: the ranges' sums added in ascending order, times f.  part [nsplit][rows][width] fp32 -> out [rows][width]
template <typename T>
__global__ __launch_bounds__(256) void xattn_sum_kernel(const float* part, T* out, long ldo, int rows, int width, int nsplit, float f, const int* cu, int batch) {
  int first = 0, last = rows;
  if (cu) owned(cu, batch, rows, first, last);
  const int nch = width / 4;
  const long n = (long)(last - first) * nch, stride = (long)rows * width;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) {
    const long row = first + i / nch;
    const int c = (int)(i % nch) * 4;
    const float* x = part + row * width + c;
    float4 s = *reinterpret_cast<const float4*>(x);
#pragma unroll 4
    for (int k = 1; k < nsplit; ++k) {
      const float4 v = *reinterpret_cast<const float4*>(x + k * stride);
      s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
    }
    Op<T>::store4(out + row * ldo + c, s.x * f, s.y * f, s.z * f, s.w * f);
  }
}

// a value the compiler knows nothing about: what follows from it is computed again where it is used
__device__ __forceinline__ int opaque(int v) {
#ifndef DH_HOST_EMU
  asm volatile("" : "+v"(v));
#endif
  return v;
}

// ------------------------------------------------------------------------------------------ backward: dq (and D)
// D = sum(do o) = sum p dp.  Where the softmax has most of its weight on a few keys dp - D cancels, and a D formed from o as it was rounded to bf16 is off by
// more than dS's own rounding: dq and dk by 7.8e-3 of their norm instead of 2.3e-3 (hd 64, 40 rows, q and k of deviation 3, 33 keys or more; two keys left
// of 700: 3.9e-3 instead of 2.0e-3).  So bf16 sums p dp itself over all keys in front of the pass that forms dS, S and dP formed twice: 36 -> 54 us for
// the captions, 191 -> 315 for the 16 pairs of 4096 rows.  fp32, whose o is as exact as p dp is, reads o.
// WHOLE: a block meets all keys, twice.  RANGE: the keys in ranges, each range's dq a partial sum; in front of it (bf16) RANGE_D, whose blocks leave their
// range's share of D.
enum Part { WHOLE, RANGE, RANGE_D };
template <typename T, int HDP, int RW, int BN, Part PART>
__global__ __launch_bounds__(64 * RW, (waves_dq<T, HDP, RW>())) void xattn_dq_kernel(XP p) {
  constexpr int EPC = Op<T>::EPC, KS = HDP / (2 * EPC), DB = HDP / 32, NB = BN / 32, BM = 32 * RW, NT = 64 * RW;
  constexpr bool SPLIT = PART != WHOLE, OWN_D = sizeof(T) == 2 && PART != RANGE;      // OWN_D: this block sums p dp over its keys
  DH_DYN_LDS_A16(unsigned char, smem);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;
  if ((int)blockIdx.x >= p.main_blocks) {
    int first, last;
    owned(p.cu_q, p.batch, p.rows_q, first, last);
    clear_rows<T>((T*)p.dq, p.lddq, p.heads * p.hd, first, last, p.rows_q, blockIdx.x - p.main_blocks, gridDim.x - p.main_blocks, tid, NT);
    return;
  }
  const Work w = work_of(p, blockIdx.x);
  if (!w.live) return;
  const Seq s = seq_of(p, w.b);
  const int M = s.nq * p.rep, nt = (s.nk + BN - 1) / BN;
  const int per = SPLIT ? (nt + p.nsplit - 1) / p.nsplit : nt, lo = SPLIT ? min(w.split * per, nt) : 0, hi = SPLIT ? min(lo + per, nt) : nt;   // this block's key tiles
  const float c = p.scale * kLog2e;
  for (int t = w.t; (long)t * BM < M; t += p.tiles) {
    const int m = t * BM + wave * 32 + (lane & 31);
    const bool live = m < M, wave_live = t * BM + wave * 32 < M;
    const long stat = live ? m_stat(p, s, w.g, m) : 0;
    const float lse = live ? p.lse[stat] : -INFINITY;
    const bool has = live && lse != -INFINITY;       // a row without a key: no gradient, whatever do holds
    const float lse2 = has ? lse * kLog2e : INFINITY;
    typename Op<T>::Frag qf[KS], df[KS];
    load_row<T, HDP>(qf, (const T*)p.q + (has ? m_offset(p, s, w.g, m, p.ldq) : 0), has, p.hd, h);
    load_row<T, HDP>(df, (const T*)p.dout + (has ? m_offset(p, s, w.g, m, p.lddo) : 0), has, p.hd, h);
    Tiles<T, HDP, BN, NT> kt_(p, s, w.g, smem);
    const T *Ks, *Vs;
    const float* bias;
    bool masked;
    auto p_dp = [&](int b, f32x16_t& sc, f32x16_t& dp, int lane) {     // p and dp of 32 keys
      sc = mma_row<T, HDP>(Ks, b * 32, qf, lane);
      dp = mma_row<T, HDP>(Vs, b * 32, df, lane);
      if (masked) mask_keys(sc, bias + b * 32, lane >> 5);
#pragma unroll
      for (int i = 0; i < 16; ++i) sc[i] = exp2_fast(fmaf(sc[i], c, -lse2));
    };
    float D = 0.f;
    if constexpr (OWN_D) {
      const int tid = opaque(threadIdx.x), lane = tid & 63;    // (places in the tiles that the two passes do not share: shared, they spill in the second)
      kt_.begin(lo, hi, tid);
      for (int kt = lo; kt < hi; ++kt) {
        masked = kt_.next(kt, hi, tid, Ks, Vs, bias);
        if (wave_live) {
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            f32x16_t sc, dp;
            p_dp(b, sc, dp, lane);
#pragma unroll
            for (int i = 0; i < 16; ++i) D = fmaf(sc[i], dp[i], D);
          }
        }
        __syncthreads();
      }
      D += other_half(D);
    } else if constexpr (sizeof(T) == 2) {
      if (live)
        for (int i = 0; i < p.nsplit; ++i) D += p.part_d[(long)i * p.heads * p.rows_q + stat];
    } else {
      typename Op<T>::Frag of[KS];
      load_row<T, HDP>(of, (const T*)p.o + (has ? m_offset(p, s, w.g, m, p.ldo) : 0), has, p.hd, h);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) D += Op<T>::dot(df[ks], of[ks]);
      D += other_half(D);
    }
    if constexpr (PART == RANGE_D) {
      if (live && h == 0) p.part_d[(long)w.split * p.heads * p.rows_q + stat] = D;
      continue;
    }
    if (live && h == 0 && (!SPLIT || w.split == 0)) p.delta[stat] = D;
    f32x16_t dq[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) dq[d][i] = 0.f;
    if (!OWN_D || hi - lo > 1) kt_.begin(lo, hi, tid);         // (an only tile is still in LDS)
    for (int kt = lo; kt < hi; ++kt) {
      masked = kt_.next(kt, hi, tid, Ks, Vs, bias);
      if (wave_live) {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          f32x16_t sc, dp;
          p_dp(b, sc, dp, lane);
#pragma unroll
          for (int i = 0; i < 16; ++i) sc[i] *= dp[i] - D;
          const typename Op<T>::PF pf = Op<T>::pack(sc);
#pragma unroll
          for (int d = 0; d < DB; ++d) Op<T>::template mma_t<HDP>(dq[d], Ks, b * 32, d * 32, pf, lane);
        }
      }
      __syncthreads();
    }
    if (SPLIT) {
      float* part = p.part_o + (long)w.split * p.rows_q * p.heads * p.hd;
      rows_out<float, HDP>(smem, dq, 1.f, p.hd, tid, [&](int r) -> float* { return t * BM + r < M ? part + m_offset(p, s, w.g, t * BM + r, (long)p.heads * p.hd) : nullptr; });
    } else {
      rows_out<T, HDP>(smem, dq, p.scale, p.hd, tid, [&](int r) -> T* { return t * BM + r < M ? (T*)p.dq + m_offset(p, s, w.g, t * BM + r, p.lddq) : nullptr; });
    }
  }
}

// ------------------------------------------------------------------------------------------ backward: dk, dv
template <typename T, int HDP, int RW, bool SPLIT>
__global__ __launch_bounds__(64 * RW, (waves_dkv<T, HDP, RW>())) void xattn_dkv_kernel(XP p) {
  constexpr int EPC = Op<T>::EPC, LD = Lay<T, HDP>::LD, KS = HDP / (2 * EPC), DB = HDP / 32, BQ = 32, BK = 32 * RW, NT = 64 * RW;
  DH_DYN_LDS_A16(unsigned char, smem);
  T* buf = reinterpret_cast<T*>(smem);                 // two buffers of Q and dO rows, lse and D of the rows
  float* stats = reinterpret_cast<float*>(buf + 4 * BQ * LD);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;
  if ((int)blockIdx.x >= p.main_blocks) {
    int first, last;
    owned(p.cu_kv, p.batch, p.rows_kv, first, last);
    const int blk = blockIdx.x - p.main_blocks, nblk = gridDim.x - p.main_blocks;
    clear_rows<T>((T*)p.dk, p.lddk, p.kv_heads * p.hd, first, last, p.rows_kv, blk, nblk, tid, NT);
    clear_rows<T>((T*)p.dv, p.lddv, p.kv_heads * p.hd, first, last, p.rows_kv, blk, nblk, tid, NT);
    return;
  }
  const Work w = work_of(p, blockIdx.x);
  if (!w.live) return;
  const Seq s = seq_of(p, w.b);
  const int M = s.nq * p.rep, nt = (M + BQ - 1) / BQ;
  const int per = SPLIT ? (nt + p.nsplit - 1) / p.nsplit : nt, lo = SPLIT ? min(w.split * per, nt) : 0, hi = SPLIT ? min(lo + per, nt) : nt;   // this block's row tiles
  const float c = p.scale * kLog2e;
  for (int t = w.t; (long)t * BK < s.nseg; t += p.tiles) {
    const int key = t * BK + wave * 32 + (lane & 31);
    const bool live = key < s.nk && (!p.key_mask || p.key_mask[s.k0 + key]);
    const bool wave_live = t * BK + wave * 32 < s.nk, block_live = t * BK < s.nk;
    typename Op<T>::Frag kf[KS], vf[KS];
    load_row<T, HDP>(kf, (const T*)p.k + (live ? (long)(s.k0 + key) * p.ldk + (long)w.g * p.hd : 0), live, p.hd, h);
    load_row<T, HDP>(vf, (const T*)p.v + (live ? (long)(s.k0 + key) * p.ldv + (long)w.g * p.hd : 0), live, p.hd, h);
    f32x16_t dk[DB], dv[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) dk[d][i] = dv[d][i] = 0.f;
    Pair2<T, HDP, BQ, NT> st;
    float nlse = 0.f, ndel = 0.f;
    auto fetch = [&](int mt, int tid) {
      const int m0 = mt * BQ;
      int q0, r0;
      m_split(p, m0, q0, r0);                          // (uniform: the tile's first row)
      auto off = [&](int r, long ld) { int q, x; m_split(p, m0 + r, q, x); return (q - q0) * (int)ld + x * p.hd; };
      st.fetch((const T*)p.q + (long)(s.q0 + q0) * p.ldq + (long)w.g * p.rep * p.hd, (const T*)p.dout + (long)(s.q0 + q0) * p.lddo + (long)w.g * p.rep * p.hd,
               [&](int r) { return off(r, p.ldq); }, [&](int r) { return off(r, p.lddo); }, M - 1 - m0, nullptr, p.hd, tid);
      if (tid < BQ) {
        const long stat = m_stat(p, s, w.g, min(mt * BQ + tid, M - 1));
        nlse = p.lse[stat];
        ndel = p.delta[stat];
      }
    };
    auto store = [&](int mt, int tid) {
      T* b = buf + (mt & 1) * 2 * BQ * LD;
      st.store(b, b + BQ * LD, (mt + 1) * BQ > M || p.hd < HDP, mt * BQ, M - 1, false, p.hd, tid);
      if (tid < BQ) {
        float* x = stats + (mt & 1) * 2 * BQ + tid;
        x[0] = mt * BQ + tid < M && nlse != -INFINITY ? nlse * kLog2e : INFINITY;      // rows that are none, rows without a key: p = 0
        x[BQ] = ndel;
      }
    };
    const int hi_mt = block_live ? hi : lo;
    if (lo < hi_mt) {
      fetch(lo, tid);
      store(lo, tid);
    }
    if constexpr (sizeof(T) == 2) { arrived(kf); arrived(vf); }      // (fp32, with accumulation registers to spare, is 3 % slower with it)
    if (lo + 1 < hi_mt) fetch(lo + 1, tid);
    if (lo < hi_mt) __syncthreads();
    for (int mt = lo; mt < hi_mt; ++mt) {
      // A thread's places in the tiles are formed anew on every turn where kept ones are spilled, a reload waiting for all loads under way: more than 64
      // columns (16 pairs of 4096 rows on 3136 keys, hd 128: 353 -> 312 us) and blocks of one wave (captions 59.7 -> 58.5 us; 197 rows on up to 77 keys 42.5 -> 44.4).
      // Four waves of up to 64 columns have the registers: formed anew 30.2 / 36.4 us, kept 29.0 / 34.8 (16 x 512 on 512 / 32 x 197 on 577, 8 heads).
      const int tid = HDP > 64 || RW == 1 ? opaque(threadIdx.x) : (int)threadIdx.x, lane = tid & 63, h = lane >> 5;
      if (mt + 1 < hi_mt) {
        store(mt + 1, tid);
        if (mt + 2 < hi_mt) fetch(mt + 2, tid);
      }
      if (wave_live) {
        const T *Qs = buf + (mt & 1) * 2 * BQ * LD, *Ds = Qs + BQ * LD;
        const float *lse2s = stats + (mt & 1) * 2 * BQ, *dels = lse2s + BQ;
        f32x16_t sc = mma_row<T, HDP>(Qs, 0, kf, lane);
        f32x16_t dp = mma_row<T, HDP>(Ds, 0, vf, lane);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float4 L = *reinterpret_cast<const float4*>(lse2s + 8 * i + 4 * h);
          const float4 D = *reinterpret_cast<const float4*>(dels + 8 * i + 4 * h);
          sc[4 * i] = exp2_fast(fmaf(sc[4 * i], c, -L.x)); dp[4 * i] = sc[4 * i] * (dp[4 * i] - D.x);
          sc[4 * i + 1] = exp2_fast(fmaf(sc[4 * i + 1], c, -L.y)); dp[4 * i + 1] = sc[4 * i + 1] * (dp[4 * i + 1] - D.y);
          sc[4 * i + 2] = exp2_fast(fmaf(sc[4 * i + 2], c, -L.z)); dp[4 * i + 2] = sc[4 * i + 2] * (dp[4 * i + 2] - D.z);
          sc[4 * i + 3] = exp2_fast(fmaf(sc[4 * i + 3], c, -L.w)); dp[4 * i + 3] = sc[4 * i + 3] * (dp[4 * i + 3] - D.w);
        }
        const typename Op<T>::PF pf = Op<T>::pack(sc), sf = Op<T>::pack(dp);
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          Op<T>::template mma_t<HDP>(dv[d], Ds, 0, d * 32, pf, lane);
          Op<T>::template mma_t<HDP>(dk[d], Qs, 0, d * 32, sf, lane);
        }
      }
      __syncthreads();
    }
    // (a masked key's column may hold anything: it is written as zeros)
    if (!live)
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) dk[d][i] = dv[d][i] = 0.f;
    if (SPLIT) {
      const long width = (long)p.kv_heads * p.hd, all = (long)p.rows_kv * width;
      float* part = p.part_o + (long)w.split * all;
      auto row = [&](float* x, int r) -> float* { return t * BK + r < s.nseg ? x + (long)(s.k0 + t * BK + r) * width + (long)w.g * p.hd : nullptr; };
      rows_out<float, HDP>(smem, dk, 1.f, p.hd, tid, [&](int r) { return row(part, r); });
      rows_out<float, HDP>(smem, dv, 1.f, p.hd, tid, [&](int r) { return row(part + p.nsplit * all, r); });
    } else {
      auto row = [&](T* x, long ld, int r) -> T* { return t * BK + r < s.nseg ? x + (long)(s.k0 + t * BK + r) * ld + (long)w.g * p.hd : nullptr; };
      rows_out<T, HDP>(smem, dk, p.scale, p.hd, tid, [&](int r) { return row((T*)p.dk, p.lddk, r); });
      rows_out<T, HDP>(smem, dv, 1.f, p.hd, tid, [&](int r) { return row((T*)p.dv, p.lddv, r); });
    }
  }
}

// ------------------------------------------------------------------------------------------ host side
int x_cus() {
  static int n = 0;
  if (!n) {
    int dev = 0;
    hipDeviceProp_t pr;
    n = (hipGetDevice(&dev) == hipSuccess && hipGetDeviceProperties(&pr, dev) == hipSuccess && pr.multiProcessorCount > 0) ? pr.multiProcessorCount : 256;
  }
  return n;
}

int64_t cdiv64(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t round4(int64_t n) { return (n + 3) & ~(int64_t)3; }

// longest length to lay the grid out for: the caller's bound, or twice the mean of a packed batch (longer ones take several rounds)
int length_hint(int given, const int* cu, int rows, int batch) {
  if (!cu) return rows / batch;
  int64_t n = given > 0 ? given : 2 * cdiv64(rows, batch);
  return (int)(n > rows ? rows : n);
}

enum Kind { FWD, DQ, DKV };
// Waves of 32 rows per block; they share the tiles of the other axis.  Long axes want many (less staging per row), short ones few: blocks of one wave
// wait for nobody and more sequences are under way at a time.  Measured in us (bf16, one / two / four waves): 2048 (sequence, head) pairs of 5 .. 77 rows
// on 197 keys fwd 31 / 39 / 42, dq 36 / 52 / 48, dkv 58 / 60 / 62; 197 rows on 5 .. 77 keys fwd 42 / 37 / 48, dq 58 / 65 / 72; 128 pairs of 512 on 512 fwd
// 26 / 23 / 18, dkv 39 / 32 / 29; 24 pairs of 2047 on 6272 fwd 226 / 198 / 147.
// More than 64 columns: eight waves (half of the staging registers each, two waves per SIMD) once they are filled: 16 pairs of 4096 rows on 3136 keys fwd
// 164 (four: 170), dq 191 (319), dkv 382 (612; both before the padding and the spill-free loop below, dq without the pass for D).  fp32: four, but one for up to
// 32 rows, although the shapes of more than 64 columns spill there (hd 128: up to 173 / 255 / 495 registers): 64 sequences of one token on up to 3136 keys, hd 64
// 70 us (four: 136), hd 80 169 (202), hd 128 290 (346); 512 pairs of 20 rows on 20 keys, hd 128 fwd 22.9 (22.8), dq 40 (29), dkv 40 (38), hd 64 9.0 (9.2), 12.2
// (11.3), 11.3 (18.4).  bf16, hd 128, 4096 rows on 30 keys (one wave, rows in ranges, 278 spilled): dkv 48 us and two sums of 4.6.
int row_waves(const dh_xattn_args* a, Kind kind, int64_t rows, int64_t other) {
  if (rows <= 32) return 1;
  if (a->dtype == DH_F32) return 4;
  if (a->hd <= 64) return rows <= 128 || other <= 256 ? 1 : 4;
  if (kind == DKV && a->hd > 96 && other <= 128) return 2;
  if (rows > 128) return 8;
  return kind == DQ ? 1 : 4;
}
// A launch over (sequence, kv head) pairs: `rows` of one axis in tiles of rw 32; the other axis (`other` long) split in ranges of at least `step` where
// the tiles alone leave compute units idle.
struct Plan { int rw, tiles, nsplit; };
Plan plan_of(const dh_xattn_args* a, Kind kind, int64_t rows, int64_t other, int step) {
  Plan r;
  r.rw = row_waves(a, kind, rows, other);
  r.tiles = (int)cdiv64(rows < 1 ? 1 : rows, 32 * r.rw);
  // Two waves per SIMD; the forward of up to 64 columns fits three, and with ranges of 1024 keys and more their partial results cost less than they
  // bring (24 pairs of 2047 on 6272: 161 us whole, 104 + 9 us in two ranges).  That is 384 blocks, the most that still split; 48 and 96 pairs run whole, two
  // waves per SIMD, in 280-297 and 445 us.
  const bool three = kind == FWD && a->dtype == DH_BF16 && a->hd <= 64 && r.rw == 4 && other >= 2048;
  const int64_t blocks = (int64_t)r.tiles * a->batch * a->kv_heads, want = (int64_t)x_cus() * ((three ? 12 : 8) / r.rw);
  if (three) step = 1024;
  int64_t ns = blocks >= want ? 1 : want / blocks;
  const int64_t most = cdiv64(other, step);
  if (ns > most) ns = most;
  if (ns > 64) ns = 64;
  r.nsplit = ns < 1 ? 1 : (int)ns;
  return r;
}
int64_t longest_m(const dh_xattn_args* a) { return (int64_t)length_hint(a->max_q, a->cu_q, a->rows_q, a->batch) * (a->heads / a->kv_heads); }
int longest_k(const dh_xattn_args* a) { return length_hint(a->max_kv, a->cu_kv, a->rows_kv, a->batch); }
// forward and dq split the keys, dkv the query rows; a range is at least 128 (fwd) / 256 long: its partial result costs as much as a few tiles
Plan plan_fwd(const dh_xattn_args* a) { return plan_of(a, FWD, longest_m(a), longest_k(a), 128); }
Plan plan_dq(const dh_xattn_args* a) { return plan_of(a, DQ, longest_m(a), longest_k(a), 256); }
Plan plan_dkv(const dh_xattn_args* a) { return plan_of(a, DKV, longest_k(a), longest_m(a), 256); }

int check_geometry(const dh_xattn_args* a, const char* who) {
  DH_REQUIRE(a, "%s: null args", who);
  DH_REQUIRE(a->dtype == DH_F32 || a->dtype == DH_BF16, "%s: dtype %d", who, a->dtype);
  DH_REQUIRE(a->batch > 0 && a->heads > 0 && a->kv_heads > 0 && a->heads % a->kv_heads == 0, "%s: batch %d, heads %d, kv_heads %d", who, a->batch, a->heads, a->kv_heads);
  DH_REQUIRE(a->hd >= 8 && a->hd <= 128 && a->hd % 8 == 0, "%s: head size %d (a multiple of 8 up to 128)", who, a->hd);
  DH_REQUIRE(a->rows_q >= 0 && a->rows_kv >= 0, "%s: negative row count", who);
  DH_REQUIRE(a->cu_q || a->rows_q % a->batch == 0, "%s: %d query rows do not divide into %d sequences", who, a->rows_q, a->batch);
  DH_REQUIRE(a->cu_kv || a->rows_kv % a->batch == 0, "%s: %d key rows do not divide into %d sequences", who, a->rows_kv, a->batch);
  DH_REQUIRE(a->scale > 0.f && a->scale < INFINITY, "%s: scale must be positive and finite", who);
  DH_REQUIRE((int64_t)a->rows_q * (a->heads / a->kv_heads) < (1ll << 30) && a->rows_kv < (1 << 30), "%s: too many rows", who);
  return DH_OK;
}
int check_args(const dh_xattn_args* a, const char* who, bool bwd) {
  if (int e = check_geometry(a, who)) return e;
  const int epc = a->dtype == DH_BF16 ? 8 : 4;
  const int64_t wq = (int64_t)a->heads * a->hd, wk = (int64_t)a->kv_heads * a->hd;
  struct { const void* p; int64_t ld, w; bool need; const char* name; } m[] = {
      {a->q, a->ldq, wq, a->rows_q > 0, "q"},       {a->k, a->ldk, wk, a->rows_kv > 0, "k"},          {a->v, a->ldv, wk, a->rows_kv > 0, "v"},
      {a->out, a->ldo, wq, a->rows_q > 0, "out"},   {a->dout, a->lddo, wq, bwd && a->rows_q > 0, "dout"}, {a->dq, a->lddq, wq, bwd && a->rows_q > 0, "dq"},
      {a->dk, a->lddk, wk, bwd && a->rows_kv > 0, "dk"}, {a->dv, a->lddv, wk, bwd && a->rows_kv > 0, "dv"}};
  for (const auto& x : m) {
    if (!x.need) continue;
    DH_REQUIRE(x.p, "%s: %s is NULL", who, x.name);
    DH_REQUIRE(((uintptr_t)x.p & 15) == 0 && x.ld >= x.w && x.ld % epc == 0 && x.ld < (1 << 22), "%s: %s needs 16-byte aligned rows, row strides up to 2^22 (row stride %lld, width %lld)", who, x.name,
               (long long)x.ld, (long long)x.w);
  }
  DH_REQUIRE(a->lse || a->rows_q == 0, "%s: lse is NULL", who);
  return DH_OK;
}

XP params(const dh_xattn_args* a) {
  XP p = {};
  p.q = a->q; p.k = a->k; p.v = a->v; p.o = a->out; p.dout = a->dout;
  p.out = a->out; p.dq = a->dq; p.dk = a->dk; p.dv = a->dv; p.lse = a->lse;
  p.cu_q = a->cu_q; p.cu_kv = a->cu_kv; p.kv_len = a->kv_len; p.key_mask = a->key_mask;
  p.ldq = a->ldq; p.ldk = a->ldk; p.ldv = a->ldv; p.ldo = a->ldo; p.lddo = a->lddo; p.lddq = a->lddq; p.lddk = a->lddk; p.lddv = a->lddv;
  p.rows_q = a->rows_q; p.rows_kv = a->rows_kv; p.batch = a->batch; p.heads = a->heads; p.kv_heads = a->kv_heads; p.rep = a->heads / a->kv_heads; p.hd = a->hd;
  p.scale = a->scale;
  p.magic = p.rep > 1 ? (unsigned)(((1ull << 32) + p.rep - 1) / p.rep) : 0u;
  p.nsplit = 1;
  return p;
}

// grid of a kernel over (sequence, kv head) pairs; `clear`: blocks behind it for the rows no sequence owns
int lay_out(XP& p, const Plan& pl, bool clear, int64_t& grid) {
  const int tiles = pl.tiles, nsplit = pl.nsplit;
  const int64_t pairs = (int64_t)p.batch * p.kv_heads;
  p.tiles = tiles < 1 ? 1 : tiles;
  p.nsplit = nsplit;
  p.by_pair = pairs % 8 == 0 || pairs >= 64;
  const int64_t main = (p.by_pair ? cdiv64(pairs, 8) * 8 : pairs) * p.tiles * nsplit;
  DH_REQUIRE((main + 64) * 64 * pl.rw < (1ll << 32), "dh_xattn: grid of %lld blocks", (long long)main);      // (a launch holds 2^32 threads)
  p.main_blocks = (int)main;
  grid = main + (clear ? 64 : 0);
  return DH_OK;
}

template <typename K>
int launch(K kernel, const XP& p, int64_t grid, int threads, size_t lds, hipStream_t st) {
  if (lds > 64 * 1024) DH_RT(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds), "hipFuncSetAttribute");
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(threads), lds, st, p);
  DH_CHECK_LAUNCH();
  return DH_OK;
}

// LDS of a block: two buffers of two tiles with `per_row` floats beside each tile row; the result rows go through it at the end (fp32 where split)
template <typename T, int HDP, int RW> constexpr size_t lds_bytes(int rows, int per_row, bool split) {
  const size_t tiles = 2 * ((size_t)2 * rows * Lay<T, HDP>::LD * sizeof(T) + (size_t)rows * per_row * 4);
  const size_t out = split || sizeof(T) == 4 ? (size_t)RW * 32 * (HDP + 4) * 4 : (size_t)RW * 32 * (HDP + Op<T>::EPC) * sizeof(T);
  return tiles > out ? tiles : out;
}
int no_shape(int rw) { DH_FAIL(DH_ERR_ARG, "dh_xattn: no blocks of %d waves at this width", rw); }
template <typename T, int HDP, int RW, int BN>
int fwd_shape(XP& p, int64_t grid, hipStream_t st) {
  static_assert(lds_bytes<T, HDP, RW>(BN, 1, true) <= 160 * 1024, "LDS");
  const size_t lds = lds_bytes<T, HDP, RW>(BN, 1, p.nsplit > 1);
  return p.nsplit > 1 ? launch(xattn_fwd_kernel<T, HDP, RW, BN, true>, p, grid, 64 * RW, lds, st) : launch(xattn_fwd_kernel<T, HDP, RW, BN, false>, p, grid, 64 * RW, lds, st);
}
template <typename T, int HDP, int RW, int BN>
int dq_shape(XP& p, int64_t grid, hipStream_t st) {
  const size_t lds = lds_bytes<T, HDP, RW>(BN, 1, p.nsplit > 1);
  if (p.nsplit == 1) return launch(xattn_dq_kernel<T, HDP, RW, BN, WHOLE>, p, grid, 64 * RW, lds, st);
  if constexpr (sizeof(T) == 2)
    if (int e = launch(xattn_dq_kernel<T, HDP, RW, BN, RANGE_D>, p, p.main_blocks, 64 * RW, lds, st)) return e;
  return launch(xattn_dq_kernel<T, HDP, RW, BN, RANGE>, p, grid, 64 * RW, lds, st);
}
template <typename T, int HDP, int RW>
int dkv_shape(XP& p, int64_t grid, hipStream_t st) {
  const size_t lds = lds_bytes<T, HDP, RW>(32, 2, p.nsplit > 1);
  if constexpr (RW != 2)                               // (two waves: up to 128 query rows, half of the least range)
    if (p.nsplit > 1) return launch(xattn_dkv_kernel<T, HDP, RW, true>, p, grid, 64 * RW, lds, st);
  if (p.nsplit > 1) return no_shape(RW);
  return launch(xattn_dkv_kernel<T, HDP, RW, false>, p, grid, 64 * RW, lds, st);
}

// the block shapes that row_waves can ask for at this width: one and four waves; more than 64 columns of bf16 eight (dq instead of four); dk / dv of more
// than 96 also two
template <Kind K, typename T, int HDP> constexpr bool shape(int rw) {
  const bool wide = sizeof(T) == 2 && HDP > 64;
  return rw == 1 || (rw == 4 && !(wide && K == DQ)) || (rw == 8 && wide) || (rw == 2 && wide && K == DKV && HDP > 96);
}
template <typename T, int HDP>
int fwd_hd(XP& p, int rw, int64_t grid, hipStream_t st) {
  constexpr int BN = sizeof(T) == 2 ? 64 : 32;
  if (rw == 1) return fwd_shape<T, HDP, 1, 32>(p, grid, st);
  if constexpr (shape<FWD, T, HDP>(4)) if (rw == 4) return fwd_shape<T, HDP, 4, BN>(p, grid, st);
  if constexpr (shape<FWD, T, HDP>(8)) if (rw == 8) return fwd_shape<T, HDP, 8, BN>(p, grid, st);
  return no_shape(rw);
}
template <typename T, int HDP>
int dq_hd(XP& p, int rw, int64_t grid, hipStream_t st) {
  constexpr int BN = sizeof(T) == 2 ? 64 : 32;
  if (rw == 1) return dq_shape<T, HDP, 1, 32>(p, grid, st);
  if constexpr (shape<DQ, T, HDP>(4)) if (rw == 4) return dq_shape<T, HDP, 4, BN>(p, grid, st);
  if constexpr (shape<DQ, T, HDP>(8)) if (rw == 8) return dq_shape<T, HDP, 8, BN>(p, grid, st);
  return no_shape(rw);
}
template <typename T, int HDP>
int dkv_hd(XP& p, int rw, int64_t grid, hipStream_t st) {
  if (rw == 1) return dkv_shape<T, HDP, 1>(p, grid, st);
  if constexpr (shape<DKV, T, HDP>(2)) if (rw == 2) return dkv_shape<T, HDP, 2>(p, grid, st);
  if constexpr (shape<DKV, T, HDP>(4)) if (rw == 4) return dkv_shape<T, HDP, 4>(p, grid, st);
  if constexpr (shape<DKV, T, HDP>(8)) if (rw == 8) return dkv_shape<T, HDP, 8>(p, grid, st);
  return no_shape(rw);
}

template <typename T>
int sum_out(const float* part, T* out, int64_t ld, int rows, int width, int nsplit, float f, const int* cu, int batch, hipStream_t st) {
  int64_t g = cdiv64((int64_t)rows * (width / 4), 256);
  if (g > 8 * x_cus()) g = 8 * x_cus();
  hipLaunchKernelGGL((xattn_sum_kernel<T>), dim3((unsigned)g), dim3(256), 0, st, part, out, (long)ld, rows, width, nsplit, f, cu, batch);
  DH_CHECK_LAUNCH();
  return DH_OK;
}

#define XATTN_HD(fn, T, ...) \
  (p.hd <= 32 ? fn<T, 32>(__VA_ARGS__) : p.hd <= 64 ? fn<T, 64>(__VA_ARGS__) : p.hd <= 96 ? fn<T, 96>(__VA_ARGS__) : fn<T, 128>(__VA_ARGS__))

template <typename T>
int join_ranges(const XP& p, hipStream_t st) {
  const int64_t pairs = (int64_t)p.rows_q * p.heads;
  if (p.nsplit > 8 && pairs < 16 * x_cus()) {
    hipLaunchKernelGGL((xattn_join_many_kernel<T>), dim3((unsigned)(pairs < 8 * x_cus() ? pairs : 8 * x_cus())), dim3(256), 0, st, p);
  } else {
    int64_t g = cdiv64(pairs * (p.hd / 4), 256);
    if (g > 32 * x_cus()) g = 32 * x_cus();
    hipLaunchKernelGGL((xattn_join_kernel<T>), dim3((unsigned)g), dim3(256), 0, st, p);
  }
  DH_CHECK_LAUNCH();
  return DH_OK;
}
// the ranges' shares of D
int64_t part_d_floats(const dh_xattn_args* a) {
  const int64_t ns = plan_dq(a).nsplit;
  return a->dtype == DH_BF16 && ns > 1 ? round4(ns * a->heads * a->rows_q) : 0;
}
template <typename T>
int bwd(const dh_xattn_args* a, hipStream_t st) {
  XP p = params(a);
  p.delta = (float*)a->ws;
  p.part_d = p.delta + round4((int64_t)a->heads * a->rows_q);
  p.part_o = p.part_d + part_d_floats(a);
  int64_t grid;
  if (a->rows_q > 0) {
    const Plan pl = plan_dq(a);
    if (int e = lay_out(p, pl, a->cu_q != nullptr, grid)) return e;
    if (int e = XATTN_HD(dq_hd, T, p, pl.rw, grid, st)) return e;
    if (pl.nsplit > 1)
      if (int e = sum_out<T>(p.part_o, (T*)a->dq, a->lddq, a->rows_q, a->heads * a->hd, pl.nsplit, a->scale, a->cu_q, a->batch, st)) return e;
  }
  if (a->rows_kv > 0) {
    const Plan pl = plan_dkv(a);
    if (int e = lay_out(p, pl, a->cu_kv != nullptr, grid)) return e;
    if (int e = XATTN_HD(dkv_hd, T, p, pl.rw, grid, st)) return e;
    if (pl.nsplit > 1) {
      const int width = a->kv_heads * a->hd;
      if (int e = sum_out<T>(p.part_o, (T*)a->dk, a->lddk, a->rows_kv, width, pl.nsplit, a->scale, a->cu_kv, a->batch, st)) return e;
      return sum_out<T>(p.part_o + (int64_t)pl.nsplit * a->rows_kv * width, (T*)a->dv, a->lddv, a->rows_kv, width, pl.nsplit, 1.f, a->cu_kv, a->batch, st);
    }
  }
  return DH_OK;
}

int64_t fwd_bytes(const dh_xattn_args* a) {
  const int64_t ns = plan_fwd(a).nsplit;
  return ns > 1 ? ns * a->heads * a->rows_q * (a->hd + 2) * 4 : 0;
}
int64_t bwd_bytes(const dh_xattn_args* a) {       // D, its ranges' shares, and the larger of the partial dq and the partial dk, dv
  const int64_t sq = plan_dq(a).nsplit, sk = plan_dkv(a).nsplit;
  const int64_t q = sq > 1 ? sq * a->rows_q * a->heads * a->hd : 0, kv = sk > 1 ? 2 * sk * a->rows_kv * a->kv_heads * a->hd : 0;
  return (round4((int64_t)a->heads * a->rows_q) + part_d_floats(a) + (q > kv ? q : kv)) * 4;
}

}  // namespace

extern "C" int64_t dh_xattn_ws_bytes(const dh_xattn_args* a, int backward) {
  if (check_geometry(a, "dh_xattn_ws_bytes")) return -1;
  return backward ? bwd_bytes(a) : fwd_bytes(a);
}

extern "C" int dh_xattn_fwd(const dh_xattn_args* a, dh_stream_t stream) {
  if (int e = check_args(a, "dh_xattn_fwd", false)) return e;
  if (a->rows_q == 0) return DH_OK;
  const Plan pl = plan_fwd(a);
  XP p = params(a);
  const int64_t need = fwd_bytes(a);
  DH_REQUIRE(need == 0 || (a->ws && a->ws_bytes >= need && ((uintptr_t)a->ws & 15) == 0), "dh_xattn_fwd: workspace of %lld bytes needed", (long long)need);
  if (need) {
    p.part_o = (float*)a->ws;
    p.part_ml = p.part_o + (int64_t)pl.nsplit * a->heads * a->rows_q * a->hd;
  }
  int64_t grid;
  if (int e = lay_out(p, pl, a->cu_q != nullptr, grid)) return e;
  const int rc = a->dtype == DH_BF16 ? XATTN_HD(fwd_hd, bf16_t, p, pl.rw, grid, (hipStream_t)stream) : XATTN_HD(fwd_hd, float, p, pl.rw, grid, (hipStream_t)stream);
  if (rc || pl.nsplit == 1) return rc;
  return a->dtype == DH_BF16 ? join_ranges<bf16_t>(p, (hipStream_t)stream) : join_ranges<float>(p, (hipStream_t)stream);
}

extern "C" int dh_xattn_bwd(const dh_xattn_args* a, dh_stream_t stream) {
  if (int e = check_args(a, "dh_xattn_bwd", true)) return e;
  const int64_t need = bwd_bytes(a);
  DH_REQUIRE(need == 0 || (a->ws && a->ws_bytes >= need && ((uintptr_t)a->ws & 15) == 0), "dh_xattn_bwd: workspace of %lld bytes needed", (long long)need);
  return a->dtype == DH_BF16 ? bwd<bf16_t>(a, (hipStream_t)stream) : bwd<float>(a, (hipStream_t)stream);
}
