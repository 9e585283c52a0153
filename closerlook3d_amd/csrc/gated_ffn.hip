// gated_ffn.hip -- the gated feed-forward of a point:  Y = (act(X Wg^T) * (X Wu^T)) Wd^T  and its gradients, on the matrix cores.
//
// X [R, C] point-major rows (R = clouds x points), Wg, Wu [H, C], Wd [C, H] as nn.Linear holds them.
//     G = X Wg^T, U = X Wu^T, h = act(G) U;   Y = h Wd^T
//     dh = dY Wd;  dG = dh U act'(G);  dU = dh act(G);   dX = dG Wg + dU Wu;   dWg = dG^T X, dWu = dU^T X, dWd = dY^T h
// Three products of 2 R C H operations forward and six backward.  G and U never reach memory: the forward kernel keeps both
// accumulators of an element in one lane and writes h, the backward kernel forms G, U and dh together (two products more) and
// writes dG, dU (h is kept from the forward pass where the caller has room for it, or formed again).  Against storing G and U that
// is 8 R H bytes less traffic for 4 R C H operations more -- at 5.1 TB/s and 1.28 PFLOP/s (a large copy, a large product) it pays
// below C = 500 -- and dG, dU come from f32 values of G, U, dh: one rounding in front of the last products instead of two.
// That rounding, of 16-bit tensors: h in front of Y and dWd, dG and dU in front of dX, dWg and dWu are rounded to the tensors' type.
// The matrix units take 16-bit operands, and a second plane of each (what f32 tensors have) would double six of the eleven products
// of a training pass.  Beside the rounding of the results themselves it is a second one of the same size: 2.3e-3 of a result's norm in bf16
// instead of 1.7e-3, 2.9e-4 instead of 2.1e-4 in f16, whose range is theirs too (above 65504 an infinity, below 2^-25 nothing).
//
// One kernel template.  D[j][i] = sum_k P(i, k) Q(j, k), i contiguous in the result; P is the first MFMA operand, so a lane of
// v_mfma_f32_16x16x32 holds four consecutive i of one j.
//   * tiles travel HBM -> LDS by buffer_load ... lds (16 bytes a lane, no registers); a lane behind the end of a row or of the
//     tensor is sent out of the descriptor's range and fills its place with zeros, so ragged sizes need no second kernel;
//   * two LDS tiles of 64 k each (projections: 32): the next one is in flight while this one is multiplied; a third tile would cost
//     a workgroup of the CU, and what bounds these short sums is what one workgroup cannot overlap with itself: its start, its
//     barriers, its stores (of the backward twin's 68 us, 27 are left without any product, 50 without the stores).
//   * an operand whose k is contiguous lies in LDS as [row][64 k], 16-byte pieces XORed with the row, read by ds_read_b128; one
//     whose row index is contiguous (Wd in dh, Wg / Wu in dX, all operands of the weight gradients) lies as [64 k][row] and is
//     read by ds_read_b64_tr_b16, which hands a lane four k of its row: no operand is transposed in memory;
//   * workgroups are numbered so that neighbours in i, which share the rows of Q, run on one XCD and share its L2.
// f32 tensors: an f32 value is the exact sum of three bf16 values (planes 0, 1, 2, each what is left rounded to nearest); a product
// takes the six largest of the nine partial products on the bf16 units, smallest first, into one f32 accumulator.  Plane 1 is at most
// 2^-8 of the value and plane 2 2^-17, so what is left out is below 2^-24 of |x||y|, of either sign: less than the rounding of an
// f32 product.  Six passes at the bf16 rate outrun the f32 MFMA (1/16 of it).  A tile holds the three planes of 32 k, so each
// fragment is read once for its two or three products.  A value that is not finite takes part in the product of the leading planes
// only, so an infinity stays one (not_finite below).
// Measured at 16 384 x 288 x 1152 in bf16: projections 36 us (610 TFLOP/s), their backward twin 66 (490), Y 19 (575), dX 34 (640),
// the three weight gradients 59 (555); 16 384 x 144 x 576 in f32, counting f32 operations: 61 (89), 101 (81), 25 (108), 49 (112), 74 (110).
#include "ff_common.h"
#include <type_traits>

namespace cl3d {

typedef unsigned short u16;

template <typename E> __device__ __forceinline__ f32x4 mfma16(s16x8 a, s16x8 b, f32x4 c);
template <> __device__ __forceinline__ f32x4 mfma16<Bf16>(s16x8 a, s16x8 b, f32x4 c) {
  typedef __bf16 v8 __attribute__((ext_vector_type(8)));
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
}
template <> __device__ __forceinline__ f32x4 mfma16<F16>(s16x8 a, s16x8 b, f32x4 c) {
  typedef _Float16 v8 __attribute__((ext_vector_type(8)));
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
}

#define CL3D_LDS(T, p) ((__attribute__((address_space(3))) T *)(p))

// s_waitcnt vmcnt(n), the other counters left alone; no memory operation moves across it (the count is of those issued before)
template <int N> __device__ __forceinline__ void wait_vm() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | (15 << 8) | ((N >> 4) << 14));
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
}
__device__ __forceinline__ void barrier_lds() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(15 | (7 << 4) | (3 << 14));  // lgkmcnt(0): this wave's LDS reads have returned
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// ---- one operand's way into LDS.  KM false: rows of 64 k; true: 64 rows of ROWS elements.  `swz` is the XOR of a 16-byte
// piece's place, chosen so that the 16 lanes of a fragment read cover all 64 banks: a k-contiguous fragment reads rows
// r .. r + 15 (or, PAIRED, rows 8 a + b, a and b in 0..3) of which every second starts at the same bank.
template <bool PAIRED, int BK> __device__ __forceinline__ int swz_kc(int row) {
  if (BK == 32) return PAIRED ? (row >> 3) & 3 : (row >> 2) & 3;
  return PAIRED ? (((row >> 1) & 1) | ((row >> 2) & 6)) : ((row >> 1) & 7);
}
template <int ROWS> __device__ __forceinline__ int swz_km(int k) {  // (32-byte blocks: ds_read_b64_tr_b16 takes them whole)
  if (ROWS % 128 == 0) return ((k & 3) | ((k >> 1) & 4)) << 1;
  if (ROWS == 96) return ((k >> 3) & 1) << 1;
  return (((k >> 1) & 1) | ((k >> 2) & 2)) << 1;  // 64
}

template <int ROWS, bool KM, bool PAIRED, int NW, int BK> struct Loader {
  static constexpr int kPieces = BK / 8;  // 16-byte pieces of a row of k
  // loads of a wave, 64 pieces each; where the tile has fewer than the waves could fetch, the last waves fetch the first pieces
  // again (the same bytes to the same place)
  static constexpr int kAll = ROWS * kPieces / 64, kPer = (kAll + NW - 1) / NW;
  static_assert(kAll * 64 == ROWS * kPieces, "a tile is a whole number of loads");
  unsigned off[kPer];
  int at[kPer];  // KM false: k of the piece

  static __device__ __forceinline__ int load_of(int wave, int q) {
    const int n = wave * kPer + q;
    return n < kAll ? n : n - kAll;
  }
  __device__ __forceinline__ void init(int ld, int rows, int wave, int lane) {
#pragma unroll
    for (int q = 0; q < kPer; ++q) {
      const int slot = load_of(wave, q) * 64 + lane;
      if (!KM) {
        const int row = slot / kPieces, chunk = (slot % kPieces) ^ swz_kc<PAIRED, BK>(row);
        at[q] = chunk * 8;
        off[q] = (unsigned)(row * ld + chunk * 8) * 2u;
      } else {
        constexpr int kc = ROWS / 8;
        const int k = slot / kc, chunk = (slot % kc) ^ swz_km<ROWS>(k);
        at[q] = 0;
        off[q] = chunk * 8 < rows ? (unsigned)(k * ld + chunk * 8) * 2u : 0x80000000u;
      }
    }
  }
  // base: the tile's first row (KM false) or first k; rows / kleft: what is left of the tensor from there (multiples of 8
  // along the contiguous axis)
  __device__ __forceinline__ void issue(const u16 *base, int ld, int rows, int kleft, char *lds, int wave) const {
    const int outer = KM ? (kleft < BK ? kleft : BK) : (rows < ROWS ? rows : ROWS), inner = KM ? rows : kleft;
    const unsigned bytes = (unsigned)((outer - 1) * ld + inner) * 2u;
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void *)base, 0, bytes, 0x00020000);
#pragma unroll
    for (int q = 0; q < kPer; ++q) {
      unsigned o = off[q];
      if (!KM && kleft < BK) o = at[q] < kleft ? o : 0x80000000u;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, CL3D_LDS(void, lds + load_of(wave, q) * 1024), 16, o, 0, 0, 0);
    }
  }
};

// fragment of 16 rows for k = 32 kk .. 32 kk + 31: lane l holds row l & 15, k = 8 (l >> 4) .. + 7.
// r0: first row of the 16 (PAIRED: of the 32; t says which half of every eight)
template <bool PAIRED, int BK> __device__ __forceinline__ s16x8 frag_kc(const char *lds, int r0, int t, int kk, int lane) {
  const int m = lane & 15, row = r0 + (PAIRED ? 8 * (m >> 2) + 4 * t + (m & 3) : m);
  return *reinterpret_cast<const s16x8 *>(lds + row * (BK * 2) + (((kk * 4 + (lane >> 4)) ^ swz_kc<PAIRED, BK>(row)) << 4));
}
template <int ROWS, bool PAIRED> __device__ __forceinline__ s16x8 frag_km(const char *lds, int r0, int t, int kk, int lane) {
  const int i = lane & 15, piece = i & 3;
  const int chunk = (r0 >> 3) + (PAIRED ? piece : piece >> 1), half = PAIRED ? t : piece & 1;
  s16x8 r;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int k = kk * 32 + 8 * (lane >> 4) + 4 * u + (i >> 2);
    const char *p = lds + k * (ROWS * 2) + ((chunk ^ swz_km<ROWS>(k)) << 4) + half * 8;
    const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16(CL3D_LDS(s16x4, p));
#pragma unroll
    for (int e = 0; e < 4; ++e) r[4 * u + e] = v[e];
  }
  return r;
}

// one operand pair of a product; P, Q at the first row of the tile
struct Pair {
  const u16 *P, *P2, *Q;  // P2: second matrix of the gated product (same shape as P)
  long long plane_p, plane_q;
  int ldp, ldq, rows_p, rows_q;
  int K, kp;  // k of the product (a multiple of 8 unless both operands are row-contiguous); rows a row-contiguous P really has
};

// bit 15 of either half: a bf16 whose exponent is all ones
__device__ __forceinline__ unsigned not_finite(unsigned two) { return (two & 0x7f807f80u) + 0x00800080u; }
// ... and 0 in its place
__device__ __forceinline__ s16x8 finite_or_0(s16x8 v) {
  union { s16x8 s; unsigned u[4]; } f{v};
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    const unsigned t = (not_finite(f.u[d]) & 0x80008000u) >> 15;
    f.u[d] &= ~(t * 0xffffu);
  }
  return f.s;
}

// acc[a][b] += the product over the tiles of k [s0, s1).  PR: rows of P in a tile (TWO: the first half from P, the second from P2).
// The wave (wi, wj) owns TI / 16 x TJ / 16 accumulators; TWO: first TI / 32 of P, then as many of P2, same rows.
template <typename E, int NP, int BK, int PR, bool PKM, bool PAIRED, bool TWO, int QR, bool QKM, int TI, int TJ, int NW>
__device__ __forceinline__ void product(f32x4 (&acc)[TI / 16][TJ / 16], const Pair &a, int s0, int s1, char *smem, int wave, int lane,
                                        int wi, int wj) {
  constexpr int kPBytes = PR * BK * 2, kQBytes = QR * BK * 2, kTile = NP * (kPBytes + kQBytes);
  constexpr int kPR = TWO ? PR / 2 : PR;
  Loader<PR, PKM, PAIRED, NW, BK> lp;
  Loader<QR, QKM, false, NW, BK> lq;
  static_assert(!(TWO && PKM), "two matrices: k contiguous");
  // TWO: this wave's pieces are all of one matrix (kPR rows are a whole number of waves' shares)
  const bool second = TWO && lp.load_of(wave, 0) * 64 / lp.kPieces >= kPR;
  static_assert(!TWO || kPR * lp.kPieces / 64 % lp.kPer == 0, "a wave loads of one matrix");
  lp.init(a.ldp, a.rows_p, wave, lane);
  lq.init(a.ldq, a.rows_q, wave, lane);
  const u16 *Pb = a.P;
  if (TWO && second) Pb = a.P2 - (long long)kPR * a.ldp;
  // rows behind the tile's end: beyond the descriptor (TWO: its rows are counted from the tile's first row)
  const int rows_p = TWO ? (second ? a.rows_p + kPR : (a.rows_p < kPR ? a.rows_p : kPR)) : a.rows_p;

  auto issue = [&](int s, int place) {
    const int k0 = s * BK;
    char *lds = smem + place * kTile;
    const u16 *P = Pb + (PKM ? (long long)k0 * a.ldp : k0), *Q = a.Q + (QKM ? (long long)k0 * a.ldq : k0);
#pragma unroll
    for (int n = 0; n < NP; ++n) {
      lp.issue(P + n * a.plane_p, a.ldp, rows_p, (PKM ? a.kp : a.K) - k0, lds + n * kPBytes, wave);
      lq.issue(Q + n * a.plane_q, a.ldq, a.rows_q, a.K - k0, lds + NP * kPBytes + n * kQBytes, wave);
    }
  };
  if (s0 >= s1) return;
  issue(s0, 0);
  int place = 0;
  for (int s = s0; s < s1; ++s) {
    // this step's tile has arrived; behind the barrier it has for every wave, and every wave has read the tile of the step
    // before, whose place the next load takes
    wait_vm<0>();
    barrier_lds();
    if (s + 1 < s1) issue(s + 1, place ^ 1);
    const char *lds = smem + place * kTile;
    place ^= 1;
#pragma unroll
    for (int kk = 0; kk < BK / 32; ++kk) {
      if (s * BK + kk * 32 >= a.K) break;
      s16x8 p[NP][TI / 16], q[NP][TJ / 16];
#pragma unroll
      for (int n = 0; n < NP; ++n) {
#pragma unroll
        for (int u = 0; u < TI / 16; ++u) {
          const int half = TWO ? u / (TI / 32) : 0, v = TWO ? u % (TI / 32) : u;
          const int r0 = half * kPR + wi * (TWO ? TI / 2 : TI) + (PAIRED ? (v >> 1) * 32 : v * 16);
          const char *at = lds + n * kPBytes;
          if constexpr (PKM) p[n][u] = frag_km<PR, PAIRED>(at, r0, v & 1, kk, lane);
          else p[n][u] = frag_kc<PAIRED, BK>(at, r0, v & 1, kk, lane);
        }
#pragma unroll
        for (int u = 0; u < TJ / 16; ++u) {
          const char *at = lds + NP * kPBytes + n * kQBytes;
          if constexpr (QKM) q[n][u] = frag_km<QR, false>(at, wj * TJ + u * 16, 0, kk, lane);
          else q[n][u] = frag_kc<false, BK>(at, wj * TJ + u * 16, 0, kk, lane);
        }
      }
      if constexpr (NP == 1) {
#pragma unroll
        for (int u = 0; u < TI / 16; ++u)
#pragma unroll
          for (int v = 0; v < TJ / 16; ++v) acc[u][v] = mfma16<E>(p[0][u], q[0][v], acc[u][v]);
      } else {
        auto all = [&](const s16x8 (&x)[TI / 16], const s16x8 (&y)[TJ / 16]) {
#pragma unroll
          for (int u = 0; u < TI / 16; ++u)
#pragma unroll
            for (int v = 0; v < TJ / 16; ++v) acc[u][v] = mfma16<E>(x[u], y[v], acc[u][v]);
        };
        unsigned odd = 0;
#pragma unroll
        for (int u = 0; u < TI / 16; ++u) {
          union { s16x8 s; unsigned d[4]; } f{p[0][u]};
#pragma unroll
          for (int d = 0; d < 4; ++d) odd |= not_finite(f.d[d]);
        }
#pragma unroll
        for (int u = 0; u < TJ / 16; ++u) {
          union { s16x8 s; unsigned d[4]; } f{q[0][u]};
#pragma unroll
          for (int d = 0; d < 4; ++d) odd |= not_finite(f.d[d]);
        }
        if (__builtin_expect(__any((odd & 0x80008000u) != 0u), 0)) {
          s16x8 pf[TI / 16], qf[TJ / 16];
#pragma unroll
          for (int u = 0; u < TI / 16; ++u) pf[u] = finite_or_0(p[0][u]);
#pragma unroll
          for (int u = 0; u < TJ / 16; ++u) qf[u] = finite_or_0(q[0][u]);
          all(p[2], qf);  // (in the order of the other branch: what is finite keeps its bits beside an infinity)
          all(pf, q[2]);
          all(p[1], q[1]);
          all(p[1], qf);
          all(pf, q[1]);
          all(p[0], q[0]);
        } else {
          all(p[2], q[0]);
          all(p[0], q[2]);
          all(p[1], q[1]);
          all(p[1], q[0]);
          all(p[0], q[1]);
          all(p[0], q[0]);
        }
      }
    }
  }
  barrier_lds();  // (another product may follow in the same tiles)
}

// ---- activations (CL3D_ACT_SILU / _GELU / _RELU): value and slope at g.  exp2 and the reciprocal are the hardware's (one step
// each).  The error function by its complement, erfc(z) = exp(-z^2) t Q(t) with t = 1 / (1 + 0.45 z), so that the tails keep their
// digits; Q, of degree nine, is fitted to exp(z^2) erfc(z) / t over all z >= 0 for the smallest relative error: 3e-8, 3.3e-7 as
// evaluated in f32.  That is below what the f32 sum in g carries.
__device__ __forceinline__ void activate(int act, float g, float &value, float &slope) {
  if (act == CL3D_ACT_SILU) {
    const float s = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * g));
    value = g * s;
    slope = s * __builtin_fmaf(g, 1.f - s, 1.f);
  } else if (act == CL3D_ACT_GELU) {
    const float z = 0.70710678118654752f * fabsf(g), t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.45f, z, 1.f));
    float q = -0.0414836183f;
    q = __builtin_fmaf(q, t, 0.191090241f);
    q = __builtin_fmaf(q, t, -0.301313758f);
    q = __builtin_fmaf(q, t, 0.143121704f);
    q = __builtin_fmaf(q, t, -0.022776071f);
    q = __builtin_fmaf(q, t, 0.120095469f);
    q = __builtin_fmaf(q, t, 0.175222933f);
    q = __builtin_fmaf(q, t, 0.228274778f);
    q = __builtin_fmaf(q, t, 0.253883004f);
    q = __builtin_fmaf(q, t, 0.253885329f);
    const float e = __builtin_amdgcn_exp2f(-1.4426950408889634f * z * z), tail = 0.5f * q * t * e;
    const float c = g < 0.f ? tail : 1.f - tail;
    value = g * c;
    slope = __builtin_fmaf(g, 0.3989422804014327f * e, c);
  } else {  // relu; a NaN stays one, the slope at 0 is 0
    value = g < 0.f ? 0.f : g;
    slope = g > 0.f ? 1.f : (g <= 0.f ? 0.f : g);
  }
}

// an f32 value as the exact sum of three bf16 values, each rounded to nearest (8, 8 and the last 8 of 24 bits; truncated, the products
// left out would be up to 2^-21 of |x||y| and all of its sign).  Where rounding would make an infinity of a finite value the leading
// one is truncated; what is not finite is the leading one alone.
struct Split {
  u16 p[3];
};
__device__ __forceinline__ Split split3(float x) {
  const unsigned b = __float_as_uint(x);
  Split s;
  if ((b & 0x7f800000u) == 0x7f800000u) {
    s.p[0] = (u16)(b >> 16);
    if (b & 0x007fffffu) s.p[0] |= 0x40;  // a NaN whose payload sits in the low half stays a NaN
    s.p[1] = s.p[2] = 0;
    return s;
  }
  s.p[0] = Bf16::put(x);
  if ((s.p[0] & 0x7f80u) == 0x7f80u) s.p[0] = (u16)(b >> 16);
  const float r = x - Bf16::get(s.p[0]);
  s.p[1] = Bf16::put(r);
  s.p[2] = Bf16::put(r - Bf16::get(s.p[1]));
  return s;
}

struct GemmArgs {
  const u16 *P, *P2, *Q;     // first product
  const u16 *Pb, *Qb;        // GATED_BWD: dh = Wd, dY; NN: the second pair of dX
  long long plane_p, plane_q, plane_pb, plane_qb;
  int ldp, ldq, ldpb, ldqb;
  int I, J, K, Kb, kp;       // K, Kb multiples of 8 (zero-padded operands); kp: rows of the P whose rows run along i
  int act;
  void *D;                   // result rows of ldd elements of the tensor type
  int ldd, vec;              // vec: rows start 16-byte aligned
  u16 *h, *dgu;              // operand-type intermediates, ldh and 2 ldh a row, zero up to ldh; 3 planes when split
  long long plane_h, plane_dgu;
  int ldh, planes;
  const void *dh;            // GATED_BWD without a down projection: dh itself, rows of lddh
  int lddh;
};

// four or eight consecutive elements of an internal row: operand type, or the three planes
template <typename E, int N> __device__ __forceinline__ void put_internal(u16 *row, long long plane, int planes, const float *v) {
  if (planes == 1) {
    u16 o[N];
#pragma unroll
    for (int e = 0; e < N; ++e) o[e] = E::put(v[e]);
    if constexpr (N == 8) *reinterpret_cast<s16x8 *>(row) = *reinterpret_cast<s16x8 *>(o);
    else *reinterpret_cast<s16x4 *>(row) = *reinterpret_cast<s16x4 *>(o);
    return;
  }
  u16 o[3][N];
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const Split s = split3(v[e]);
#pragma unroll
    for (int p = 0; p < 3; ++p) o[p][e] = s.p[p];
  }
#pragma unroll
  for (int p = 0; p < 3; ++p) {
    if constexpr (N == 8) *reinterpret_cast<s16x8 *>(row + p * plane) = *reinterpret_cast<s16x8 *>(o[p]);
    else *reinterpret_cast<s16x4 *>(row + p * plane) = *reinterpret_cast<s16x4 *>(o[p]);
  }
}
// N consecutive elements of a row of the caller's tensor, `left` of them inside it
template <typename T, int N> __device__ __forceinline__ void put_row(typename T::storage *row, int left, bool vec, const float *v) {
  if (vec && left >= N) {
    typename T::storage o[N];
#pragma unroll
    for (int e = 0; e < N; ++e) o[e] = T::put(v[e]);
    if constexpr (sizeof(o) >= 16) {
#pragma unroll
      for (int q = 0; q < (int)sizeof(o) / 16; ++q) reinterpret_cast<s16x8 *>(row)[q] = reinterpret_cast<s16x8 *>(o)[q];
    } else {
      *reinterpret_cast<s16x4 *>(row) = *reinterpret_cast<s16x4 *>(o);
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < N; ++e)
    if (e < left) row[e] = T::put(v[e]);
}

enum { GEMM_NT = 0, GEMM_NN = 1, GEMM_GATED = 2, GEMM_GATED_BWD = 3 };

// linear workgroup number -> tile: the hardware deals workgroups to the 8 XCDs in turn; each XCD gets a run of neighbours
__device__ __forceinline__ int xcd_order(int id, int total) {
  const int x = id & 7, q = id >> 3, per = total >> 3, rem = total & 7;
  return x * per + (x < rem ? x : rem) + q;
}

// E: operand type; T: type of the caller's tensors.  A workgroup of WI x WJ waves owns BI x BJ results (GATED*: BI is twice the
// channels).
template <int KIND, typename E, typename T, int NP, int BI, int BJ, int WI, int WJ, int BK>
__global__ __launch_bounds__(64 * WI * WJ) void ffn_gemm_kernel(GemmArgs a) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  constexpr int NW = WI * WJ, TI = BI / WI, TJ = BJ / WJ;
  constexpr bool kTwo = KIND == GEMM_GATED || KIND == GEMM_GATED_BWD;
  constexpr int kCh = kTwo ? BI / 2 : BI;  // result columns of the workgroup
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wi = wave / WJ, wj = wave % WJ;
  const int ti = (a.I + kCh - 1) / kCh;
  const int id = xcd_order(blockIdx.x, gridDim.x), row = __builtin_amdgcn_readfirstlane(id / ti);
  const int i0 = (id - row * ti) * kCh, j0 = row * BJ;
  const int ip = (a.I + 7) & ~7, g = lane >> 4;

  f32x4 acc[TI / 16][TJ / 16];
#pragma unroll
  for (int u = 0; u < TI / 16; ++u)
#pragma unroll
    for (int v = 0; v < TJ / 16; ++v) acc[u][v] = (f32x4){0.f, 0.f, 0.f, 0.f};

  if constexpr (KIND == GEMM_GATED || KIND == GEMM_GATED_BWD) {
    Pair pr{a.P + (long long)i0 * a.ldp, a.P2 + (long long)i0 * a.ldp, a.Q + (long long)j0 * a.ldq, a.plane_p, a.plane_q,
            a.ldp, a.ldq, a.I - i0, a.J - j0, a.K, a.K};
    const int steps = (a.K + BK - 1) / BK;
    product<E, NP, BK, BI, false, true, true, BJ, false, TI, TJ, NW>(acc, pr, 0, steps, smem, wave, lane, wi, wj);
    f32x4 dh[TI / 32][TJ / 16];
    if constexpr (KIND == GEMM_GATED_BWD) {
#pragma unroll
      for (int u = 0; u < TI / 32; ++u)
#pragma unroll
        for (int v = 0; v < TJ / 16; ++v) dh[u][v] = (f32x4){0.f, 0.f, 0.f, 0.f};
      if (a.Qb != nullptr) {
        Pair pb{a.Pb + i0, nullptr, a.Qb + (long long)j0 * a.ldqb, a.plane_pb, a.plane_qb, a.ldpb, a.ldqb, ip - i0, a.J - j0, a.Kb,
                a.kp};
        const int sb = (a.Kb + BK - 1) / BK;
        product<E, NP, BK, BI / 2, true, true, false, BJ, false, TI / 2, TJ, NW>(dh, pb, 0, sb, smem, wave, lane, wi, wj);
      }
    }
#pragma unroll
    for (int b = 0; b < TI / 64; ++b) {
      const int c0 = i0 + wi * (TI / 2) + b * 32 + 8 * g;  // this lane's eight channels
      if (c0 >= ip) continue;
#pragma unroll
      for (int v = 0; v < TJ / 16; ++v) {
        const int j = j0 + wj * TJ + v * 16 + (lane & 15);
        if (j >= a.J) continue;
        float h[8], dg[8] = {}, du[8] = {};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float gv = acc[2 * b + (e >> 2)][v][e & 3], uv = acc[TI / 32 + 2 * b + (e >> 2)][v][e & 3];
          float val, slope;
          activate(a.act, gv, val, slope);
          h[e] = val * uv;
          if constexpr (KIND == GEMM_GATED_BWD) {
            float d = dh[2 * b + (e >> 2)][v][e & 3];
            if (a.Qb == nullptr)
              d = c0 + e < a.I ? T::get(static_cast<const typename T::storage *>(a.dh)[(long long)j * a.lddh + c0 + e]) : 0.f;
            dg[e] = d * uv * slope;
            du[e] = d * val;
          }
          if (c0 + e >= a.I) h[e] = dg[e] = du[e] = 0.f;  // the padding of an internal row is zero, whatever 0 x inf makes
        }
        if (KIND == GEMM_GATED && a.D != nullptr) {
          put_row<T, 8>(static_cast<typename T::storage *>(a.D) + (long long)j * a.ldd + c0, a.I - c0, a.vec, h);
          continue;
        }
        if (a.h != nullptr) put_internal<E, 8>(a.h + (long long)j * a.ldh + c0, a.plane_h, a.planes, h);
        if constexpr (KIND == GEMM_GATED_BWD) {
          u16 *row = a.dgu + (long long)j * 2 * a.ldh + c0;
          put_internal<E, 8>(row, a.plane_dgu, a.planes, dg);
          put_internal<E, 8>(row + a.ldh, a.plane_dgu, a.planes, du);
        }
      }
    }
  } else if constexpr (KIND == GEMM_NT || KIND == GEMM_NN) {
    constexpr bool kKm = KIND == GEMM_NN;  // NN: P's rows are contiguous in i
    constexpr bool kPair = !kKm && TI % 32 == 0;  // eight consecutive results a lane instead of four
    Pair pr{kKm ? a.P + i0 : a.P + (long long)i0 * a.ldp, nullptr, a.Q + (long long)j0 * a.ldq, a.plane_p, a.plane_q, a.ldp, a.ldq,
            kKm ? ip - i0 : a.I - i0, a.J - j0, a.K, a.kp};
    const int steps = (a.K + BK - 1) / BK;
    product<E, NP, BK, BI, kKm, kPair, false, BJ, false, TI, TJ, NW>(acc, pr, 0, steps, smem, wave, lane, wi, wj);
    if (kKm && a.Pb != nullptr) {  // dX = dG Wg + dU Wu
      pr.P = a.Pb + i0;
      pr.Q = a.Qb + (long long)j0 * a.ldq;
      product<E, NP, BK, BI, kKm, kPair, false, BJ, false, TI, TJ, NW>(acc, pr, 0, steps, smem, wave, lane, wi, wj);
    }
    auto *D = static_cast<typename T::storage *>(a.D);
#pragma unroll
    for (int v = 0; v < TJ / 16; ++v) {
      const int j = j0 + wj * TJ + v * 16 + (lane & 15);
      if (j >= a.J) continue;
      if constexpr (kPair) {
#pragma unroll
        for (int b = 0; b < TI / 32; ++b) {
          const int c0 = i0 + wi * TI + b * 32 + 8 * g;
          float o[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) o[e] = acc[2 * b + (e >> 2)][v][e & 3];
          if (c0 < a.I) put_row<T, 8>(D + (long long)j * a.ldd + c0, a.I - c0, a.vec, o);
        }
      } else {
#pragma unroll
        for (int u = 0; u < TI / 16; ++u) {
          const int c0 = i0 + wi * TI + u * 16 + 4 * g;
          float o[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] = acc[u][v][e];
          if (c0 < a.I) put_row<T, 4>(D + (long long)j * a.ldd + c0, a.I - c0, a.vec, o);
        }
      }
    }
  }
}

// The weight gradients of a call, up to three products D[j][i] = sum over the points of P(i, r) Q(j, r), both operands' rows running
// along i and j; a workgroup owns a tile of one of them for a slice of the points: f32 partials [product][slice][J][I].
struct WeightArgs {
  const u16 *P[3], *Q[3];
  float *D[3];
  long long plane_p[3], plane_q[3];
  int I[3], J[3], ldp[3], ldq[3], vec[3];
  int products, K, slices;
};
template <typename E, int NP, int BI, int BJ, int WI, int WJ, int BK>
__global__ __launch_bounds__(64 * WI * WJ) void ffn_weight_kernel(WeightArgs a) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  constexpr int NW = WI * WJ, TI = BI / WI, TJ = BJ / WJ;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wi = wave / WJ, wj = wave % WJ, g = lane >> 4;
  const int per_slice = gridDim.x / a.slices;
  int id = xcd_order(blockIdx.x, gridDim.x);
  const int slice = __builtin_amdgcn_readfirstlane(id / per_slice);
  id -= slice * per_slice;
  int w = 0, ti = (a.I[0] + BI - 1) / BI;
  for (int t = ti * ((a.J[0] + BJ - 1) / BJ); w + 1 < a.products && id >= t; t = ti * ((a.J[w] + BJ - 1) / BJ)) {
    id -= t;
    ++w;
    ti = (a.I[w] + BI - 1) / BI;
  }
  const int row = __builtin_amdgcn_readfirstlane(id / ti), i0 = (id - row * ti) * BI, j0 = row * BJ, I = a.I[w], J = a.J[w];
  f32x4 acc[TI / 16][TJ / 16];
#pragma unroll
  for (int u = 0; u < TI / 16; ++u)
#pragma unroll
    for (int v = 0; v < TJ / 16; ++v) acc[u][v] = (f32x4){0.f, 0.f, 0.f, 0.f};
  Pair pr{a.P[w] + i0, nullptr, a.Q[w] + j0, a.plane_p[w], a.plane_q[w], a.ldp[w], a.ldq[w], ((I + 7) & ~7) - i0, ((J + 7) & ~7) - j0, a.K, a.K};
  const long long steps = (a.K + BK - 1) / BK;
  const int s0 = __builtin_amdgcn_readfirstlane((int)(steps * slice / a.slices));
  const int s1 = __builtin_amdgcn_readfirstlane((int)(steps * (slice + 1) / a.slices));
  product<E, NP, BK, BI, true, false, false, BJ, true, TI, TJ, NW>(acc, pr, s0, s1, smem, wave, lane, wi, wj);
  float *D = a.D[w] + (long long)slice * J * I;
#pragma unroll
  for (int v = 0; v < TJ / 16; ++v) {
    const int j = j0 + wj * TJ + v * 16 + (lane & 15);
    if (j >= J) continue;
#pragma unroll
    for (int u = 0; u < TI / 16; ++u) {
      const int c0 = i0 + wi * TI + u * 16 + 4 * g;
      float o[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = acc[u][v][e];
      if (c0 < I) put_row<F32, 4>(D + (long long)j * I + c0, I - c0, a.vec[w], o);
    }
  }
}

// dst[e] = sum over slices of src[slice][e], in slice order, for up to three weight gradients (blockIdx.y); V elements a lane
struct SliceSums {
  const float *src[3];
  void *dst[3];
  long long n[3];
  int slices[3];
};
template <typename T, int V> __global__ __launch_bounds__(256) void ffn_slices_kernel(SliceSums a) {
  const int w = blockIdx.y, slices = a.slices[w];
  const long long n = a.n[w], stride = (long long)gridDim.x * 256 * V;
  const float *src = a.src[w];
  auto *dst = static_cast<typename T::storage *>(a.dst[w]);
  if (dst == nullptr) return;
  for (long long e = ((long long)blockIdx.x * 256 + threadIdx.x) * V; e < n; e += stride) {
    float s[V];
#pragma unroll
    for (int v = 0; v < V; ++v) s[v] = 0.f;
#pragma unroll 4
    for (int z = 0; z < slices; ++z) {
      if constexpr (V == 4) {
        const f32x4 t = *reinterpret_cast<const f32x4 *>(src + (long long)z * n + e);
#pragma unroll
        for (int v = 0; v < 4; ++v) s[v] += t[v];
      } else {
        s[0] += src[(long long)z * n + e];
      }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) dst[e + v] = T::put(s[v]);
  }
}

// ---- operands that are not what the products read: another memory order, odd rows, f32 ---------------------------------
// source element (b, r, c) at src + b sb + r sr + c sc, one of sr, sc being 1; out rows [(b, r)] of ld elements, zero behind C.
// `planes` 3: the split of an f32 value; 1: one rounding to E (none when S is E).  All operands of a call in one launch: most are
// weights, and a launch costs more than their copy.
struct PackJob {
  const void *src;
  u16 *dst;
  long long sb, sr, sc, plane;
  int Rb, C, ld, tiles_c, tiles;  // tiles of 32 rows x 64 columns: of a batch's columns, of a batch
  int first;                      // workgroup at which this job begins
};
constexpr int kPackJobs = 5;
struct PackArgs {
  PackJob job[kPackJobs];
  int jobs, planes;
};
template <typename S, typename E> __global__ __launch_bounds__(256) void ffn_pack_kernel(PackArgs a) {
  __shared__ float tile[32][65];
  int which = 0;
  while (which + 1 < a.jobs && (int)blockIdx.x >= a.job[which + 1].first) ++which;
  const PackJob &j = a.job[which];
  int id = blockIdx.x - j.first;
  const int b = id / j.tiles;
  id -= b * j.tiles;
  const int r0 = id / j.tiles_c * 32, c0 = id % j.tiles_c * 64, tid = threadIdx.x;
  const auto *s = static_cast<const typename S::storage *>(j.src) + (long long)b * j.sb;
  float in[8];
#pragma unroll
  for (int q = 0; q < 8; ++q) {  // (all eight on their way before the first is put down)
    const int e = q * 256 + tid, r = j.sc == 1 ? e >> 6 : e & 31, c = j.sc == 1 ? e & 63 : e >> 5;
    in[q] = r0 + r < j.Rb && c0 + c < j.C ? S::get(s[(r0 + r) * j.sr + (c0 + c) * j.sc]) : 0.f;
  }
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    const int e = q * 256 + tid;
    tile[j.sc == 1 ? e >> 6 : e & 31][j.sc == 1 ? e & 63 : e >> 5] = in[q];
  }
  __syncthreads();
  const int r = tid >> 3, c = (tid & 7) * 8;  // 32 rows x 8 pieces of 8
  if (r0 + r >= j.Rb || c0 + c >= j.ld) return;
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = tile[r][c + e];
  put_internal<E, 8>(j.dst + ((long long)b * j.Rb + r0 + r) * j.ld + c0 + c, j.plane, a.planes, v);
}

// ---- few points: the weights are read once, straight into fragments -------------------------------------------------------
// A workgroup of eight waves owns 16 results i (GATED: of both projections) for up to JT x 16 points; its waves take pieces of k in
// turn and their accumulators are joined in LDS, in wave order.  No operand passes through LDS (each weight is used by one wave
// only), U pieces of every matrix are in flight per wave, the tensors are read as they are: no packed copies, f32 by the f32 MFMA.
// Bound: the read of the weights.  VEC: rows start on 16 bytes (K a multiple of a piece); else element by element.
template <typename T, bool VEC> struct Piece {
  typename T::storage v[T::kVec];
  __device__ __forceinline__ void load(const typename T::storage *row, int k, int K) {
    if (VEC) {
      if (k < K) *reinterpret_cast<Vec16<T> *>(v) = *reinterpret_cast<const Vec16<T> *>(row + k);
      else *reinterpret_cast<Vec16<T> *>(v) = Vec16<T>{};
    } else {
#pragma unroll
      for (int e = 0; e < T::kVec; ++e) v[e] = k + e < K ? row[k + e] : typename T::storage(0);
    }
  }
} __attribute__((aligned(16)));
template <typename T, bool VEC> __device__ __forceinline__ f32x4 mul_piece(const Piece<T, VEC> &p, const Piece<T, VEC> &q, f32x4 c) {
  if constexpr (std::is_same<T, F32>::value) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(p.v[e], q.v[e], c, 0, 0, 0);
    return c;
  } else {
    return mfma16<T>(*reinterpret_cast<const s16x8 *>(p.v), *reinterpret_cast<const s16x8 *>(q.v), c);
  }
}

struct RowsArgs {
  const void *P, *P2, *Q;
  void *D;
  int I, J, K, ldp, ldq, ldd, act, vec_out;
};

constexpr int kRowsWaves = 8, kRowsMost = CL3D_FFN_FEW;  // points of a call that goes this way, at most

template <bool GATED, typename T, int JT, bool VEC>
__global__ __launch_bounds__(64 * kRowsWaves) void ffn_rows_kernel(RowsArgs a) {
  using S = typename T::storage;
  constexpr int M = GATED ? 2 : 1, U = JT == 4 ? 2 : 4, V = T::kVec;
  __shared__ f32x4 s_acc[kRowsWaves][M][JT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4;
  const int i0 = blockIdx.x * 16;
  const long long i = i0 + (lane & 15) < a.I ? i0 + (lane & 15) : a.I - 1;  // (a row behind the end: read, not stored)
  const S *P = static_cast<const S *>(a.P) + i * a.ldp, *P2 = GATED ? static_cast<const S *>(a.P2) + i * a.ldp : nullptr;
  const S *Q[JT];
  f32x4 acc[M][JT];
#pragma unroll
  for (int t = 0; t < JT; ++t) {
    const int j = t * 16 + (lane & 15);
    Q[t] = static_cast<const S *>(a.Q) + (long long)(j < a.J ? j : a.J - 1) * a.ldq;
#pragma unroll
    for (int m = 0; m < M; ++m) acc[m][t] = (f32x4){0.f, 0.f, 0.f, 0.f};
  }
  // two sets of pieces: one on its way while the other is multiplied
  Piece<T, VEC> p[2][U], p2[2][GATED ? U : 1], q[2][JT][U];
  constexpr int kTurn = kRowsWaves * U * 4 * V;
  auto fetch = [&](int set, int k0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + (u * 4 + g) * V;
      p[set][u].load(P, k, a.K);
      if (GATED) p2[set][u].load(P2, k, a.K);
#pragma unroll
      for (int t = 0; t < JT; ++t) q[set][t][u].load(Q[t], k, a.K);
    }
  };
  auto multiply = [&](int set) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int t = 0; t < JT; ++t) {
        acc[0][t] = mul_piece<T, VEC>(p[set][u], q[set][t][u], acc[0][t]);
        if (GATED) acc[M - 1][t] = mul_piece<T, VEC>(p2[set][u], q[set][t][u], acc[M - 1][t]);
      }
  };
  const int k0 = wave * U * 4 * V;
  if (k0 < a.K) fetch(0, k0);
  for (int k = k0; k < a.K; k += 2 * kTurn) {
    if (k + kTurn < a.K) fetch(1, k + kTurn);
    multiply(0);
    if (k + 2 * kTurn < a.K) fetch(0, k + 2 * kTurn);
    if (k + kTurn < a.K) multiply(1);
  }
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int t = 0; t < JT; ++t) s_acc[wave][m][t][lane] = acc[m][t];
  __syncthreads();
  if (threadIdx.x >= JT * 64) return;
  const int t = threadIdx.x >> 6;  // (a wave per 16 points)
  f32x4 sum[M];
#pragma unroll
  for (int m = 0; m < M; ++m) {
    sum[m] = s_acc[0][m][t][lane];
#pragma unroll
    for (int w = 1; w < kRowsWaves; ++w) sum[m] += s_acc[w][m][t][lane];
  }
  const int j = t * 16 + (lane & 15), c0 = i0 + 4 * g;
  if (j >= a.J || c0 >= a.I) return;
  float o[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    o[e] = sum[0][e];
    if (GATED) {
      float slope;
      activate(a.act, sum[0][e], o[e], slope);
      o[e] *= sum[M - 1][e];
    }
  }
  put_row<T, 4>(static_cast<S *>(a.D) + (long long)j * a.ldd + c0, a.I - c0, a.vec_out, o);
}

// ---- narrow points, many of them: the whole forward pass in one kernel -----------------------------------------------------------
// Up to 224 channels a wave keeps its 16 NJ points in registers -- their x as fragments, their y as accumulators -- and the workgroup
// walks the hidden channels, 32 at a time: G and U of a chunk, h = act(G) U, y += Wd h.  The accumulators of G and U are laid out so
// that a lane's eight values of h (channels 8 g .. 8 g + 7 of one point) are what the last product wants as its second operand, so h
// passes from one product to the next without leaving the lane.  Only the weights travel: a chunk's rows of Wg and Wu and columns
// of Wd, by way of LDS, the next chunk in flight; x is read and y written once, h is written only if the caller keeps it.
// CF: 32-channel fragments of x, odd (a row of 64 CF bytes then starts at a quarter of its own of the 64 banks).
// Measured against the two kernels it replaces (us, a launch by itself, bf16): 65 536 x 144 x 576 60 (83; 51 where passes follow each
// other), 131 072 x 72 x 288 41 (63), 32 768 x 144 x 576 39 (42), 65 536 x 200 x 800 91 (121); 16 384 x 144 x 576 37 (25): below 32 768 points there are fewer than 256 workgroups of
// 128, one for each CU.  Bound: per chunk a wave waits for its weights, reads each fragment for one or two products and then is in
// the activation; the two workgroups of a CU cover each other's waits in part.
constexpr int kFusedMostC = 224, kFusedFewest = 32768;
struct FusedArgs {
  const u16 *G, *U, *D, *X;  // G, U: rows of ldw, D: rows of ldd, X: rows of ldx
  void *Y;
  u16 *h;                    // nullable: rows of hp
  int J, C, H, hp, ldw, ldd, ldx, ldy, act, vec;
};
template <typename E, typename T, int CF, int NJ, int NW>
__global__ __launch_bounds__(64 * NW) void ffn_fused_kernel(FusedArgs a) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  constexpr int kPart = 2048 * CF, kTile = 3 * kPart;  // 32 rows of 64 CF bytes; 32 CF rows of 64 bytes
  constexpr int kAll = 6 * CF, kPer = (kAll + NW - 1) / NW;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, m = lane & 15, cp = (a.C + 7) & ~7;
  const int j0 = (xcd_order(blockIdx.x, gridDim.x) * NW + wave) * NJ * 16;

  unsigned off[kPer];
#pragma unroll
  for (int q = 0; q < kPer; ++q) {
    const int n0 = wave * kPer + q, n = n0 < kAll ? n0 : n0 - kAll, part = n / (2 * CF), slot = (n - part * 2 * CF) * 64 + lane;
    if (part < 2) {
      const int row = slot / (4 * CF), piece = slot - row * 4 * CF, chunk = (piece & ~3) | ((piece & 3) ^ ((row >> 3) & 3));
      off[q] = chunk * 8 < cp ? (unsigned)(row * a.ldw + chunk * 8) * 2u : 0x80000000u;
    } else {
      const int row = slot >> 2, chunk = (slot & 3) ^ ((row >> 3) & 3);
      off[q] = (unsigned)(row * a.ldd + chunk * 8) * 2u;
    }
  }
  auto issue = [&](int h0, int place) {
    const int rows = a.H - h0 < 32 ? a.H - h0 : 32, cols = a.hp - h0 < 32 ? a.hp - h0 : 32;
#pragma unroll
    for (int q = 0; q < kPer; ++q) {
      const int n0 = wave * kPer + q, n = n0 < kAll ? n0 : n0 - kAll, part = n / (2 * CF);
      const u16 *base = part == 0 ? a.G + (long long)h0 * a.ldw : part == 1 ? a.U + (long long)h0 * a.ldw : a.D + h0;
      const unsigned bytes = part < 2 ? (unsigned)((rows - 1) * a.ldw + cp) * 2u : (unsigned)((a.C - 1) * a.ldd + cols) * 2u;
      unsigned o = off[q];
      if (part == 2 && cols < 32) {  // the last columns of Wd: what follows them in memory is the next row
        const int slot = (n - 4 * CF) * 64 + lane, chunk = (slot & 3) ^ (((slot >> 2) >> 3) & 3);
        o = chunk * 8 < cols ? o : 0x80000000u;
      }
      const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void *)base, 0, bytes, 0x00020000);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, CL3D_LDS(void, smem + place * kTile + n * 1024), 16, o, 0, 0, 0);
    }
  };
  issue(0, 0);

  s16x8 x[CF][NJ];
#pragma unroll
  for (int t = 0; t < NJ; ++t) {
    const int j = j0 + t * 16 + m;
    const u16 *row = a.X + (long long)(j < a.J ? j : a.J - 1) * a.ldx;
#pragma unroll
    for (int kk = 0; kk < CF; ++kk) {
      const int k = kk * 32 + 8 * g;
      x[kk][t] = k < cp ? *reinterpret_cast<const s16x8 *>(row + k) : (s16x8){0, 0, 0, 0, 0, 0, 0, 0};
    }
  }
  f32x4 y[2 * CF][NJ];
#pragma unroll
  for (int u = 0; u < 2 * CF; ++u)
#pragma unroll
    for (int t = 0; t < NJ; ++t) y[u][t] = (f32x4){0.f, 0.f, 0.f, 0.f};

  f32x4 s[4][NJ];
  auto project = [&](const char *lds) {  // G and U of a chunk
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int t = 0; t < NJ; ++t) s[u][t] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kk = 0; kk < CF; ++kk) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {  // gate, gate, up, up
        const int row = 8 * (m >> 2) + 4 * (u & 1) + (m & 3);
        const s16x8 p = *reinterpret_cast<const s16x8 *>(lds + (u >> 1) * kPart + row * (64 * CF) + ((kk * 4 + (g ^ ((row >> 3) & 3))) << 4));
#pragma unroll
        for (int t = 0; t < NJ; ++t) s[u][t] = mfma16<E>(p, x[kk][t], s[u][t]);
      }
    }
  };
  auto finish = [&](const char *lds, int h0) {  // h of the chunk, and what it adds to y
    s16x8 h[NJ];
#pragma unroll
    for (int t = 0; t < NJ; ++t) {
      u16 o[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float v, slope;
        activate(a.act, s[e >> 2][t][e & 3], v, slope);
        o[e] = E::put(v * s[2 + (e >> 2)][t][e & 3]);
      }
      if (h0 + 32 > a.H) {  // behind the last channel: zero, whatever 0 x inf made
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (h0 + 8 * g + e >= a.H) o[e] = 0;
      }
      h[t] = *reinterpret_cast<s16x8 *>(o);
      const int j = j0 + t * 16 + m;
      if (a.h != nullptr && j < a.J && h0 + 8 * g < a.hp) *reinterpret_cast<s16x8 *>(a.h + (long long)j * a.hp + h0 + 8 * g) = h[t];
    }
#pragma unroll
    for (int u = 0; u < 2 * CF; ++u) {
      const int row = (u >> 1) * 32 + 8 * (m >> 2) + 4 * (u & 1) + (m & 3);
      const s16x8 p = *reinterpret_cast<const s16x8 *>(lds + 2 * kPart + row * 64 + ((g ^ ((row >> 3) & 3)) << 4));
#pragma unroll
      for (int t = 0; t < NJ; ++t) y[u][t] = mfma16<E>(p, h[t], y[u][t]);
    }
  };
  int place = 0;
  // a chunk's weights are older than the NJ stores of the chunk before, if every lane made them: those need not be waited for
  const bool all_store = a.h != nullptr && j0 + NJ * 16 <= a.J;
  for (int h0 = 0; h0 < a.hp; h0 += 32) {
    if (all_store && h0 > 0) wait_vm<NJ>();  // (the chunk before was a whole one)
    else wait_vm<0>();
    barrier_lds();
    if (h0 + 32 < a.hp) issue(h0 + 32, place ^ 1);
    const char *lds = smem + place * kTile;
    place ^= 1;
    project(lds);
    finish(lds, h0);
  }
  auto *Y = static_cast<typename T::storage *>(a.Y);
#pragma unroll
  for (int t = 0; t < NJ; ++t) {
    const int j = j0 + t * 16 + m;
    if (j >= a.J) continue;
#pragma unroll
    for (int b = 0; b < CF; ++b) {
      const int c0 = b * 32 + 8 * g;
      if (c0 >= a.C) continue;
      float o[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = y[2 * b + (e >> 2)][t][e & 3];
      put_row<T, 8>(Y + (long long)j * a.ldy + c0, a.C - c0, a.vec, o);
    }
  }
}

// ---- host side -----------------------------------------------------------------------------------------------------
struct Operand {
  const u16 *p = nullptr;
  int ld = 0;
  long long plane = 0;
};

struct FfnShape {
  int dtype, order, B, N, C, H, act, split;  // split: f32 tensors at f32 precision
  bool down;
  long long R() const { return (long long)B * N; }
  bool channel() const { return order == CL3D_CHANNEL_MAJOR && N > 1 && C > 0; }
  bool convert() const { return dtype == CL3D_F32; }
};

// the operands of one call: the caller's own memory where the products can read it, else a packed copy in the launch to come
struct Operands {
  const FfnShape &s;
  Arena &ar;
  PackArgs a{};
  long long groups = 0;
  Operands(const FfnShape &s_, Arena &ar_) : s(s_), ar(ar_) { a.planes = s.split ? 3 : 1; }

  // rows [(b, r)][C]
  Operand take(const void *src, bool channel, int B, int Rb, int C) {
    const int ld = (C + 7) & ~7;
    if (!s.convert() && !channel && C % 8 == 0) return {static_cast<const u16 *>(src), C, 0};
    const long long plane = (long long)B * Rb * ld;
    u16 *dst = static_cast<u16 *>(ar.take((size_t)plane * a.planes * 2));
    // (rows that follow each other without regard to the cloud are one batch)
    const int b = channel ? B : 1, rb = channel ? Rb : B * Rb, tiles_c = ceil_div(ld, 64), tiles = tiles_c * ceil_div(rb, 32);
    a.job[a.jobs++] = {src, dst, (long long)C * Rb, channel ? 1 : C, channel ? Rb : 1, plane, rb, C, ld, tiles_c, tiles, (int)groups};
    groups += (long long)tiles * b;
    return {dst, ld, plane};
  }
  int launch(hipStream_t st) {
    if (a.jobs == 0) return CL3D_OK;
    if (groups > 0x7fffffffll) return fail(CL3D_E_UNSUPPORTED, "gated_ffn: sizes outside what the kernels index");
    const dim3 grid((unsigned)groups);
    if (s.dtype == CL3D_F32) hipLaunchKernelGGL((ffn_pack_kernel<F32, Bf16>), grid, dim3(256), 0, st, a);
    else if (s.dtype == CL3D_BF16) hipLaunchKernelGGL((ffn_pack_kernel<Bf16, Bf16>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((ffn_pack_kernel<F16, F16>), grid, dim3(256), 0, st, a);
    return CL3D_OK;
  }
};

template <int KIND, typename E, typename T, int NP, int BI, int BJ, int WI, int WJ, int BK>
static int gemm_as(const GemmArgs &a, hipStream_t st) {
  constexpr int kCh = KIND == GEMM_GATED || KIND == GEMM_GATED_BWD ? BI / 2 : BI;
  constexpr int kLds = 2 * NP * (BI + BJ) * BK * 2;
  const auto kernel = ffn_gemm_kernel<KIND, E, T, NP, BI, BJ, WI, WJ, BK>;
  static std::atomic<unsigned long long> granted{0};
  if (kLds > 65536) {
    const int rc = lds_opt_in(granted, reinterpret_cast<const void *>(kernel), kLds, "gated_ffn");
    if (rc != CL3D_OK) return rc;
  }
  const long long tiles = (long long)ceil_div(a.I, kCh) * ceil_div(a.J, BJ);
  if (tiles > 0x7fffffffll) return fail(CL3D_E_UNSUPPORTED, "gated_ffn: sizes outside what the kernels index");
  hipLaunchKernelGGL(kernel, dim3((unsigned)tiles), dim3(64 * WI * WJ), kLds, st, a);
  return CL3D_OK;
}

static bool pads_less_by_96(int I) { return ceil_div(I, 96) * 96 < ceil_div(I, 128) * 128; }

// The tile of a product.  Measured at 16 384 x 288 x 1152 in bf16 and 16 384 x 144 x 576 in f32 (us):
//   * dX and Y: rows of tiles of 96 results where they pad the width less than 128 do (widths 144, 288, 576 fit 96), 64 points a
//     tile, so that three workgroups share a CU and 768 of them come out even: dX 36 (96 x 128: 39, 128 x 128: 42), Y 20 (23, 24);
//     split: dX in 64 x 64, three workgroups a CU, 51 (96 x 128 by eight waves: 62), Y in 96 x 128 26 (64 x 64: 29, 128 x 128: 30);
//   * projections, forward and backward: 64 channels of both x 128 points by eight waves, 36 and 68 (four waves: 50, 86; 64 k a
//     tile forward: 39, 32 backward: 79); split: 64 points by four waves, two workgroups a CU: 65, 105 (128 points: 68, 128);
//   * weight gradients (ffn_weight_kernel): 128 or 96 x 128 by eight waves (four: 39 us for 33); split: 64 x 128, two workgroups a
//     CU (128 x 128, one: 58 us for 43).
// Two tiles of k in LDS: a third one costs a workgroup of the CU (dX 44 -> 64).
template <int KIND, typename E, typename T, int NP> static int gemm_tile(const GemmArgs &a, hipStream_t st) {
  [[maybe_unused]] const bool by96 = pads_less_by_96(a.I);
  if constexpr (KIND == GEMM_NT || KIND == GEMM_NN) {
    if constexpr (NP == 3 && KIND == GEMM_NN) return gemm_as<KIND, E, T, 3, 64, 64, 2, 2, 32>(a, st);
    else if constexpr (NP == 3) return by96 ? gemm_as<KIND, E, T, 3, 96, 128, 2, 4, 32>(a, st) : gemm_as<KIND, E, T, 3, 128, 128, 2, 4, 32>(a, st);
    else return by96 ? gemm_as<KIND, E, T, 1, 96, 64, 2, 2, 64>(a, st) : gemm_as<KIND, E, T, 1, 128, 64, 2, 2, 64>(a, st);
  } else {
    if constexpr (NP == 3) return gemm_as<KIND, E, T, 3, 128, 64, 2, 2, 32>(a, st);
    else return gemm_as<KIND, E, T, 1, 128, 128, 2, 4, KIND == GEMM_GATED ? 32 : 64>(a, st);
  }
}

template <int KIND> static int gemm(const FfnShape &s, const GemmArgs &a, hipStream_t st) {
  if (a.I <= 0 || a.J <= 0) return CL3D_OK;
  if (s.split) return gemm_tile<KIND, Bf16, F32, 3>(a, st);
  if (s.dtype == CL3D_F32) return gemm_tile<KIND, Bf16, F32, 1>(a, st);
  if (s.dtype == CL3D_BF16) return gemm_tile<KIND, Bf16, Bf16, 1>(a, st);
  return gemm_tile<KIND, F16, F16, 1>(a, st);
}

static bool row_vec(const FfnShape &s, const void *D, int ldd) { return aligned16(D) && ldd % (s.dtype == CL3D_F32 ? 4 : 8) == 0; }

// The weight gradients' tiles (128 or 96 results along i, whichever pads the products of the call less; split: 64) and slices: as many
// workgroups as the chip holds at once (two on a CU), not one more -- a few workgroups of a second round would take as long as the
// whole first one (540 on 512 places: 49 us, 486: 30) --, four tiles of k in each at least
struct WeightPlan {
  int bi, tiles, slices;
};
static WeightPlan weight_plan(const FfnShape &s, bool gate_up, bool down) {
  WeightPlan best{0, 0, 0};
  long long least = 0;
  for (int bi = s.split ? 64 : 96; bi <= (s.split ? 64 : 128); bi += 32) {
    const long long gu = gate_up ? 2ll * ceil_div(s.C, bi) * ceil_div(s.H, 128) : 0, d = down ? (long long)ceil_div(s.H, bi) * ceil_div(s.C, 128) : 0;
    if (best.bi == 0 || (gu + d) * bi < least) {
      best.bi = bi;
      best.tiles = (int)(gu + d);
      least = (gu + d) * bi;
    }
  }
  const long long steps = (s.R() + 63) / 64;
  long long n = best.tiles > 0 ? 512 / best.tiles : 1;
  if (n > steps / 4) n = steps / 4;
  best.slices = (int)(n < 1 ? 1 : n > 256 ? 256 : n);
  return best;
}

template <typename E, int NP, int BI, int BJ, int WI, int WJ, int BK>
static int weights_as(const WeightArgs &a, const WeightPlan &p, hipStream_t st) {
  constexpr int kLds = 2 * NP * (BI + BJ) * BK * 2;
  const auto kernel = ffn_weight_kernel<E, NP, BI, BJ, WI, WJ, BK>;
  static std::atomic<unsigned long long> granted{0};
  if (kLds > 65536) {
    const int rc = lds_opt_in(granted, reinterpret_cast<const void *>(kernel), kLds, "gated_ffn");
    if (rc != CL3D_OK) return rc;
  }
  hipLaunchKernelGGL(kernel, dim3((unsigned)p.tiles * p.slices), dim3(64 * WI * WJ), kLds, st, a);
  return CL3D_OK;
}
template <typename E> static int weights_of(const WeightArgs &a, const WeightPlan &p, hipStream_t st) {
  return p.bi == 96 ? weights_as<E, 1, 96, 128, 2, 4, 64>(a, p, st) : weights_as<E, 1, 128, 128, 2, 4, 64>(a, p, st);
}
static int weights(const FfnShape &s, const WeightArgs &a, const WeightPlan &p, hipStream_t st) {
  if (s.split) return weights_as<Bf16, 3, 64, 128, 2, 4, 32>(a, p, st);
  return s.dtype == CL3D_F16 ? weights_of<F16>(a, p, st) : weights_of<Bf16>(a, p, st);
}

template <typename T> static void slices_sum(const SliceSums &a, hipStream_t st) {
  long long most = 0;
  bool quads = true;
  for (int w = 0; w < 3; ++w) {
    most = a.n[w] > most ? a.n[w] : most;
    quads = quads && a.n[w] % 4 == 0;
  }
  const long long lanes = quads ? most / 4 : most;
  const dim3 grid((unsigned)(lanes < 256 * 1024 ? (lanes + 255) / 256 : 1024), 3);
  if (quads) hipLaunchKernelGGL((ffn_slices_kernel<T, 4>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((ffn_slices_kernel<T, 1>), grid, dim3(256), 0, st, a);
}

static GemmArgs gemm_args(const FfnShape &s) {
  GemmArgs a{};
  a.planes = s.split ? 3 : 1;
  a.act = s.act;
  return a;
}

template <bool GATED, typename T> static void rows_launch(const RowsArgs &a, hipStream_t st) {
  const bool vec = a.ldp % T::kVec == 0 && a.ldq % T::kVec == 0 && a.K % T::kVec == 0;
  const dim3 grid(ceil_div(a.I, 16)), block(64 * kRowsWaves);
#define CL3D_ROWS(JT) \
  do { \
    if (vec) hipLaunchKernelGGL((ffn_rows_kernel<GATED, T, JT, true>), grid, block, 0, st, a); \
    else hipLaunchKernelGGL((ffn_rows_kernel<GATED, T, JT, false>), grid, block, 0, st, a); \
  } while (0)
  if (a.J <= 16) CL3D_ROWS(1);
  else if (a.J <= 32) CL3D_ROWS(2);
  else CL3D_ROWS(4);
#undef CL3D_ROWS
}
template <bool GATED> static void rows(int dtype, const RowsArgs &a, hipStream_t st) {
  if (dtype == CL3D_F32) rows_launch<GATED, F32>(a, st);
  else if (dtype == CL3D_BF16) rows_launch<GATED, Bf16>(a, st);
  else rows_launch<GATED, F16>(a, st);
}

// x and y as point-major rows, at most kRowsMost of them
static void ffn_forward_rows(const FfnShape &s, const void *x, const void *wg, const void *wu, const void *wd, void *y, void *h, hipStream_t st) {
  const int R = (int)s.R(), hp = (s.H + 7) & ~7, quad = s.dtype == CL3D_F32 ? 4 : 8;
  rows<true>(s.dtype, {wg, wu, x, s.down ? h : y, s.H, R, s.C, s.C, s.C, s.down ? hp : s.H, s.act, s.down || s.H % quad == 0}, st);
  if (s.down) rows<false>(s.dtype, {wd, nullptr, h, y, s.C, R, s.H, s.H, hp, s.C, s.act, s.C % quad == 0}, st);
}

template <typename E, typename T, int CF, int NJ, int NW> static int fused_as(const FusedArgs &a, hipStream_t st) {
  const auto kernel = ffn_fused_kernel<E, T, CF, NJ, NW>;
  constexpr int kLds = 2 * 3 * 2048 * CF;
  static std::atomic<unsigned long long> granted{0};
  if (kLds > 65536) {
    const int rc = lds_opt_in(granted, reinterpret_cast<const void *>(kernel), kLds, "gated_ffn");
    if (rc != CL3D_OK) return rc;
  }
  hipLaunchKernelGGL(kernel, dim3(ceil_div(a.J, NW * NJ * 16)), dim3(64 * NW), kLds, st, a);
  return CL3D_OK;
}
// Eight waves of 16 points: two workgroups a CU (65 536 x 144: 60 us; of 32 points, one a CU: 59, but 53 against 39 at half the
// points).  At 7 fragments only one fits either way, and 32 points read each weight half as often (65 536 x 200: 91, 125).
template <typename E, typename T, int CF> static int fused_width(const FusedArgs &a, hipStream_t st) {
  if constexpr (CF == 7)
    if (a.J >= 65536) return fused_as<E, T, CF, 2, 8>(a, st);
  return fused_as<E, T, CF, 1, 8>(a, st);
}
template <typename E, typename T> static int fused(const FusedArgs &a, hipStream_t st) {
  const int cf = (a.C + 31) / 32;
  if (cf <= 1) return fused_width<E, T, 1>(a, st);
  if (cf <= 3) return fused_width<E, T, 3>(a, st);
  if (cf <= 5) return fused_width<E, T, 5>(a, st);
  return fused_width<E, T, 7>(a, st);
}

// x in the layout of `s`, its rows of C
static int ffn_forward(const FfnShape &s, const void *x, const void *wg, const void *wu, const void *wd, void *y, void *hidden, Arena &ar,
                       bool launch, hipStream_t st) {
  const int R = (int)s.R(), hp = (s.H + 7) & ~7, out = s.down ? s.C : s.H;
  if (R <= kRowsMost && (s.split || !s.convert())) {
    const size_t e = elem_bytes(s.dtype);
    void *h = s.down ? ar.take((size_t)R * hp * e) : nullptr, *xr = s.channel() ? ar.take((size_t)R * s.C * e) : nullptr;
    void *yr = s.channel() ? ar.take((size_t)R * out * e) : y;
    if (!launch) return CL3D_OK;
    int rc = s.channel() ? transposed(s.dtype, x, s.B, s.C, s.N, xr, st) : CL3D_OK;
    if (rc != CL3D_OK) return rc;
    ffn_forward_rows(s, s.channel() ? xr : x, wg, wu, wd, yr, h, st);
    return s.channel() ? transposed(s.dtype, yr, s.B, s.N, out, y, st) : CL3D_OK;
  }
  Operands ops(s, ar);
  const Operand X = ops.take(x, s.channel(), s.B, s.N, s.C);
  const Operand G = ops.take(wg, false, 1, s.H, s.C), U = ops.take(wu, false, 1, s.H, s.C);
  Operand D, h;
  const bool whole = s.down && !s.split && s.C <= kFusedMostC && R >= kFusedFewest;
  if (s.down) {
    D = ops.take(wd, false, 1, s.C, s.H);
    if (!whole) h = {static_cast<u16 *>(hidden ? hidden : ar.take((size_t)R * hp * 2 * (s.split ? 3 : 1))), hp, (long long)R * hp};
  }
  void *rows = s.channel() ? ar.take((size_t)R * out * elem_bytes(s.dtype)) : y;
  if (!launch) return CL3D_OK;
  int rc = ops.launch(st);
  if (rc != CL3D_OK) return rc;
  if (whole) {
    const FusedArgs f{G.p, U.p, D.p, X.p, rows, static_cast<u16 *>(hidden), R, s.C, s.H, hp, G.ld, D.ld, X.ld, s.C, s.act, row_vec(s, rows, s.C)};
    if (s.dtype == CL3D_F32) rc = fused<Bf16, F32>(f, st);
    else if (s.dtype == CL3D_BF16) rc = fused<Bf16, Bf16>(f, st);
    else rc = fused<F16, F16>(f, st);
    if (rc != CL3D_OK) return rc;
    return s.channel() ? transposed(s.dtype, rows, s.B, s.N, out, y, st) : CL3D_OK;
  }
  GemmArgs a = gemm_args(s);
  a.P = G.p; a.P2 = U.p; a.Q = X.p;
  a.plane_p = G.plane; a.plane_q = X.plane;  // (wg and wu: one shape, one plane stride)
  a.ldp = G.ld; a.ldq = X.ld;
  a.I = s.H; a.J = R; a.K = a.kp = X.ld;
  if (s.down) {
    a.h = const_cast<u16 *>(h.p); a.plane_h = h.plane; a.ldh = hp;
  } else {
    a.D = rows; a.ldd = s.H; a.vec = row_vec(s, rows, s.H);
  }
  rc = gemm<GEMM_GATED>(s, a, st);
  if (rc != CL3D_OK) return rc;
  if (s.down) {
    a = gemm_args(s);
    a.P = D.p; a.Q = h.p;
    a.plane_p = D.plane; a.plane_q = h.plane;
    a.ldp = D.ld; a.ldq = hp;
    a.I = s.C; a.J = R; a.K = a.kp = hp;
    a.D = rows; a.ldd = s.C; a.vec = row_vec(s, rows, s.C);
    rc = gemm<GEMM_NT>(s, a, st);
    if (rc != CL3D_OK) return rc;
  }
  return s.channel() ? transposed(s.dtype, rows, s.B, s.N, out, y, st) : CL3D_OK;
}

static int ffn_backward(const FfnShape &s, const void *x, const void *wg, const void *wu, const void *wd, const void *dy,
                        const void *hidden, void *dx, void *dwg, void *dwu, void *dwd, unsigned wants, Arena &ar, bool launch, hipStream_t st) {
  const int R = (int)s.R(), hp = (s.H + 7) & ~7, planes = s.split ? 3 : 1;
  const bool want_x = wants & CL3D_FFN_DX, want_gu = wants & CL3D_FFN_DW_IN, want_d = s.down && (wants & CL3D_FFN_DW_DOWN);
  Operands ops(s, ar);
  const Operand X = ops.take(x, s.channel(), s.B, s.N, s.C);
  const Operand G = ops.take(wg, false, 1, s.H, s.C), U = ops.take(wu, false, 1, s.H, s.C);
  Operand D, dY, h;
  const void *dh_rows = dy;
  if (s.down) {
    D = ops.take(wd, false, 1, s.C, s.H);
    dY = ops.take(dy, s.channel(), s.B, s.N, s.C);
    if (want_d) h = {static_cast<const u16 *>(hidden ? hidden : ar.take((size_t)R * hp * 2 * planes)), hp, (long long)R * hp};
  } else if (s.channel()) {
    void *t = ar.take((size_t)R * s.H * elem_bytes(s.dtype));
    if (launch) {
      const int rc = transposed(s.dtype, dy, s.B, s.H, s.N, t, st);
      if (rc != CL3D_OK) return rc;
    }
    dh_rows = t;
  }
  u16 *dgu = static_cast<u16 *>(ar.take((size_t)R * 2 * hp * 2 * planes));
  void *dx_rows = dx;
  if (s.channel() && want_x) dx_rows = ar.take((size_t)R * s.C * elem_bytes(s.dtype));
  const WeightPlan plan = weight_plan(s, want_gu, want_d);
  const long long n = (long long)s.H * s.C;
  float *part = want_gu || want_d ? static_cast<float *>(ar.take((size_t)((want_gu ? 2 : 0) + (want_d ? 1 : 0)) * plan.slices * n * 4)) : nullptr;
  if (!launch) return CL3D_OK;
  int rc = ops.launch(st);
  if (rc != CL3D_OK) return rc;
  GemmArgs a = gemm_args(s);
  a.P = G.p; a.P2 = U.p; a.Q = X.p;
  a.plane_p = G.plane; a.plane_q = X.plane;
  a.ldp = G.ld; a.ldq = X.ld;
  a.I = s.H; a.J = R; a.K = X.ld;
  if (s.down) {
    a.Pb = D.p; a.Qb = dY.p;
    a.plane_pb = D.plane; a.plane_qb = dY.plane;
    a.ldpb = D.ld; a.ldqb = dY.ld;
    a.Kb = dY.ld; a.kp = s.C;
    if (!hidden) { a.h = const_cast<u16 *>(h.p); a.plane_h = h.plane; }
  } else {
    a.dh = dh_rows; a.lddh = s.H;
  }
  a.dgu = dgu; a.plane_dgu = (long long)R * 2 * hp; a.ldh = hp;
  rc = gemm<GEMM_GATED_BWD>(s, a, st);
  if (rc != CL3D_OK) return rc;
  if (want_x) {
    a = gemm_args(s);
    a.P = G.p; a.Pb = U.p; a.Q = dgu; a.Qb = dgu + hp;
    a.plane_p = G.plane; a.plane_q = (long long)R * 2 * hp;
    a.ldp = G.ld; a.ldq = 2 * hp;
    a.I = s.C; a.J = R; a.K = hp; a.kp = s.H;
    a.D = dx_rows; a.ldd = s.C; a.vec = row_vec(s, dx_rows, s.C);
    rc = gemm<GEMM_NN>(s, a, st);
    if (rc != CL3D_OK) return rc;
    if (s.channel()) rc = transposed(s.dtype, dx_rows, s.B, s.N, s.C, dx, st);
    if (rc != CL3D_OK) return rc;
  }
  if (!want_gu && !want_d) return CL3D_OK;
  WeightArgs w{};
  SliceSums sums{};
  w.K = R;
  w.slices = plan.slices;
  auto add = [&](const Operand &p, const u16 *q, long long plane_q, int ldq, int I, int J, void *dst) {
    const int k = w.products++;
    w.P[k] = p.p; w.Q[k] = q;
    w.plane_p[k] = p.plane; w.plane_q[k] = plane_q;
    w.ldp[k] = p.ld; w.ldq[k] = ldq;
    w.I[k] = I; w.J[k] = J; w.vec[k] = I % 4 == 0;
    w.D[k] = part + k * n * plan.slices;
    sums.src[k] = w.D[k]; sums.dst[k] = dst; sums.n[k] = n; sums.slices[k] = plan.slices;
  };
  if (want_gu) {
    add(X, dgu, (long long)R * 2 * hp, 2 * hp, s.C, s.H, dwg);
    add(X, dgu + hp, (long long)R * 2 * hp, 2 * hp, s.C, s.H, dwu);
  }
  if (want_d) add(h, dY.p, dY.plane, dY.ld, s.H, s.C, dwd);
  rc = weights(s, w, plan, st);
  if (rc != CL3D_OK) return rc;
  if (s.dtype == CL3D_F32) slices_sum<F32>(sums, st);
  else if (s.dtype == CL3D_BF16) slices_sum<Bf16>(sums, st);
  else slices_sum<F16>(sums, st);
  return CL3D_OK;
}

static int ffn_shape(FfnShape &s, int dtype, int order, int B, int N, int C, int H, int activation, int precision, bool down,
                     const char *who) {
  CL3D_REQUIRE(dtype == CL3D_F32 || dtype == CL3D_BF16 || dtype == CL3D_F16, "%s: unknown element type %d", who, dtype);
  CL3D_REQUIRE(order == CL3D_POINT_MAJOR || order == CL3D_CHANNEL_MAJOR, "%s: unknown memory order %d", who, order);
  CL3D_REQUIRE(activation >= CL3D_ACT_SILU && activation <= CL3D_ACT_RELU, "%s: unknown activation %d", who, activation);
  CL3D_REQUIRE(precision == 0 || precision == 1, "%s: unknown precision %d", who, precision);
  CL3D_REQUIRE(B >= 0 && N >= 0 && C > 0 && H > 0, "%s: bad sizes", who);
  // descriptors of a tile span 64 rows of 2 H or 128 rows of C elements with 31 bits
  if (C > (1 << 20) || H > (1 << 20) || (long long)B * N > 0x7fffff00ll ||
      (order == CL3D_CHANNEL_MAJOR && (B > 65535 || N > 65535 * 64)))
    return fail(CL3D_E_UNSUPPORTED, "%s: sizes outside what the kernels index", who);
  s = {dtype, order, B, N, C, H, activation, dtype == CL3D_F32 && precision == 0, down};
  return CL3D_OK;
}

size_t gated_ffn_workspace(int B, int N, int H, int flags, int C) {
  // flags: element type | order << 2 | precision << 3 | down << 4 | backward << 5 | wanted gradients << 6 | hidden kept << 9
  FfnShape s;
  if (ffn_shape(s, flags & 3, (flags >> 2) & 1, B, N, C, H, CL3D_ACT_SILU, (flags >> 3) & 1, (flags >> 4) & 1, "gated_ffn") != CL3D_OK)
    return 0;
  Arena ar(nullptr);
  char kept;  // (only asked whether it is there)
  void *hidden = (flags >> 9) & 1 ? &kept : nullptr;
  if ((flags >> 5) & 1)
    ffn_backward(s, nullptr, nullptr, nullptr, nullptr, nullptr, hidden, nullptr, nullptr, nullptr, nullptr, ((unsigned)flags >> 6) & 7u, ar, false, nullptr);
  else ffn_forward(s, nullptr, nullptr, nullptr, nullptr, nullptr, hidden, ar, false, nullptr);
  return ar.used;
}

}  // namespace cl3d

extern "C" int cl3d_gated_ffn_fwd(const void *x, const void *w_gate, const void *w_up, const void *w_down, int dtype, int order, int B,
                                  int C, int N, int H, int activation, int precision, void *y, void *hidden, void *ws, size_t ws_bytes,
                                  cl3d_stream_t stream) {
  using namespace cl3d;
  FfnShape s;
  int rc = ffn_shape(s, dtype, order, B, N, C, H, activation, precision, w_down != nullptr, "gated_ffn_fwd");
  if (rc != CL3D_OK) return rc;
  if (s.R() == 0) return CL3D_OK;
  CL3D_REQUIRE(x && w_gate && w_up && y, "gated_ffn_fwd: null pointer");
  CL3D_REQUIRE(aligned16(x) && aligned16(w_gate) && aligned16(w_up) && aligned16(w_down) && aligned16(y) && aligned16(hidden) &&
                   aligned16(ws),
               "gated_ffn_fwd: tensors start on 16 bytes");
  CL3D_REQUIRE(!hidden || (w_down && s.R() > CL3D_FFN_FEW), "gated_ffn_fwd: no hidden activations are kept here");
  Arena need(nullptr), ar(ws);
  ffn_forward(s, x, w_gate, w_up, w_down, y, hidden, need, false, nullptr);
  if (ws_bytes < need.used || (need.used && !ws)) return fail(CL3D_E_WORKSPACE, "gated_ffn_fwd: %zu bytes of scratch, %zu needed", ws_bytes, need.used);
  rc = ffn_forward(s, x, w_gate, w_up, w_down, y, hidden, ar, true, (hipStream_t)stream);
  return rc != CL3D_OK ? rc : check_launch("cl3d_gated_ffn_fwd");
}

extern "C" int cl3d_gated_ffn_bwd(const void *x, const void *w_gate, const void *w_up, const void *w_down, const void *dy,
                                  const void *hidden, int dtype, int order, int B, int C, int N, int H, int activation, int precision, void *dx, void *dw_gate,
                                  void *dw_up, void *dw_down, void *ws, size_t ws_bytes, cl3d_stream_t stream) {
  using namespace cl3d;
  FfnShape s;
  int rc = ffn_shape(s, dtype, order, B, N, C, H, activation, precision, w_down != nullptr, "gated_ffn_bwd");
  if (rc != CL3D_OK) return rc;
  CL3D_REQUIRE(s.R() > 0, "gated_ffn_bwd: no points (their gradients are zeros: nothing to launch)");
  CL3D_REQUIRE(x && w_gate && w_up && dy, "gated_ffn_bwd: null pointer");
  CL3D_REQUIRE(w_down != nullptr || dw_down == nullptr, "gated_ffn_bwd: a gradient for a projection that is not there");
  CL3D_REQUIRE(aligned16(x) && aligned16(w_gate) && aligned16(w_up) && aligned16(w_down) && aligned16(dy) && aligned16(hidden) && aligned16(dx) &&
                   aligned16(dw_gate) && aligned16(dw_up) && aligned16(dw_down) && aligned16(ws),
               "gated_ffn_bwd: tensors start on 16 bytes");
  const unsigned wants = (dx ? CL3D_FFN_DX : 0u) | (dw_gate || dw_up ? CL3D_FFN_DW_IN : 0u) | (dw_down ? CL3D_FFN_DW_DOWN : 0u);
  if (wants == 0) return CL3D_OK;
  Arena need(nullptr), ar(ws);
  ffn_backward(s, x, w_gate, w_up, w_down, dy, hidden, dx, dw_gate, dw_up, dw_down, wants, need, false, nullptr);
  if (ws_bytes < need.used || (need.used && !ws)) return fail(CL3D_E_WORKSPACE, "gated_ffn_bwd: %zu bytes of scratch, %zu needed", ws_bytes, need.used);
  rc = ffn_backward(s, x, w_gate, w_up, w_down, dy, hidden, dx, dw_gate, dw_up, dw_down, wants, ar, true, (hipStream_t)stream);
  return rc != CL3D_OK ? rc : check_launch("cl3d_gated_ffn_bwd");
}
