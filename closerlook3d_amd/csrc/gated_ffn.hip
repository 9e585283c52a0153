// gated_ffn.hip -- the gated feed-forward of a point:  Y = (act(X Wg^T) * (X Wu^T)) Wd^T  and its gradients, on the matrix cores.
//
// X [R, C] point-major rows (R = clouds x points), Wg, Wu [H, C], Wd [C, H] as nn.Linear holds them.
//     G = X Wg^T, U = X Wu^T, h = act(G) U;   Y = h Wd^T
//     dh = dY Wd;  dG = dh U act'(G);  dU = dh act(G);   dX = dG Wg + dU Wu;   dWg = dG^T X, dWu = dU^T X, dWd = dY^T h
// Three products of 2 R C H operations forward and six backward.  G and U never reach memory: the forward kernel keeps both
// accumulators of an element in one lane and writes h, the backward kernel forms G, U and dh together (two products more) and
// writes h, dG, dU.  Against storing G and U that is 8 R H bytes less traffic for 4 R C H operations more -- at 5.1 TB/s and
// 1.28 PFLOP/s (a large copy, a large product) it pays below C = 500 -- and dG, dU come from f32 values of G, U, dh: one
// rounding in front of the last products instead of two.
//
// One kernel template.  D[j][i] = sum_k P(i, k) Q(j, k), i contiguous in the result; P is the first MFMA operand, so a lane of
// v_mfma_f32_16x16x32 holds four consecutive i of one j.
//   * tiles travel HBM -> LDS by buffer_load ... lds (16 bytes a lane, no registers); a lane behind the end of a row or of the
//     tensor is sent out of the descriptor's range and fills its place with zeros, so ragged sizes need no second kernel;
//   * two LDS tiles of 64 k each: the next one is in flight while this one is multiplied;
//   * an operand whose k is contiguous lies in LDS as [row][64 k], 16-byte pieces XORed with the row, read by ds_read_b128; one
//     whose row index is contiguous (Wd in dh, Wg / Wu in dX, all operands of the weight gradients) lies as [64 k][row] and is
//     read by ds_read_b64_tr_b16, which hands a lane four k of its row: no operand is transposed in memory;
//   * workgroups are numbered so that neighbours in i, which share the rows of Q, run on one XCD and share its L2.
// f32 tensors: an f32 value is the exact sum of three bf16 values (8 significant bits each, by truncation); the product takes the
// six largest of the nine partial products on the bf16 units, smallest first, into one f32 accumulator.  What is left out is
// below 2^-23 of |x||y|, as much as the rounding of an f32 product.  Six passes at the bf16 rate outrun the f32 MFMA (1/16 of it).
// A value that is not finite takes part in the leading product only (a fourth plane holds 0 for it), so an infinity stays one.
#include "ff_common.h"

namespace cl3d {

typedef unsigned short u16;

constexpr int kBK = 64;                // k per LDS tile
constexpr int kRowBytes = kBK * 2;

// which plane of P and Q each pass of a split product takes (0 leading, 1 middle, 2 last, 3 leading but 0 if not finite): hex
// digits, the first pass lowest -- (2,3) (3,2) (1,1) (1,3) (3,1) (0,0)
constexpr unsigned kSegP = 0x031132u, kSegQ = 0x013123u;

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

// s_waitcnt vmcnt(n), the other counters left alone
template <int N> __device__ __forceinline__ void wait_vm() {
  __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | (15 << 8) | ((N >> 4) << 14));
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
template <bool PAIRED> __device__ __forceinline__ int swz_kc(int row) {
  return PAIRED ? (((row >> 1) & 1) | ((row >> 2) & 6)) : ((row >> 1) & 7);
}
template <int ROWS> __device__ __forceinline__ int swz_km(int k) {  // (32-byte blocks: ds_read_b64_tr_b16 takes them whole)
  return ROWS >= 128 ? (((k & 3) | ((k >> 1) & 4)) << 1) : ((((k >> 1) & 1) | ((k >> 2) & 2)) << 1);
}

template <int ROWS, bool KM, bool PAIRED, int NW> struct Loader {
  static constexpr int kPer = ROWS * 8 / (64 * NW);  // 16-byte pieces per lane
  static_assert(kPer >= 1 && kPer * 64 * NW == ROWS * 8, "tile and workgroup do not match");
  unsigned off[kPer];
  int at[kPer];  // KM false: k of the piece

  __device__ __forceinline__ void init(int ld, int rows, int wave, int lane) {
#pragma unroll
    for (int q = 0; q < kPer; ++q) {
      const int slot = (wave * kPer + q) * 64 + lane;
      if (!KM) {
        const int row = slot >> 3, chunk = (slot & 7) ^ swz_kc<PAIRED>(row);
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
    const int outer = KM ? (kleft < kBK ? kleft : kBK) : (rows < ROWS ? rows : ROWS), inner = KM ? rows : kleft;
    const unsigned bytes = (unsigned)((outer - 1) * ld + inner) * 2u;
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void *)base, 0, bytes, 0x00020000);
#pragma unroll
    for (int q = 0; q < kPer; ++q) {
      unsigned o = off[q];
      if (!KM && kleft < kBK) o = at[q] < kleft ? o : 0x80000000u;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, CL3D_LDS(void, lds + (wave * kPer + q) * 1024), 16, o, 0, 0, 0);
    }
  }
};

// fragment of 16 rows for k = 32 kk .. 32 kk + 31: lane l holds row l & 15, k = 8 (l >> 4) .. + 7.
// r0: first row of the 16 (PAIRED: of the 32; t says which half of every eight)
template <bool PAIRED> __device__ __forceinline__ s16x8 frag_kc(const char *lds, int r0, int t, int kk, int lane) {
  const int m = lane & 15, row = r0 + (PAIRED ? 8 * (m >> 2) + 4 * t + (m & 3) : m);
  return *reinterpret_cast<const s16x8 *>(lds + row * kRowBytes + (((kk * 4 + (lane >> 4)) ^ swz_kc<PAIRED>(row)) << 4));
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

// acc[a][b] += the product over steps [s0, s1) of nseg * ceil(K / 64).  PR: rows of P in a tile (TWO: the first half from P, the
// second from P2).  The wave (wi, wj) owns TI / 16 x TJ / 16 accumulators; TWO: first TI / 32 of P, then as many of P2, same rows.
template <typename E, int PR, bool PKM, bool PAIRED, bool TWO, int QR, bool QKM, int TI, int TJ, int NW>
__device__ __forceinline__ void product(f32x4 (&acc)[TI / 16][TJ / 16], const Pair &a, int nseg, int s0, int s1, char *smem,
                                        int wave, int lane, int wi, int wj) {
  constexpr int kPBytes = PR * kRowBytes, kStage = (PR + QR) * kRowBytes;
  constexpr int kPR = TWO ? PR / 2 : PR;
  Loader<PR, PKM, PAIRED, NW> lp;
  Loader<QR, QKM, false, NW> lq;
  static_assert(!(TWO && PKM), "two matrices: k contiguous");
  // TWO: this wave's pieces are all of one matrix (kPR rows are a whole number of waves' shares)
  const bool second = TWO && wave * lp.kPer * 8 >= kPR;
  lp.init(a.ldp, a.rows_p, wave, lane);
  lq.init(a.ldq, a.rows_q, wave, lane);
  const int ksteps = (a.K + kBK - 1) / kBK;
  const u16 *Pb = a.P;
  if (TWO && second) Pb = a.P2 - (long long)kPR * a.ldp;

  // (what a step reads is counted up, not divided out: a quotient is formed in vector registers, and the descriptors with it)
  int seg = 0, k_next = 0, k_now = 0;
  if (s0 > 0) {
    seg = __builtin_amdgcn_readfirstlane(s0 / ksteps);
    k_next = k_now = (s0 - seg * ksteps) * kBK;
  }
  auto issue = [&](int buf) {
    const long long pp = nseg > 1 ? (long long)((kSegP >> 4 * seg) & 15u) * a.plane_p : 0, pq = nseg > 1 ? (long long)((kSegQ >> 4 * seg) & 15u) * a.plane_q : 0;
    char *lds = smem + buf * kStage;
    const u16 *P = Pb + pp + (PKM ? (long long)k_next * a.ldp : k_next), *Q = a.Q + pq + (QKM ? (long long)k_next * a.ldq : k_next);
    // rows behind the tile's end: beyond the descriptor (TWO: its rows are counted from the tile's first row)
    lp.issue(P, a.ldp, TWO && second ? a.rows_p + kPR : (TWO ? (a.rows_p < kPR ? a.rows_p : kPR) : a.rows_p),
             (PKM ? a.kp : a.K) - k_next, lds, wave);
    lq.issue(Q, a.ldq, a.rows_q, a.K - k_next, lds + kPBytes, wave);
    k_next += kBK;
    if (k_next >= a.K) {
      k_next = 0;
      ++seg;
    }
  };
  if (s0 >= s1) return;
  issue(0);
  int buf = 0;
  for (int s = s0; s < s1; ++s) {
    if (s + 1 < s1) {
      issue(buf ^ 1);
      wait_vm<lp.kPer + lq.kPer>();
    } else {
      wait_vm<0>();
    }
    barrier_lds();
    const char *lds = smem + buf * kStage;
    const int k0 = k_now;
    k_now = k_now + kBK >= a.K ? 0 : k_now + kBK;
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      if (k0 + kk * 32 < a.K) {
        s16x8 p[TI / 16], q[TJ / 16];
#pragma unroll
        for (int u = 0; u < TI / 16; ++u) {
          const int half = TWO ? u / (TI / 32) : 0, v = TWO ? u % (TI / 32) : u;
          const int r0 = half * kPR + wi * (TWO ? TI / 2 : TI) + (PAIRED ? (v >> 1) * 32 : v * 16);
          p[u] = PKM ? frag_km<PR, PAIRED>(lds, r0, v & 1, kk, lane) : frag_kc<PAIRED>(lds, r0, v & 1, kk, lane);
        }
#pragma unroll
        for (int u = 0; u < TJ / 16; ++u) {
          const int r0 = wj * TJ + u * 16;
          q[u] = QKM ? frag_km<QR, false>(lds + kPBytes, r0, 0, kk, lane) : frag_kc<false>(lds + kPBytes, r0, 0, kk, lane);
        }
#pragma unroll
        for (int u = 0; u < TI / 16; ++u)
#pragma unroll
          for (int v = 0; v < TJ / 16; ++v) acc[u][v] = mfma16<E>(p[u], q[v], acc[u][v]);
      }
    }
    barrier_lds();
    buf ^= 1;
  }
}

// ---- activations (CL3D_ACT_SILU / _GELU / _RELU): value and slope at g
__device__ __forceinline__ void activate(int act, float g, float &value, float &slope) {
  if (act == CL3D_ACT_SILU) {
    const float s = 1.f / (1.f + expf(-g));
    value = g * s;
    slope = s * __builtin_fmaf(g, 1.f - s, 1.f);
  } else if (act == CL3D_ACT_GELU) {
    const float c = 0.5f * (1.f + erff(g * 0.70710678118654752f));
    value = g * c;
    slope = __builtin_fmaf(g, 0.3989422804014327f * expf(-0.5f * g * g), c);
  } else {  // relu; a NaN stays one, the slope at 0 is 0
    value = g < 0.f ? 0.f : g;
    slope = g > 0.f ? 1.f : (g <= 0.f ? 0.f : g);
  }
}

// an f32 value as the exact sum of three bf16 values by truncation; plane 3 is the leading one, 0 where x is not finite
struct Split {
  u16 p[4];
};
__device__ __forceinline__ Split split3(float x) {
  const unsigned b = __float_as_uint(x), hi = b & 0xffff0000u;
  Split s;
  s.p[0] = (u16)(hi >> 16);
  if ((b & 0x7f800000u) == 0x7f800000u) {
    if (b & 0x007fffffu) s.p[0] |= 0x40;  // a NaN whose payload sits in the low half stays a NaN
    s.p[1] = s.p[2] = s.p[3] = 0;
    return s;
  }
  const float r = x - __uint_as_float(hi);
  const unsigned mid = __float_as_uint(r) & 0xffff0000u;
  s.p[1] = (u16)(mid >> 16);
  s.p[2] = (u16)(__float_as_uint(r - __uint_as_float(mid)) >> 16);
  s.p[3] = s.p[0];
  return s;
}

struct GemmArgs {
  const u16 *P, *P2, *Q;     // first product
  const u16 *Pb, *Qb;        // GATED_BWD: dh = Wd, dY; NN: the second pair of dX
  long long plane_p, plane_q, plane_pb, plane_qb;
  int ldp, ldq, ldpb, ldqb;
  int I, J, K, Kb, kp;       // K, Kb multiples of 8 (zero-padded operands); kp: rows of the P whose rows run along i
  int nseg, act;
  int slices;                // weight gradients: pieces of k
  int batch_q, batch_d;      // weight gradients: blockIdx.z picks Q + z * batch_q, D + z * batch_d
  void *D;                   // result rows of ldd elements of the tensor type (or f32 partials [slice][J][I])
  int ldd, vec;              // vec: rows start 16-byte aligned
  u16 *h, *dgu;              // operand-type intermediates, ldh and 2 ldh a row, zero up to ldh; 4 planes when split
  long long plane_h, plane_dgu;
  int ldh, planes;
  const void *dh;            // GATED_BWD without a down projection: dh itself, rows of lddh
  int lddh;
};

// four or eight consecutive elements of an internal row: operand type, or the four planes
template <typename E, int N> __device__ __forceinline__ void put_internal(u16 *row, long long plane, int planes, const float *v) {
  if (planes == 1) {
    u16 o[N];
#pragma unroll
    for (int e = 0; e < N; ++e) o[e] = E::put(v[e]);
    if constexpr (N == 8) *reinterpret_cast<s16x8 *>(row) = *reinterpret_cast<s16x8 *>(o);
    else *reinterpret_cast<s16x4 *>(row) = *reinterpret_cast<s16x4 *>(o);
    return;
  }
  u16 o[4][N];
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const Split s = split3(v[e]);
#pragma unroll
    for (int p = 0; p < 4; ++p) o[p][e] = s.p[p];
  }
#pragma unroll
  for (int p = 0; p < 4; ++p) {
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

enum { GEMM_NT = 0, GEMM_NN = 1, GEMM_TN = 2, GEMM_GATED = 3, GEMM_GATED_BWD = 4 };

// linear workgroup number -> tile: the hardware deals workgroups to the 8 XCDs in turn; each XCD gets a run of neighbours
__device__ __forceinline__ int xcd_order(int id, int total) {
  const int x = id & 7, q = id >> 3, per = total >> 3, rem = total & 7;
  return x * per + (x < rem ? x : rem) + q;
}

// E: operand type; T: type of the caller's tensors.  A workgroup of WI x WJ waves owns BI x BJ results (GATED*: BI is twice the
// channels).
template <int KIND, typename E, typename T, int BI, int BJ, int WI, int WJ>
__global__ __launch_bounds__(64 * WI * WJ) void ffn_gemm_kernel(GemmArgs a) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  constexpr int NW = WI * WJ, TI = BI / WI, TJ = BJ / WJ;
  constexpr bool kTwo = KIND == GEMM_GATED || KIND == GEMM_GATED_BWD;
  constexpr int kCh = kTwo ? BI / 2 : BI;  // result columns of the workgroup
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wi = wave / WJ, wj = wave % WJ;
  const int ti = (a.I + kCh - 1) / kCh, tj = (a.J + BJ - 1) / BJ;
  int id = xcd_order(blockIdx.x, gridDim.x);
  const int slice = KIND == GEMM_TN ? __builtin_amdgcn_readfirstlane(id / (ti * tj)) : 0;
  id -= slice * (ti * tj);
  const int row = __builtin_amdgcn_readfirstlane(id / ti);
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
    const int steps = (a.K + kBK - 1) / kBK * a.nseg;
    product<E, BI, false, true, true, BJ, false, TI, TJ, NW>(acc, pr, a.nseg, 0, steps, smem, wave, lane, wi, wj);
    f32x4 dh[TI / 32][TJ / 16];
    if constexpr (KIND == GEMM_GATED_BWD) {
#pragma unroll
      for (int u = 0; u < TI / 32; ++u)
#pragma unroll
        for (int v = 0; v < TJ / 16; ++v) dh[u][v] = (f32x4){0.f, 0.f, 0.f, 0.f};
      if (a.Qb != nullptr) {
        Pair pb{a.Pb + i0, nullptr, a.Qb + (long long)j0 * a.ldqb, a.plane_pb, a.plane_qb, a.ldpb, a.ldqb, ip - i0, a.J - j0, a.Kb,
                a.kp};
        const int sb = (a.Kb + kBK - 1) / kBK * a.nseg;
        product<E, BI / 2, true, true, false, BJ, false, TI / 2, TJ, NW>(dh, pb, a.nseg, 0, sb, smem, wave, lane, wi, wj);
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
    Pair pr{kKm ? a.P + i0 : a.P + (long long)i0 * a.ldp, nullptr, a.Q + (long long)j0 * a.ldq, a.plane_p, a.plane_q, a.ldp, a.ldq,
            kKm ? ip - i0 : a.I - i0, a.J - j0, a.K, a.kp};
    const int steps = (a.K + kBK - 1) / kBK * a.nseg;
    product<E, BI, kKm, !kKm, false, BJ, false, TI, TJ, NW>(acc, pr, a.nseg, 0, steps, smem, wave, lane, wi, wj);
    if (kKm && a.Pb != nullptr) {  // dX = dG Wg + dU Wu
      pr.P = a.Pb + i0;
      pr.Q = a.Qb + (long long)j0 * a.ldq;
      product<E, BI, kKm, !kKm, false, BJ, false, TI, TJ, NW>(acc, pr, a.nseg, 0, steps, smem, wave, lane, wi, wj);
    }
    auto *D = static_cast<typename T::storage *>(a.D);
#pragma unroll
    for (int v = 0; v < TJ / 16; ++v) {
      const int j = j0 + wj * TJ + v * 16 + (lane & 15);
      if (j >= a.J) continue;
      if constexpr (!kKm) {
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
  } else {  // TN: a slice of a weight gradient, f32 partials [batch][slice][J][I]
    const int z = blockIdx.z, jp = (a.J + 7) & ~7;
    Pair pr{a.P + i0, nullptr, a.Q + (long long)z * a.batch_q + j0, a.plane_p, a.plane_q, a.ldp, a.ldq, ip - i0, jp - j0, a.K,
            a.K};
    const long long steps = (long long)((a.K + kBK - 1) / kBK) * a.nseg;
    const int s0 = __builtin_amdgcn_readfirstlane((int)(steps * slice / a.slices));
    const int s1 = __builtin_amdgcn_readfirstlane((int)(steps * (slice + 1) / a.slices));
    product<E, BI, true, false, false, BJ, true, TI, TJ, NW>(acc, pr, a.nseg, s0, s1, smem, wave, lane, wi, wj);
    float *D = static_cast<float *>(a.D) + ((long long)z * a.slices + slice) * a.J * a.I;
#pragma unroll
    for (int v = 0; v < TJ / 16; ++v) {
      const int j = j0 + wj * TJ + v * 16 + (lane & 15);
      if (j >= a.J) continue;
#pragma unroll
      for (int u = 0; u < TI / 16; ++u) {
        const int c0 = i0 + wi * TI + u * 16 + 4 * g;
        float o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = acc[u][v][e];
        if (c0 < a.I) put_row<F32, 4>(D + (long long)j * a.I + c0, a.I - c0, a.vec, o);
      }
    }
  }
}

// dst[e] = sum over slices of src[slice][e], in slice order
template <typename T>
__global__ __launch_bounds__(256) void ffn_slices_kernel(const float *__restrict__ src, long long n, int slices,
                                                         typename T::storage *__restrict__ dst) {
  for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < n; e += (long long)gridDim.x * 256) {
    float s = 0.f;
    for (int z = 0; z < slices; ++z) s += src[(long long)z * n + e];
    dst[e] = T::put(s);
  }
}

// ---- operands that are not what the products read: another memory order, odd rows, f32 ---------------------------------
// source element (b, r, c) at src + b sb + r sr + c sc, one of sr, sc being 1; out rows [(b, r)] of ld elements, zero behind C.
// `planes` 4: the split of an f32 value; 1: one rounding to E (none when S is E).
template <typename S, typename E>
__global__ __launch_bounds__(256) void ffn_pack_kernel(const typename S::storage *__restrict__ src, long long sb, long long sr,
                                                       long long sc, int Rb, int C, u16 *__restrict__ dst, int ld, long long plane,
                                                       int planes) {
  __shared__ float tile[32][65];
  const int b = blockIdx.z, r0 = blockIdx.x * 32, c0 = blockIdx.y * 64;
  const int tid = threadIdx.x;
  const typename S::storage *s = src + (long long)b * sb;
  for (int e = tid; e < 32 * 64; e += 256) {
    const int r = sc == 1 ? e >> 6 : e & 31, c = sc == 1 ? e & 63 : e >> 5;
    tile[r][c] = r0 + r < Rb && c0 + c < C ? S::get(s[(r0 + r) * sr + (c0 + c) * sc]) : 0.f;
  }
  __syncthreads();
  const int r = tid >> 3, c = (tid & 7) * 8;  // 32 rows x 8 pieces of 8
  if (r0 + r >= Rb || c0 + c >= ld) return;
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = tile[r][c + e];
  put_internal<E, 8>(dst + ((long long)b * Rb + r0 + r) * ld + c0 + c, plane, planes, v);
}

// ---- host side -----------------------------------------------------------------------------------------------------
// scratch in order; without a base it only counts
struct Arena {
  char *base;
  size_t used = 0;
  explicit Arena(void *p) : base(static_cast<char *>(p)) {}
  void *take(size_t bytes) {
    used = (used + 255) & ~(size_t)255;
    char *p = base ? base + used : nullptr;
    used += bytes;
    return p;
  }
};

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

template <typename S, typename E>
static void pack_launch(const void *src, long long sb, long long sr, long long sc, int B, int Rb, int C, u16 *dst, int ld, long long plane,
                        int planes, hipStream_t st) {
  const dim3 grid(ceil_div(Rb, 32), ceil_div(ld, 64), B);
  hipLaunchKernelGGL((ffn_pack_kernel<S, E>), grid, dim3(256), 0, st, static_cast<const typename S::storage *>(src), sb, sr, sc, Rb, C, dst,
                     ld, plane, planes);
}

// rows [(b, r)][C] as the products read them: the caller's own memory where it is already that, else a packed copy
static Operand operand(Arena &ar, const FfnShape &s, const void *src, bool channel, int B, int Rb, int C, bool launch, hipStream_t st) {
  const int ld = (C + 7) & ~7;
  if (!s.convert() && !channel && C % 8 == 0) return {static_cast<const u16 *>(src), C, 0};
  const long long plane = (long long)B * Rb * ld;
  const int planes = s.split ? 4 : 1;
  u16 *dst = static_cast<u16 *>(ar.take((size_t)plane * planes * 2));
  if (launch) {
    // rows that follow each other without regard to the cloud are one batch
    const int b = channel ? B : 1, rb = channel ? Rb : B * Rb;
    const long long sb = (long long)C * Rb, sr = channel ? 1 : C, sc = channel ? Rb : 1;
    if (s.dtype == CL3D_F32) pack_launch<F32, Bf16>(src, sb, sr, sc, b, rb, C, dst, ld, plane, planes, st);
    else if (s.dtype == CL3D_BF16) pack_launch<Bf16, Bf16>(src, sb, sr, sc, b, rb, C, dst, ld, plane, planes, st);
    else pack_launch<F16, F16>(src, sb, sr, sc, b, rb, C, dst, ld, plane, planes, st);
  }
  return {dst, ld, plane};
}

// [b][R][C] -> [b][C][R] of the tensor type
static int transposed(int dtype, const void *src, int B, int R, int C, void *dst, hipStream_t st) {
  if (dtype == CL3D_F32) return cl3d_transpose(static_cast<const float *>(src), B, R, C, static_cast<float *>(dst), st);
  return cl3d_transpose16(src, B, R, C, dst, st);
}

template <int KIND, typename E, typename T, int BI, int BJ, int WI, int WJ>
static int gemm_as(const GemmArgs &a, int batches, hipStream_t st) {
  constexpr int kCh = KIND == GEMM_GATED || KIND == GEMM_GATED_BWD ? BI / 2 : BI;
  constexpr int kLds = 2 * (BI + BJ) * kRowBytes;
  const auto kernel = ffn_gemm_kernel<KIND, E, T, BI, BJ, WI, WJ>;
  static std::atomic<unsigned long long> granted{0};
  if (kLds > 65536) {
    const int rc = lds_opt_in(granted, reinterpret_cast<const void *>(kernel), kLds, "gated_ffn");
    if (rc != CL3D_OK) return rc;
  }
  const long long tiles = (long long)ceil_div(a.I, kCh) * ceil_div(a.J, BJ) * (KIND == GEMM_TN ? a.slices : 1);
  hipLaunchKernelGGL(kernel, dim3((unsigned)tiles, 1, batches), dim3(64 * WI * WJ), kLds, st, a);
  return CL3D_OK;
}

template <int KIND> static int gemm(const FfnShape &s, const GemmArgs &a, int batches, hipStream_t st) {
  if (a.I <= 0 || a.J <= 0) return CL3D_OK;
  if (s.dtype == CL3D_F32) return gemm_as<KIND, Bf16, F32, 128, 128, 2, 2>(a, batches, st);
  if (s.dtype == CL3D_BF16) return gemm_as<KIND, Bf16, Bf16, 128, 128, 2, 2>(a, batches, st);
  return gemm_as<KIND, F16, F16, 128, 128, 2, 2>(a, batches, st);
}

static bool row_vec(const FfnShape &s, const void *D, int ldd) { return aligned16(D) && ldd % (s.dtype == CL3D_F32 ? 4 : 8) == 0; }

// pieces of k in a weight gradient: enough workgroups for two on every CU, four tiles of k in each at least
static int weight_slices(const FfnShape &s, int I, int J, int batches) {
  const long long tiles = (long long)ceil_div(I, 128) * ceil_div(J, 128) * batches;
  const long long steps = (s.R() + kBK - 1) / kBK * (s.split ? 6 : 1);
  long long n = (512 + tiles - 1) / tiles;
  if (n > steps / 4) n = steps / 4;
  return (int)(n < 1 ? 1 : n > 256 ? 256 : n);
}

static int slices_sum(const FfnShape &s, const float *src, long long n, int slices, void *dst, hipStream_t st) {
  long long grid = (n + 255) / 256;
  if (grid > 2048) grid = 2048;
  if (s.dtype == CL3D_F32)
    hipLaunchKernelGGL(ffn_slices_kernel<F32>, dim3((unsigned)grid), dim3(256), 0, st, src, n, slices, static_cast<float *>(dst));
  else if (s.dtype == CL3D_BF16)
    hipLaunchKernelGGL(ffn_slices_kernel<Bf16>, dim3((unsigned)grid), dim3(256), 0, st, src, n, slices, static_cast<u16 *>(dst));
  else
    hipLaunchKernelGGL(ffn_slices_kernel<F16>, dim3((unsigned)grid), dim3(256), 0, st, src, n, slices, static_cast<u16 *>(dst));
  return CL3D_OK;
}

static GemmArgs gemm_args(const FfnShape &s) {
  GemmArgs a{};
  a.nseg = s.split ? 6 : 1;
  a.planes = s.split ? 4 : 1;
  a.act = s.act;
  a.slices = 1;
  return a;
}

// x in the layout of `s`, its rows of C
static int ffn_forward(const FfnShape &s, const void *x, const void *wg, const void *wu, const void *wd, void *y, Arena &ar, bool launch,
                       hipStream_t st) {
  const int R = (int)s.R(), hp = (s.H + 7) & ~7, out = s.down ? s.C : s.H;
  const Operand X = operand(ar, s, x, s.channel(), s.B, s.N, s.C, launch, st);
  const Operand G = operand(ar, s, wg, false, 1, s.H, s.C, launch, st), U = operand(ar, s, wu, false, 1, s.H, s.C, launch, st);
  Operand D, h;
  if (s.down) {
    D = operand(ar, s, wd, false, 1, s.C, s.H, launch, st);
    h = {static_cast<u16 *>(ar.take((size_t)R * hp * 2 * (s.split ? 4 : 1))), hp, (long long)R * hp};
  }
  void *rows = s.channel() ? ar.take((size_t)R * out * elem_bytes(s.dtype)) : y;
  if (!launch) return CL3D_OK;
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
  int rc = gemm<GEMM_GATED>(s, a, 1, st);
  if (rc != CL3D_OK) return rc;
  if (s.down) {
    a = gemm_args(s);
    a.P = D.p; a.Q = h.p;
    a.plane_p = D.plane; a.plane_q = h.plane;
    a.ldp = D.ld; a.ldq = hp;
    a.I = s.C; a.J = R; a.K = a.kp = hp;
    a.D = rows; a.ldd = s.C; a.vec = row_vec(s, rows, s.C);
    rc = gemm<GEMM_NT>(s, a, 1, st);
    if (rc != CL3D_OK) return rc;
  }
  return s.channel() ? transposed(s.dtype, rows, s.B, s.N, out, y, st) : CL3D_OK;
}

static int ffn_backward(const FfnShape &s, const void *x, const void *wg, const void *wu, const void *wd, const void *dy, void *dx,
                        void *dwg, void *dwu, void *dwd, unsigned wants, Arena &ar, bool launch, hipStream_t st) {
  const int R = (int)s.R(), hp = (s.H + 7) & ~7, planes = s.split ? 4 : 1;
  const bool want_x = wants & CL3D_FFN_DX, want_gu = wants & CL3D_FFN_DW_IN, want_d = s.down && (wants & CL3D_FFN_DW_DOWN);
  const Operand X = operand(ar, s, x, s.channel(), s.B, s.N, s.C, launch, st);
  const Operand G = operand(ar, s, wg, false, 1, s.H, s.C, launch, st), U = operand(ar, s, wu, false, 1, s.H, s.C, launch, st);
  Operand D, dY, h;
  const void *dh_rows = dy;
  if (s.down) {
    D = operand(ar, s, wd, false, 1, s.C, s.H, launch, st);
    dY = operand(ar, s, dy, s.channel(), s.B, s.N, s.C, launch, st);
    if (want_d) h = {static_cast<u16 *>(ar.take((size_t)R * hp * 2 * planes)), hp, (long long)R * hp};
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
  const int slices_in = weight_slices(s, s.C, s.H, 2), slices_d = weight_slices(s, s.H, s.C, 1);
  float *part_in = want_gu ? static_cast<float *>(ar.take((size_t)2 * slices_in * s.H * s.C * 4)) : nullptr;
  float *part_d = want_d ? static_cast<float *>(ar.take((size_t)slices_d * s.H * s.C * 4)) : nullptr;
  if (!launch) return CL3D_OK;

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
    a.h = const_cast<u16 *>(h.p); a.plane_h = h.plane;
  } else {
    a.dh = dh_rows; a.lddh = s.H;
  }
  a.dgu = dgu; a.plane_dgu = (long long)R * 2 * hp; a.ldh = hp;
  int rc = gemm<GEMM_GATED_BWD>(s, a, 1, st);
  if (rc != CL3D_OK) return rc;
  if (want_x) {
    a = gemm_args(s);
    a.P = G.p; a.Pb = U.p; a.Q = dgu; a.Qb = dgu + hp;
    a.plane_p = G.plane; a.plane_q = (long long)R * 2 * hp;
    a.ldp = G.ld; a.ldq = 2 * hp;
    a.I = s.C; a.J = R; a.K = hp; a.kp = s.H;
    a.D = dx_rows; a.ldd = s.C; a.vec = row_vec(s, dx_rows, s.C);
    rc = gemm<GEMM_NN>(s, a, 1, st);
    if (rc != CL3D_OK) return rc;
    if (s.channel()) rc = transposed(s.dtype, dx_rows, s.B, s.N, s.C, dx, st);
    if (rc != CL3D_OK) return rc;
  }
  if (want_gu) {
    a = gemm_args(s);
    a.P = X.p; a.Q = dgu; a.batch_q = hp;
    a.plane_p = X.plane; a.plane_q = (long long)R * 2 * hp;
    a.ldp = X.ld; a.ldq = 2 * hp;
    a.I = s.C; a.J = s.H; a.K = a.kp = R;
    a.slices = slices_in;
    a.D = part_in; a.vec = s.C % 4 == 0;
    rc = gemm<GEMM_TN>(s, a, 2, st);
    if (rc != CL3D_OK) return rc;
    const long long n = (long long)s.H * s.C;
    if (dwg) slices_sum(s, part_in, n, slices_in, dwg, st);
    if (dwu) slices_sum(s, part_in + n * slices_in, n, slices_in, dwu, st);
  }
  if (want_d) {
    a = gemm_args(s);
    a.P = h.p; a.Q = dY.p;
    a.plane_p = h.plane; a.plane_q = dY.plane;
    a.ldp = hp; a.ldq = dY.ld;
    a.I = s.H; a.J = s.C; a.K = a.kp = R;
    a.slices = slices_d;
    a.D = part_d; a.vec = s.H % 4 == 0;
    rc = gemm<GEMM_TN>(s, a, 1, st);
    if (rc != CL3D_OK) return rc;
    slices_sum(s, part_d, (long long)s.H * s.C, slices_d, dwd, st);
  }
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
  // flags: element type | order << 2 | precision << 3 | down << 4 | backward << 5 | wanted gradients << 6
  FfnShape s;
  if (ffn_shape(s, flags & 3, (flags >> 2) & 1, B, N, C, H, CL3D_ACT_SILU, (flags >> 3) & 1, (flags >> 4) & 1, "gated_ffn") != CL3D_OK)
    return 0;
  Arena ar(nullptr);
  if ((flags >> 5) & 1) ffn_backward(s, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, (unsigned)flags >> 6, ar, false, nullptr);
  else ffn_forward(s, nullptr, nullptr, nullptr, nullptr, nullptr, ar, false, nullptr);
  return ar.used;
}

}  // namespace cl3d

extern "C" int cl3d_gated_ffn_fwd(const void *x, const void *w_gate, const void *w_up, const void *w_down, int dtype, int order, int B,
                                  int C, int N, int H, int activation, int precision, void *y, void *ws, size_t ws_bytes,
                                  cl3d_stream_t stream) {
  using namespace cl3d;
  FfnShape s;
  int rc = ffn_shape(s, dtype, order, B, N, C, H, activation, precision, w_down != nullptr, "gated_ffn_fwd");
  if (rc != CL3D_OK) return rc;
  if (s.R() == 0) return CL3D_OK;
  CL3D_REQUIRE(x && w_gate && w_up && y, "gated_ffn_fwd: null pointer");
  CL3D_REQUIRE(aligned16(x) && aligned16(w_gate) && aligned16(w_up) && aligned16(w_down) && aligned16(y) && aligned16(ws),
               "gated_ffn_fwd: tensors start on 16 bytes");
  Arena need(nullptr), ar(ws);
  ffn_forward(s, x, w_gate, w_up, w_down, y, need, false, nullptr);
  if (ws_bytes < need.used || (need.used && !ws)) return fail(CL3D_E_WORKSPACE, "gated_ffn_fwd: %zu bytes of scratch, %zu needed", ws_bytes, need.used);
  rc = ffn_forward(s, x, w_gate, w_up, w_down, y, ar, true, (hipStream_t)stream);
  return rc != CL3D_OK ? rc : check_launch("cl3d_gated_ffn_fwd");
}

extern "C" int cl3d_gated_ffn_bwd(const void *x, const void *w_gate, const void *w_up, const void *w_down, const void *dy, int dtype,
                                  int order, int B, int C, int N, int H, int activation, int precision, void *dx, void *dw_gate,
                                  void *dw_up, void *dw_down, void *ws, size_t ws_bytes, cl3d_stream_t stream) {
  using namespace cl3d;
  FfnShape s;
  int rc = ffn_shape(s, dtype, order, B, N, C, H, activation, precision, w_down != nullptr, "gated_ffn_bwd");
  if (rc != CL3D_OK) return rc;
  CL3D_REQUIRE(s.R() > 0, "gated_ffn_bwd: no points (their gradients are zeros: nothing to launch)");
  CL3D_REQUIRE(x && w_gate && w_up && dy, "gated_ffn_bwd: null pointer");
  CL3D_REQUIRE(w_down != nullptr || dw_down == nullptr, "gated_ffn_bwd: a gradient for a projection that is not there");
  CL3D_REQUIRE(aligned16(x) && aligned16(w_gate) && aligned16(w_up) && aligned16(w_down) && aligned16(dy) && aligned16(dx) &&
                   aligned16(dw_gate) && aligned16(dw_up) && aligned16(dw_down) && aligned16(ws),
               "gated_ffn_bwd: tensors start on 16 bytes");
  const unsigned wants = (dx ? CL3D_FFN_DX : 0u) | (dw_gate || dw_up ? CL3D_FFN_DW_IN : 0u) | (dw_down ? CL3D_FFN_DW_DOWN : 0u);
  if (wants == 0) return CL3D_OK;
  Arena need(nullptr), ar(ws);
  ffn_backward(s, x, w_gate, w_up, w_down, dy, dx, dw_gate, dw_up, dw_down, wants, need, false, nullptr);
  if (ws_bytes < need.used || (need.used && !ws)) return fail(CL3D_E_WORKSPACE, "gated_ffn_bwd: %zu bytes of scratch, %zu needed", ws_bytes, need.used);
  rc = ffn_backward(s, x, w_gate, w_up, w_down, dy, dx, dw_gate, dw_up, dw_down, wants, ar, true, (hipStream_t)stream);
  return rc != CL3D_OK ? rc : check_launch("cl3d_gated_ffn_bwd");
}
