// ff_common.h -- what the feed-forward operators (gated_ffn.hip, point_norm.hip, dropout.hip) share: element types, the
// activation and its slope, the counter-based generator.
#pragma once
#include "cl3d_common.h"

namespace cl3d {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// element types of the C ABI (CL3D_F32 / CL3D_BF16 / CL3D_F16); arithmetic is f32 everywhere, a 16-bit element is rounded to
// nearest even once, where it is stored
struct F32 {
  using storage = float;
  static constexpr int kVec = 4;  // elements of 16 bytes
  static __device__ __forceinline__ float get(float v) { return v; }
  static __device__ __forceinline__ float put(float v) { return v; }
};
struct Bf16 {
  using storage = unsigned short;
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float get(unsigned short v) { return __uint_as_float((unsigned)v << 16); }
  static __device__ __forceinline__ unsigned short put(float v) { return __builtin_bit_cast(unsigned short, (__bf16)v); }
};
struct F16 {
  using storage = unsigned short;
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float get(unsigned short v) { return (float)__builtin_bit_cast(_Float16, v); }
  static __device__ __forceinline__ unsigned short put(float v) { return __builtin_bit_cast(unsigned short, (_Float16)v); }
};

// 16 bytes of elements
template <typename T> struct Vec16 {
  typename T::storage v[T::kVec];
} __attribute__((aligned(16)));

inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline size_t elem_bytes(int dtype) { return dtype == CL3D_F32 ? 4 : 2; }

// ---- Philox 4x32 with ten rounds (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011): a
// bijection of the 128-bit counter under a 64-bit key.  Block b of a draw is the counter (offset + b, 0); element i of a tensor
// takes word i % 4 of block i / 4, so a mask is a pure function of (seed, offset, element) and is formed again in the backward
// pass instead of being stored.  Twenty 32 x 32 -> 64 bit products and as
// many three-input exclusive ors per four elements.
struct Words {
  unsigned w[4];
};
__device__ __forceinline__ unsigned xor3(unsigned a, unsigned b, unsigned c) { return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96); }
__device__ __forceinline__ Words philox(unsigned long long counter, unsigned long long seed) {
  unsigned c0 = (unsigned)counter, c1 = (unsigned)(counter >> 32), c2 = 0u, c3 = 0u;
  unsigned k0 = (unsigned)seed, k1 = (unsigned)(seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const unsigned long long p0 = (unsigned long long)c0 * 0xD2511F53u, p1 = (unsigned long long)c2 * 0xCD9E8D57u;
    c0 = xor3((unsigned)(p1 >> 32), c1, k0);
    c1 = (unsigned)p1;
    c2 = xor3((unsigned)(p0 >> 32), c3, k1);
    c3 = (unsigned)p0;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return {{c0, c1, c2, c3}};
}

// what a dropout does: an element whose word is at least `threshold` stays and is multiplied by `scale`, the others become 0.
// `state`: two 64-bit numbers in device memory (seed, offset), so that a captured launch reads the values of its replay.
struct Drop {
  const unsigned long long *state;
  unsigned threshold;
  int all;  // p = 1: nothing stays
  float scale;
};
inline int make_drop(Drop &d, const void *state, double p, const char *who) {
  if (!(p >= 0.0 && p <= 1.0)) return fail(CL3D_E_INVALID, "%s: a probability is in [0, 1]", who);
  if (p > 0.0 && state == nullptr) return fail(CL3D_E_INVALID, "%s: dropout needs a generator state", who);
  d.state = static_cast<const unsigned long long *>(state);
  d.all = p >= 1.0;
  d.threshold = d.all ? 0u : (unsigned)(unsigned long long)(p * 4294967296.0);
  d.scale = d.all ? 0.f : (float)(1.0 / (1.0 - p));
  return CL3D_OK;
}

// scratch of a call, handed out in order; without a base it only counts
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

// [b][R][C] -> [b][C][R] of the tensor type
inline int transposed(int dtype, const void *src, int B, int R, int C, void *dst, hipStream_t st) {
  if (dtype == CL3D_F32) return cl3d_transpose(static_cast<const float *>(src), B, R, C, static_cast<float *>(dst), st);
  return cl3d_transpose16(src, B, R, C, dst, st);
}

}  // namespace cl3d
