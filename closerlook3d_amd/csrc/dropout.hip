// dropout.hip -- dropout from a counter: element i of a dense tensor stays when word i of the generator's draw (ff_common.h:
// philox) is at least floor(p 2^32), and is multiplied by 1 / (1 - p).  The mask is never stored: the gradient is the same
// kernel on the incoming gradient with the same (seed, offset).
// One pass, 16 bytes a lane; floor: one read and one write of the tensor.  Per four elements the generator costs 20 32 x 32 -> 64
// bit products (a quarter of the f32 rate each) and 20 exclusive ors.  Measured: 9.4 M bf16 elements in 9.7 us, 3.9 TB/s.
#include "ff_common.h"

namespace cl3d {

template <typename T, bool VEC>
__global__ __launch_bounds__(256) void dropout_kernel(const typename T::storage *__restrict__ x, long long n, Drop d,
                                                      typename T::storage *__restrict__ out) {
  const unsigned long long seed = d.state[0], offset = d.state[1];
  constexpr int V = VEC ? T::kVec : 4;
  const long long pieces = (n + V - 1) / V, stride = (long long)gridDim.x * 256;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < pieces; i += stride) {
    const long long e0 = i * V;
    Vec16<T> v;
    const bool whole = VEC && e0 + V <= n;
    if (whole) v = reinterpret_cast<const Vec16<T> *>(x)[i];
#pragma unroll
    for (int q = 0; q < V / 4; ++q) {
      const Words w = philox(offset + (unsigned long long)(i * (V / 4) + q), seed);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const long long at = e0 + 4 * q + e;
        const bool stays = !d.all && w.w[e] >= d.threshold;
        if (whole) v.v[4 * q + e] = T::put(stays ? T::get(v.v[4 * q + e]) * d.scale : 0.f);
        else if (at < n) out[at] = T::put(stays ? T::get(x[at]) * d.scale : 0.f);
      }
    }
    if (whole) reinterpret_cast<Vec16<T> *>(out)[i] = v;
  }
}

// Point-major features: element (b, c, n) is number (b C + c) N + n of the draw, as where they lie channel-major, and lies at
// (b N + n) C + c.  A lane takes one block of the draw, the up to four points of its channel that the block numbers, so that each block
// is formed once (twice where a channel ends inside it); lanes side by side have channels side by side, which lie together.  A
// workgroup has `per` blocks of every channel of a cloud.  Bound: the generator and single-element loads.  Measured: 16 x 144 x 4096
// bf16 18.5 us, f32 16.7; by a strided copy into the other order 50 and 53, and the result lay that way.
template <typename T>
__global__ __launch_bounds__(256) void dropout_points_kernel(const typename T::storage *__restrict__ x, int B, int C, int N, int per, Drop d,
                                                             typename T::storage *__restrict__ out) {
  const unsigned long long seed = d.state[0], offset = d.state[1];
  const long long blocks = ((long long)N + 6) / 4;  // of a channel, at most
  for (int b = blockIdx.y; b < B; b += gridDim.y)
    for (long long k0 = (long long)blockIdx.x * per; k0 < blocks; k0 += (long long)gridDim.x * per)
      for (unsigned e = threadIdx.x; e < (unsigned)per * (unsigned)C; e += 256) {
        const unsigned k = e / (unsigned)C, c = e - k * (unsigned)C;
        const long long first = ((long long)b * C + c) * N;
        const long long n0 = 4 * (k0 + k) - (first & 3);  // of the block's first number
        if (n0 >= N) continue;
        const Words w = philox(offset + (unsigned long long)((first + n0) >> 2), seed);
        const long long at = ((long long)b * N + n0) * C + c;
        typename T::storage v[4];
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (n0 + q >= 0 && n0 + q < N) v[q] = x[at + (long long)q * C];
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (n0 + q >= 0 && n0 + q < N) out[at + (long long)q * C] = T::put(!d.all && w.w[q] >= d.threshold ? T::get(v[q]) * d.scale : 0.f);
      }
}

__global__ void rng_take_kernel(unsigned long long *state, unsigned long long blocks, unsigned long long *out) {
  out[0] = state[0];
  out[1] = atomicAdd(&state[1], blocks);  // two streams that draw at once get different counters
}

template <typename T> static void dropout_launch(const void *x, long long n, const Drop &d, void *out, hipStream_t st) {
  using S = typename T::storage;
  const bool vec = aligned16(x) && aligned16(out);
  const long long pieces = vec ? (n + T::kVec - 1) / T::kVec : (n + 3) / 4;
  const long long grid = pieces < 256ll * 4096 ? (pieces + 255) / 256 : 4096;
  if (vec)
    hipLaunchKernelGGL((dropout_kernel<T, true>), dim3((unsigned)grid), dim3(256), 0, st, static_cast<const S *>(x), n, d, static_cast<S *>(out));
  else
    hipLaunchKernelGGL((dropout_kernel<T, false>), dim3((unsigned)grid), dim3(256), 0, st, static_cast<const S *>(x), n, d, static_cast<S *>(out));
}

template <typename T> static void dropout_points_launch(const void *x, int B, int C, int N, const Drop &d, void *out, hipStream_t st) {
  using S = typename T::storage;
  const int per = C < 1024 ? ceil_div(1024, C) : 1;
  const long long tiles = (((long long)N + 6) / 4 + per - 1) / per;
  const dim3 grid((unsigned)(tiles < 16384 ? tiles : 16384), (unsigned)(B < 512 ? B : 512));
  hipLaunchKernelGGL(dropout_points_kernel<T>, grid, dim3(256), 0, st, static_cast<const S *>(x), B, C, N, per, d, static_cast<S *>(out));
}

}  // namespace cl3d

extern "C" int cl3d_dropout(const void *x, int dtype, long long n, double p, const int64_t *rng, void *out, cl3d_stream_t stream) {
  using namespace cl3d;
  CL3D_REQUIRE(dtype == CL3D_F32 || dtype == CL3D_BF16 || dtype == CL3D_F16, "dropout: unknown element type %d", dtype);
  CL3D_REQUIRE(n >= 0, "dropout: bad size");
  Drop d;
  const int rc = make_drop(d, rng, p, "dropout");
  if (rc != CL3D_OK) return rc;
  if (n == 0) return CL3D_OK;
  CL3D_REQUIRE(x && out && rng, "dropout: null pointer");
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == CL3D_F32) dropout_launch<F32>(x, n, d, out, st);
  else if (dtype == CL3D_BF16) dropout_launch<Bf16>(x, n, d, out, st);
  else dropout_launch<F16>(x, n, d, out, st);
  return check_launch("cl3d_dropout");
}

extern "C" int cl3d_dropout_point_major(const void *x, int dtype, int B, int C, int N, double p, const int64_t *rng, void *out,
                                        cl3d_stream_t stream) {
  using namespace cl3d;
  CL3D_REQUIRE(dtype == CL3D_F32 || dtype == CL3D_BF16 || dtype == CL3D_F16, "dropout_point_major: unknown element type %d", dtype);
  CL3D_REQUIRE(B >= 0 && C >= 0 && N >= 0, "dropout_point_major: bad size");
  Drop d;
  const int rc = make_drop(d, rng, p, "dropout_point_major");
  if (rc != CL3D_OK) return rc;
  if (B == 0 || C == 0 || N == 0) return CL3D_OK;
  CL3D_REQUIRE(x && out && rng, "dropout_point_major: null pointer");
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == CL3D_F32) dropout_points_launch<F32>(x, B, C, N, d, out, st);
  else if (dtype == CL3D_BF16) dropout_points_launch<Bf16>(x, B, C, N, d, out, st);
  else dropout_points_launch<F16>(x, B, C, N, d, out, st);
  return check_launch("cl3d_dropout_point_major");
}

extern "C" int cl3d_rng_take(int64_t *state, long long blocks, int64_t *out, cl3d_stream_t stream) {
  using namespace cl3d;
  CL3D_REQUIRE(blocks >= 0, "rng_take: bad size");
  CL3D_REQUIRE(state && out && state != out, "rng_take: null pointer, or a draw into the state itself");
  hipLaunchKernelGGL(rng_take_kernel, dim3(1), dim3(1), 0, (hipStream_t)stream, reinterpret_cast<unsigned long long *>(state),
                     (unsigned long long)blocks, reinterpret_cast<unsigned long long *>(out));
  return check_launch("cl3d_rng_take");
}
