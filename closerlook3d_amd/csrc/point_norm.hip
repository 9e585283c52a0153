// point_norm.hip -- the norms either side of a block, fused with its gate, its dropout and the residual, over the C channels of a
// point (rows [R, C], R = clouds x points):
//     n = norm(y) w + b          norm 0 none, 1 rms: y / sqrt(mean y^2 + eps), 2 layer: (y - mean) / sqrt(var + eps)
//     o = alpha x + gate * drop(n)                      (exit of a block; gate per channel, or per cloud and channel)
//     h = norm(o) w2 + b2                               (entry of the next; alone: h = norm(x) w2 + b2)
// Each direction is one pass over the rows: a row lives in the registers of TPR lanes from the load to the store (statistics in
// two steps over the registers, f32, so a mean far from zero costs no digits), parameters in registers across the rows of a
// workgroup.  Bound: memory -- forward x, y in and o, h out; backward do, dh, x, y in and dx, dy out, a mean and a reciprocal
// deviation per row kept from the forward pass.  Measured in bf16: 65 536 x 144, exit and entry, 20 us (3.8 TB/s); with dropout the
// generator is half of the vector instructions: 81 920 x 288 forward 73 us (2.6 TB/s), backward 125 (2.3 TB/s).
// Parameter gradients are sums over the rows: a workgroup keeps its rows' sums in registers, f32, one partial row per workgroup
// goes to scratch and a second launch adds them in order (no atomics: bit-identical run to run).  A workgroup's rows are of one
// cloud, so a gate per cloud is summed by the same partials.
#include "ff_common.h"
#include <type_traits>

namespace cl3d {

struct NormArgs {
  const void *x, *y;                  // x: the residual stream (or the one input)
  const void *w1, *b1, *gate, *w2, *b2;
  const void *dout, *dnext;
  void *o, *h, *dx, *dy;
  float *stats;                       // [R][4]: mean, 1 / deviation of y; the same of o
  float *partial;                     // [workgroup][5][C]: w, b, gate, w2, b2
  long long N;                        // rows of a cloud
  int B, C, chunks, per;              // workgroups and rows of one for each cloud
  int kind1, kind2, exit, next, gate_cloud, param_f32;
  float alpha, eps1, eps2;
  Drop drop;
  int has_drop;
};

// V parameters from number i on, `none` where there are none; a workgroup loads them once
template <typename T, int V> __device__ __forceinline__ void params(const void *p, long long i, int f32, float none, float *v) {
  if (p == nullptr) {
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = none;
  } else if (V == 1) {
    v[0] = f32 ? static_cast<const float *>(p)[i] : T::get(static_cast<const typename T::storage *>(p)[i]);
  } else if (f32) {
#pragma unroll
    for (int q = 0; q < V / 4; ++q) {
      const f32x4 t = *reinterpret_cast<const f32x4 *>(static_cast<const float *>(p) + i + 4 * q);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[4 * q + e] = t[e];
    }
  } else {
    const auto t = *reinterpret_cast<const Vec16<T> *>(static_cast<const typename T::storage *>(p) + i);
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = T::get(t.v[e % T::kVec]);
  }
}

// v + v of the lane that the DPP control names (within 16 lanes)
template <int CTRL> __device__ __forceinline__ float add_dpp(float v) {
  return v + __uint_as_float((unsigned)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), CTRL, 0xf, 0xf, true));
}
// the sum over 16, 32 or 64 lanes, in every one of them: neighbour, pair, half row and row by DPP, rows and halves of the wave by the
// swaps of gfx950 (a shuffle through LDS costs a round trip a step, and a row takes up to eight sums)
template <int LANES> __device__ __forceinline__ float lane_sum(float v) {
  v = add_dpp<0xB1>(v);   // quad_perm [1, 0, 3, 2]
  v = add_dpp<0x4E>(v);   // quad_perm [2, 3, 0, 1]
  v = add_dpp<0x141>(v);  // row_half_mirror
  v = add_dpp<0x140>(v);  // row_mirror
  if (LANES > 16) {
    auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    if (LANES > 32) {
      s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
      v = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    }
  }
  return v;
}

// sums of two values over the TPR lanes of a row
template <int TPR> __device__ __forceinline__ void row_sum(float &a, float &b, float *s_red) {
  a = lane_sum<(TPR < 64 ? TPR : 64)>(a);
  b = lane_sum<(TPR < 64 ? TPR : 64)>(b);
  if (TPR > 64) {  // the whole workgroup is one row
    const int wave = threadIdx.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) { s_red[2 * wave] = a; s_red[2 * wave + 1] = b; }
    __syncthreads();
    a = b = 0.f;
#pragma unroll
    for (int w = 0; w < TPR / 64; ++w) { a += s_red[2 * w]; b += s_red[2 * w + 1]; }
  }
}

// V consecutive elements to p (16 bytes, or one)
template <typename T, int V> __device__ __forceinline__ void store_v(void *base, long long at, const float *v) {
  auto *p = static_cast<typename T::storage *>(base) + at;
  if constexpr (V == 1) {
    *p = T::put(v[0]);
  } else {
    Vec16<T> q;
#pragma unroll
    for (int e = 0; e < V; ++e) q.v[e] = T::put(v[e]);
    *reinterpret_cast<Vec16<T> *>(p) = q;
  }
}

// V consecutive elements on their way, and their values
template <typename T, int V> struct Raw {
  typename std::conditional<V == 1, typename T::storage, Vec16<T>>::type v;
  __device__ __forceinline__ void load(const void *base, long long at) {
    v = *reinterpret_cast<const decltype(v) *>(static_cast<const typename T::storage *>(base) + at);
  }
  __device__ __forceinline__ void get(float *f) const {
    if constexpr (V == 1) {
      f[0] = T::get(v);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) f[e] = T::get(v.v[e]);
    }
  }
};

// which of the V elements from `at` on stay (V > 1: at is a multiple of 4)
template <int V> __device__ __forceinline__ void stay_v(const Drop &d, unsigned long long seed, unsigned long long offset, long long at, bool *m) {
  if constexpr (V == 1) {
    const Words w = philox(offset + (unsigned long long)(at >> 2), seed);
    const int e = (int)(at & 3);
    const unsigned word = e < 2 ? (e ? w.w[1] : w.w[0]) : (e == 2 ? w.w[2] : w.w[3]);
    m[0] = !d.all && word >= d.threshold;
  } else {
#pragma unroll
    for (int q = 0; q < V / 4; ++q) {
      const Words w = philox(offset + (unsigned long long)((at >> 2) + q), seed);
#pragma unroll
      for (int e = 0; e < 4; ++e) m[4 * q + e] = !d.all && w.w[e] >= d.threshold;
    }
  }
}

// mean and reciprocal deviation of a row held as v[NV][V]; `on`: which pieces exist (the others hold zeros)
template <int TPR, int NV, int V>
__device__ __forceinline__ void row_stats(const float (&v)[NV][V], const bool (&on)[NV], int kind, float eps, float inv_c, float *s_red,
                                          float &mean, float &rinv) {
  mean = 0.f;
  if (kind == CL3D_NORM_LAYER) {
    float a = 0.f, none = 0.f;
#pragma unroll
    for (int q = 0; q < NV; ++q)
#pragma unroll
      for (int e = 0; e < V; ++e) a += v[q][e];
    row_sum<TPR>(a, none, s_red);
    mean = a * inv_c;
  }
  float a = 0.f, none = 0.f;
#pragma unroll
  for (int q = 0; q < NV; ++q) {
    float t = 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) t = __builtin_fmaf(v[q][e] - mean, v[q][e] - mean, t);
    a += on[q] ? t : 0.f;
  }
  row_sum<TPR>(a, none, s_red);
  rinv = 1.f / sqrtf(a * inv_c + eps);
}

template <typename T, int TPR, int NV, int V, bool DROP>
__global__ __launch_bounds__(256) void norm_fwd_kernel(NormArgs a) {
  __shared__ float s_red[8];
  const int lane = threadIdx.x % TPR, group = threadIdx.x / TPR;
  const int b = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
  const long long first = (long long)b * a.N + (long long)chunk * a.per;
  long long last = first + a.per, end = (long long)(b + 1) * a.N;
  if (last > end) last = end;
  const float inv_c = 1.f / (float)a.C;
  bool on[NV];
  int col[NV];
  float w1[NV][V], b1[NV][V], gate[NV][V], w2[NV][V], b2[NV][V];
#pragma unroll
  for (int q = 0; q < NV; ++q) {
    col[q] = (q * TPR + lane) * V;
    on[q] = col[q] < a.C;
    const int c = on[q] ? col[q] : 0;
    params<T, V>(a.w1, c, a.param_f32, 1.f, w1[q]);
    params<T, V>(a.b1, c, a.param_f32, 0.f, b1[q]);
    params<T, V>(a.gate, (a.gate_cloud ? (long long)b * a.C : 0) + c, a.param_f32, 1.f, gate[q]);
    params<T, V>(a.w2, c, a.param_f32, 1.f, w2[q]);
    params<T, V>(a.b2, c, a.param_f32, 0.f, b2[q]);
  }
  unsigned long long seed = 0, offset = 0;
  if (DROP) { seed = a.drop.state[0]; offset = a.drop.state[1]; }
  // every lane walks the same number of rows (row_sum's barriers): a group behind the last row works on the last one, unstored.
  // The next rows are on their way while these are worked on: a wave's time is the latency of its row, and few rows fit a CU
  constexpr int kStep = 256 / TPR;
  Raw<T, V> nx[NV], ny[NV];
  auto fetch = [&](long long r) {
    r = r < last ? r : last - 1;
#pragma unroll
    for (int q = 0; q < NV; ++q)
      if (on[q]) {
        nx[q].load(a.x, r * a.C + col[q]);
        if (a.exit) ny[q].load(a.y, r * a.C + col[q]);
      }
  };
  fetch(first + group);
  for (long long r0 = first; r0 < last; r0 += kStep) {
    const bool live = r0 + group < last;
    const long long r = live ? r0 + group : last - 1;
    // (a lane without a piece works on zeros: the arithmetic below runs in all lanes, the memory does not)
    float v[NV][V], y[NV][V];
#pragma unroll
    for (int q = 0; q < NV; ++q) {
      if (on[q]) {
        nx[q].get(v[q]);
        if (a.exit) ny[q].get(y[q]);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) v[q][e] = y[q][e] = 0.f;
      }
    }
    if (r0 + kStep < last) fetch(r0 + kStep + group);
    if (a.exit) {
      float mean = 0.f, rinv = 1.f;
      if (a.kind1 != CL3D_NORM_NONE) row_stats<TPR, NV, V>(y, on, a.kind1, a.eps1, inv_c, s_red, mean, rinv);
      if (a.stats && live && lane == 0) *reinterpret_cast<float2 *>(a.stats + 4 * r) = make_float2(mean, rinv);
#pragma unroll
      for (int q = 0; q < NV; ++q) {
        bool m[V];
        if (DROP) stay_v<V>(a.drop, seed, offset, r * a.C + col[q], m);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          float n = __builtin_fmaf((y[q][e] - mean) * rinv, w1[q][e], b1[q][e]);
          if (DROP) n = m[e] ? n * a.drop.scale : 0.f;
          v[q][e] = __builtin_fmaf(a.alpha, v[q][e], gate[q][e] * n);
        }
        if (live && on[q]) store_v<T, V>(a.o, r * a.C + col[q], v[q]);
        if (!on[q]) {
#pragma unroll
          for (int e = 0; e < V; ++e) v[q][e] = 0.f;
        }
      }
    }
    if (a.next) {
      float mean = 0.f, rinv = 1.f;
      row_stats<TPR, NV, V>(v, on, a.kind2, a.eps2, inv_c, s_red, mean, rinv);
      if (a.stats && live && lane == 0) *reinterpret_cast<float2 *>(a.stats + 4 * r + 2) = make_float2(mean, rinv);
#pragma unroll
      for (int q = 0; q < NV; ++q) {
#pragma unroll
        for (int e = 0; e < V; ++e) v[q][e] = __builtin_fmaf((v[q][e] - mean) * rinv, w2[q][e], b2[q][e]);
        if (live && on[q]) store_v<T, V>(a.h, r * a.C + col[q], v[q]);
      }
    }
  }
}

// d of norm: dhat -> d = rinv (dhat - hat mean(dhat hat) - [layer] mean(dhat))
template <typename T, int TPR, int NV, int V, bool DROP, bool BIAS>
__global__ __launch_bounds__(256) void norm_bwd_kernel(NormArgs a) {
  __shared__ float s_red[8];
  __shared__ float s_sum[TPR < 256 ? 256 / TPR : 1][TPR < 256 ? TPR * NV * V : 1];
  const int lane = threadIdx.x % TPR, group = threadIdx.x / TPR;
  const int b = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
  const long long first = (long long)b * a.N + (long long)chunk * a.per;
  long long last = first + a.per, end = (long long)(b + 1) * a.N;
  if (last > end) last = end;
  const float inv_c = 1.f / (float)a.C;
  bool on[NV];
  int col[NV];
  float w1[NV][V], b1[NV][V], gate[NV][V], w2[NV][V];
  float s_w1[NV][V], s_b1[NV][V], s_gate[NV][V], s_w2[NV][V], s_b2[NV][V];
#pragma unroll
  for (int q = 0; q < NV; ++q) {
    col[q] = (q * TPR + lane) * V;
    on[q] = col[q] < a.C;
    const int c = on[q] ? col[q] : 0;
    params<T, V>(a.w1, c, a.param_f32, 1.f, w1[q]);
    params<T, V>(BIAS ? a.b1 : nullptr, c, a.param_f32, 0.f, b1[q]);
    params<T, V>(a.gate, (a.gate_cloud ? (long long)b * a.C : 0) + c, a.param_f32, 1.f, gate[q]);
    params<T, V>(a.w2, c, a.param_f32, 1.f, w2[q]);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      s_w1[q][e] = s_b1[q][e] = s_gate[q][e] = s_w2[q][e] = s_b2[q][e] = 0.f;
    }
  }
  unsigned long long seed = 0, offset = 0;
  if (DROP) { seed = a.drop.state[0]; offset = a.drop.state[1]; }
  constexpr int kStep = 256 / TPR;
  Raw<T, V> nx[NV], ny[NV], nd[NV], nh[NV];
  f32x4 ns;
  auto fetch = [&](long long r) {  // (as in the forward kernel)
    r = r < last ? r : last - 1;
    ns = *reinterpret_cast<const f32x4 *>(a.stats + 4 * r);
#pragma unroll
    for (int q = 0; q < NV; ++q)
      if (on[q]) {
        if (a.exit) ny[q].load(a.y, r * a.C + col[q]);
        if (a.dout) nd[q].load(a.dout, r * a.C + col[q]);
        if (a.dnext) {
          nx[q].load(a.x, r * a.C + col[q]);
          nh[q].load(a.dnext, r * a.C + col[q]);
        }
      }
  };
  fetch(first + group);
  for (long long r0 = first; r0 < last; r0 += kStep) {
    const bool live = r0 + group < last;
    const long long r = live ? r0 + group : last - 1;
    const f32x4 st = ns;
    // a lane without a piece works on zeros, a group behind the last row on zero gradients: only memory is guarded below
    float hat1[NV][V], d[NV][V], hat[NV][V], dh[NV][V];
#pragma unroll
    for (int q = 0; q < NV; ++q) {
#pragma unroll
      for (int e = 0; e < V; ++e) hat1[q][e] = d[q][e] = hat[q][e] = dh[q][e] = 0.f;
      if (on[q]) {
        if (a.exit) ny[q].get(hat1[q]);
        if (a.dnext) nx[q].get(hat[q]);
        if (live) {
          if (a.dout) nd[q].get(d[q]);
          if (a.dnext) nh[q].get(dh[q]);
        }
      }
    }
    if (r0 + kStep < last) fetch(r0 + kStep + group);
    // the exit once more, from x and y: out as the forward pass had it before it was rounded costs no more traffic than the
    // rounded one, and the y hats are needed below anyway.  nk: what was left of the norm of y
    bool stays[NV][V];
    float nk[NV][V];
    if (a.exit) {
#pragma unroll
      for (int q = 0; q < NV; ++q) {
        if (DROP) stay_v<V>(a.drop, seed, offset, r * a.C + col[q], stays[q]);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          hat1[q][e] = (hat1[q][e] - st[0]) * st[1];
          nk[q][e] = __builtin_fmaf(hat1[q][e], w1[q][e], b1[q][e]);
          if (DROP) nk[q][e] = stays[q][e] ? nk[q][e] * a.drop.scale : 0.f;
          if (!live) hat1[q][e] = nk[q][e] = 0.f;  // (its gradients are zeros, but 0 x inf is a NaN)
        }
      }
    }
    if (a.dnext) {
      float p1 = 0.f, p2 = 0.f;
#pragma unroll
      for (int q = 0; q < NV; ++q) {
        float t1 = 0.f, t2 = 0.f;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          if (a.exit) hat[q][e] = __builtin_fmaf(a.alpha, hat[q][e], gate[q][e] * nk[q][e]);
          hat[q][e] = live ? (hat[q][e] - st[2]) * st[3] : 0.f;
          s_w2[q][e] = __builtin_fmaf(dh[q][e], hat[q][e], s_w2[q][e]);
          if (BIAS) s_b2[q][e] += dh[q][e];
          dh[q][e] *= w2[q][e];
          t1 = __builtin_fmaf(dh[q][e], hat[q][e], t1);
          t2 += dh[q][e];
        }
        p1 += on[q] ? t1 : 0.f;
        p2 += on[q] ? t2 : 0.f;
      }
      row_sum<TPR>(p1, p2, s_red);
      p1 *= inv_c;
      p2 = a.kind2 == CL3D_NORM_LAYER ? p2 * inv_c : 0.f;
#pragma unroll
      for (int q = 0; q < NV; ++q)
#pragma unroll
        for (int e = 0; e < V; ++e) d[q][e] = __builtin_fmaf(st[3], dh[q][e] - __builtin_fmaf(hat[q][e], p1, p2), d[q][e]);
    }
    if (a.dx && live) {
#pragma unroll
      for (int q = 0; q < NV; ++q) {
        if (!on[q]) continue;
        float o[V];
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = a.exit ? a.alpha * d[q][e] : d[q][e];
        store_v<T, V>(a.dx, r * a.C + col[q], o);
      }
    }
    if (a.exit) {
      float p1 = 0.f, p2 = 0.f;
#pragma unroll
      for (int q = 0; q < NV; ++q) {
        float t1 = 0.f, t2 = 0.f;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          float dm = live ? d[q][e] : 0.f;
          s_gate[q][e] = __builtin_fmaf(dm, nk[q][e], s_gate[q][e]);
          if (DROP) dm = stays[q][e] ? dm * a.drop.scale : 0.f;
          dm *= gate[q][e];
          s_w1[q][e] = __builtin_fmaf(dm, DROP && !stays[q][e] ? 0.f : hat1[q][e], s_w1[q][e]);  // (dropped: nothing, whatever y is)
          if (BIAS) s_b1[q][e] += dm;
          dm *= w1[q][e];
          t1 = __builtin_fmaf(dm, hat1[q][e], t1);
          t2 += dm;
          d[q][e] = dm;
        }
        p1 += on[q] ? t1 : 0.f;
        p2 += on[q] ? t2 : 0.f;
      }
      if (a.dy) {
        if (a.kind1 != CL3D_NORM_NONE) {
          row_sum<TPR>(p1, p2, s_red);
          p1 *= inv_c;
          p2 = a.kind1 == CL3D_NORM_LAYER ? p2 * inv_c : 0.f;
        } else {  // (y does not enter its own gradient, whatever it is)
          p1 = p2 = 0.f;
#pragma unroll
          for (int q = 0; q < NV; ++q)
#pragma unroll
            for (int e = 0; e < V; ++e) hat1[q][e] = 0.f;
        }
        if (live)
#pragma unroll
          for (int q = 0; q < NV; ++q) {
            if (!on[q]) continue;
            float o[V];
#pragma unroll
            for (int e = 0; e < V; ++e) o[e] = st[1] * (d[q][e] - __builtin_fmaf(hat1[q][e], p1, p2));
            store_v<T, V>(a.dy, r * a.C + col[q], o);
          }
      }
    }
  }
  if (!a.partial) return;
  // the groups' sums of a column, in group order
  auto flush = [&](const float (&s)[NV][V], int which) {
    float *dst = a.partial + ((long long)blockIdx.x * 5 + which) * a.C;
    if constexpr (TPR == 256) {
#pragma unroll
      for (int q = 0; q < NV; ++q)
        if (on[q])
#pragma unroll
          for (int e = 0; e < V; ++e) dst[col[q] + e] = s[q][e];
    } else {
      __syncthreads();
#pragma unroll
      for (int q = 0; q < NV; ++q)
#pragma unroll
        for (int e = 0; e < V; ++e) s_sum[group][(q * TPR + lane) * V + e] = s[q][e];
      __syncthreads();
      for (int c = threadIdx.x; c < a.C; c += 256) {
        float t = 0.f;
#pragma unroll
        for (int g = 0; g < 256 / TPR; ++g) t += s_sum[g][c];
        dst[c] = t;
      }
    }
  };
  if (a.exit) {
    if (a.w1) flush(s_w1, 0);
    if (BIAS && a.b1) flush(s_b1, 1);
    if (a.gate) flush(s_gate, 2);
  }
  if (a.w2) flush(s_w2, 3);
  if (BIAS && a.b2) flush(s_b2, 4);
}

// ---- channel-major features [B][C][N] of up to 1024 channels, a multiple of 4: no transposed copies.  A workgroup has P = 64, 32 or
// 16 points of a cloud, a lane one of them; the 64 / P lane groups of its W waves have the channels 4 (g + G i) .. + 3, i < QN, of
// G = W 64 / P (fours: one block of the generator).  A channel is read and written P elements in a row, the values stay in registers,
// sums over channels go through LDS: a buffer for each, so that a barrier each is enough.  Parameter gradients: P points by
// lane_sum, one partial row per workgroup.
// Measured: 16 x 144 x 4096 bf16, exit and next norm, 19 us (4.0 TB/s; by transposed copies 91), with the gradients 75 (250); 4 x 72 x
// 10 000 f32, exit with dropout and its gradients 29 (72).
constexpr int kCmMaxC = 1024, kCmWaves = 16;

// LDS of a workgroup: four buffers of a float per lane, then w, b, gate, w2, b2 [C] each
static size_t cm_lds_bytes(int waves, int C) { return (4 * 64 * (size_t)waves + 5 * (size_t)C) * sizeof(float); }
template <typename T> __device__ __forceinline__ void cm_params(const NormArgs &a, int b, float *par) {
  for (int c = threadIdx.x; c < a.C; c += blockDim.x) {
    params<T, 1>(a.w1, c, a.param_f32, 1.f, par + c);
    params<T, 1>(a.b1, c, a.param_f32, 0.f, par + a.C + c);
    params<T, 1>(a.gate, (a.gate_cloud ? (long long)b * a.C : 0) + c, a.param_f32, 1.f, par + 2 * a.C + c);
    params<T, 1>(a.w2, c, a.param_f32, 1.f, par + 3 * a.C + c);
    params<T, 1>(a.b2, c, a.param_f32, 0.f, par + 4 * a.C + c);
  }
}

// a point's elements of QN quads of channels; what a lane does not have is 0
template <typename S, int QN>
__device__ __forceinline__ void cm_fetch(const void *p, bool wanted, const long long (&at)[QN], const bool (&on)[QN], long long N, S (&raw)[QN][4]) {
#pragma unroll
  for (int q = 0; q < QN; ++q)
#pragma unroll
    for (int e = 0; e < 4; ++e) raw[q][e] = 0;
  if (!wanted) return;
#pragma unroll
  for (int q = 0; q < QN; ++q)
    if (on[q]) {
#pragma unroll
      for (int e = 0; e < 4; ++e) raw[q][e] = static_cast<const S *>(p)[at[q] + e * N];
    }
}

// the lane groups' values of a point, added in one order
template <int P> __device__ __forceinline__ float wave_sum(float v, float *s, int wave, int lane, int waves) {
  if (P < 32) {
    const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(p[0]) + __uint_as_float(p[1]);
  }
  if (P < 64) {
    const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(p[0]) + __uint_as_float(p[1]);
  }
  s[wave * 64 + lane] = v;
  __syncthreads();
  float t = 0.f;
  for (int w = 0; w < waves; ++w) t += s[w * 64 + lane];
  return t;
}
// mean and reciprocal deviation of a point held as v[QN][4] by the lane groups of a workgroup
template <int P, int QN>
__device__ __forceinline__ void cm_stats(const float (&v)[QN][4], const bool (&on)[QN], int kind, float eps, float inv_c, float *s0, float *s1,
                                         int wave, int lane, int waves, float &mean, float &rinv) {
  mean = 0.f;
  float t = 0.f;
  if (kind == CL3D_NORM_LAYER) {
#pragma unroll
    for (int q = 0; q < QN; ++q)
#pragma unroll
      for (int e = 0; e < 4; ++e) t += on[q] ? v[q][e] : 0.f;
    mean = wave_sum<P>(t, s0, wave, lane, waves) * inv_c;
  }
  t = 0.f;
#pragma unroll
  for (int q = 0; q < QN; ++q)
#pragma unroll
    for (int e = 0; e < 4; ++e) t = on[q] ? __builtin_fmaf(v[q][e] - mean, v[q][e] - mean, t) : t;
  rinv = 1.f / sqrtf(wave_sum<P>(t, s1, wave, lane, waves) * inv_c + eps);
}

template <typename T, int P, int QN, bool DROP>
__global__ __launch_bounds__(64 * kCmWaves) void norm_cm_fwd_kernel(NormArgs a) {
  using S = typename T::storage;
  extern __shared__ float s_cm[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, waves = blockDim.x >> 6;
  const int group = wave * (64 / P) + lane / P, groups = waves * (64 / P);
  float *s[4], *par[5];
#pragma unroll
  for (int k = 0; k < 4; ++k) s[k] = s_cm + k * 64 * waves;
#pragma unroll
  for (int k = 0; k < 5; ++k) par[k] = s_cm + 4 * 64 * waves + k * a.C;
  const int b = blockIdx.x / a.chunks, tile = blockIdx.x % a.chunks;
  const long long n0 = (long long)tile * P + lane % P;
  const bool live = n0 < a.N;
  const long long n = live ? n0 : a.N - 1, r = (long long)b * a.N + n;  // (a lane behind the last point works on it, unstored)
  const float inv_c = 1.f / (float)a.C;
  bool on[QN];
  int c0[QN];
  long long at[QN];
  S rx[QN][4], ry[QN][4];
  float v[QN][4], y[QN][4];
#pragma unroll
  for (int q = 0; q < QN; ++q) {
    c0[q] = 4 * (group + groups * q);
    on[q] = c0[q] < a.C;
    at[q] = ((long long)b * a.C + c0[q]) * a.N + n;
  }
  cm_fetch<S, QN>(a.x, true, at, on, a.N, rx);
  cm_fetch<S, QN>(a.y, a.exit, at, on, a.N, ry);
  cm_params<T>(a, b, par[0]);
  __syncthreads();
#pragma unroll
  for (int q = 0; q < QN; ++q)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[q][e] = T::get(rx[q][e]);
      y[q][e] = T::get(ry[q][e]);
    }
  if (a.exit) {
    float mean = 0.f, rinv = 1.f;
    if (a.kind1 != CL3D_NORM_NONE) cm_stats<P, QN>(y, on, a.kind1, a.eps1, inv_c, s[0], s[1], wave, lane, waves, mean, rinv);
    if (a.stats && live && group == 0) *reinterpret_cast<float2 *>(a.stats + 4 * r) = make_float2(mean, rinv);
    unsigned long long seed = 0, offset = 0;
    if (DROP) { seed = a.drop.state[0]; offset = a.drop.state[1]; }
#pragma unroll
    for (int q = 0; q < QN; ++q) {
      if (!on[q]) continue;
      bool m[4];
      if (DROP) stay_v<4>(a.drop, seed, offset, r * a.C + c0[q], m);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float k = __builtin_fmaf((y[q][e] - mean) * rinv, par[0][c0[q] + e], par[1][c0[q] + e]);
        if (DROP) k = m[e] ? k * a.drop.scale : 0.f;
        v[q][e] = __builtin_fmaf(a.alpha, v[q][e], par[2][c0[q] + e] * k);
        if (live) static_cast<S *>(a.o)[at[q] + e * a.N] = T::put(v[q][e]);
      }
    }
  }
  if (a.next) {
    float mean, rinv;
    cm_stats<P, QN>(v, on, a.kind2, a.eps2, inv_c, s[2], s[3], wave, lane, waves, mean, rinv);
    if (a.stats && live && group == 0) *reinterpret_cast<float2 *>(a.stats + 4 * r + 2) = make_float2(mean, rinv);
#pragma unroll
    for (int q = 0; q < QN; ++q) {
      if (!on[q] || !live) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        static_cast<S *>(a.h)[at[q] + e * a.N] =
            T::put(__builtin_fmaf((v[q][e] - mean) * rinv, par[3][c0[q] + e], par[4][c0[q] + e]));
    }
  }
}

template <typename T, int P, int QN, bool DROP>
__global__ __launch_bounds__(64 * kCmWaves) void norm_cm_bwd_kernel(NormArgs a) {
  using S = typename T::storage;
  extern __shared__ float s_cm[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, waves = blockDim.x >> 6;
  const int group = wave * (64 / P) + lane / P, groups = waves * (64 / P);
  float *s[4], *par[5];
#pragma unroll
  for (int k = 0; k < 4; ++k) s[k] = s_cm + k * 64 * waves;
#pragma unroll
  for (int k = 0; k < 5; ++k) par[k] = s_cm + 4 * 64 * waves + k * a.C;
  const int b = blockIdx.x / a.chunks, tile = blockIdx.x % a.chunks;
  const long long n0 = (long long)tile * P + lane % P;
  const bool live = n0 < a.N;
  const long long n = live ? n0 : a.N - 1, r = (long long)b * a.N + n;
  const float inv_c = 1.f / (float)a.C;
  const f32x4 st = *reinterpret_cast<const f32x4 *>(a.stats + 4 * r);
  bool on[QN];
  int c0[QN];
  long long at[QN];
  S ry[QN][4], rd[QN][4], rx[QN][4], rh[QN][4];
  float hat1[QN][4], d[QN][4], hat[QN][4], dh[QN][4], nk[QN][4];
  bool stays[QN][4];
#pragma unroll
  for (int q = 0; q < QN; ++q) {
    c0[q] = 4 * (group + groups * q);
    on[q] = c0[q] < a.C;
    at[q] = ((long long)b * a.C + c0[q]) * a.N + n;
  }
  cm_fetch<S, QN>(a.y, a.exit, at, on, a.N, ry);
  cm_fetch<S, QN>(a.dout, a.dout != nullptr, at, on, a.N, rd);
  cm_fetch<S, QN>(a.x, a.dnext != nullptr, at, on, a.N, rx);
  cm_fetch<S, QN>(a.dnext, a.dnext != nullptr, at, on, a.N, rh);
  cm_params<T>(a, b, par[0]);
  __syncthreads();
#pragma unroll
  for (int q = 0; q < QN; ++q)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      hat1[q][e] = T::get(ry[q][e]);
      d[q][e] = live ? T::get(rd[q][e]) : 0.f;  // (a lane behind the last point: zero gradients)
      hat[q][e] = T::get(rx[q][e]);
      dh[q][e] = live ? T::get(rh[q][e]) : 0.f;
      nk[q][e] = 0.f;
    }
  float *partial = a.partial ? a.partial + (long long)blockIdx.x * 5 * a.C : nullptr;
  // a lane group's sums over its points of a quad's four columns
  auto flush = [&](int which, int c, float v0, float v1, float v2, float v3) {
    const f32x4 t = {lane_sum<P>(v0), lane_sum<P>(v1), lane_sum<P>(v2), lane_sum<P>(v3)};
    if (lane % P == 0) *reinterpret_cast<f32x4 *>(partial + (long long)which * a.C + c) = t;
  };
  if (a.exit) {  // (as in norm_bwd_kernel: the exit once more)
    unsigned long long seed = 0, offset = 0;
    if (DROP) { seed = a.drop.state[0]; offset = a.drop.state[1]; }
#pragma unroll
    for (int q = 0; q < QN; ++q) {
      if (!on[q]) continue;
      if (DROP) stay_v<4>(a.drop, seed, offset, r * a.C + c0[q], stays[q]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        hat1[q][e] = (hat1[q][e] - st[0]) * st[1];
        nk[q][e] = __builtin_fmaf(hat1[q][e], par[0][c0[q] + e], par[1][c0[q] + e]);
        if (DROP) nk[q][e] = stays[q][e] ? nk[q][e] * a.drop.scale : 0.f;
        if (!live) hat1[q][e] = nk[q][e] = 0.f;  // (its gradients are zeros, but 0 x inf is a NaN)
      }
    }
  }
  if (a.dnext) {
    float p1 = 0.f, p2 = 0.f;
#pragma unroll
    for (int q = 0; q < QN; ++q) {
      if (!on[q]) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (a.exit) hat[q][e] = __builtin_fmaf(a.alpha, hat[q][e], par[2][c0[q] + e] * nk[q][e]);
        hat[q][e] = live ? (hat[q][e] - st[2]) * st[3] : 0.f;
      }
      if (partial) {
        if (a.w2) flush(3, c0[q], dh[q][0] * hat[q][0], dh[q][1] * hat[q][1], dh[q][2] * hat[q][2], dh[q][3] * hat[q][3]);
        if (a.b2) flush(4, c0[q], dh[q][0], dh[q][1], dh[q][2], dh[q][3]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        dh[q][e] *= par[3][c0[q] + e];
        p1 = __builtin_fmaf(dh[q][e], hat[q][e], p1);
        p2 += dh[q][e];
      }
    }
    p1 = wave_sum<P>(p1, s[0], wave, lane, waves) * inv_c;
    p2 = a.kind2 == CL3D_NORM_LAYER ? wave_sum<P>(p2, s[1], wave, lane, waves) * inv_c : 0.f;
#pragma unroll
    for (int q = 0; q < QN; ++q)
#pragma unroll
      for (int e = 0; e < 4; ++e) d[q][e] = __builtin_fmaf(st[3], dh[q][e] - __builtin_fmaf(hat[q][e], p1, p2), d[q][e]);
  } else if (partial && a.next) {  // (the next norm's result was not used)
#pragma unroll
    for (int q = 0; q < QN; ++q) {
      if (!on[q]) continue;
      if (a.w2) flush(3, c0[q], 0.f, 0.f, 0.f, 0.f);
      if (a.b2) flush(4, c0[q], 0.f, 0.f, 0.f, 0.f);
    }
  }
  if (a.dx && live) {
#pragma unroll
    for (int q = 0; q < QN; ++q) {
      if (!on[q]) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e) static_cast<S *>(a.dx)[at[q] + e * a.N] = T::put(a.exit ? a.alpha * d[q][e] : d[q][e]);
    }
  }
  if (!a.exit) return;
  float p1 = 0.f, p2 = 0.f;
#pragma unroll
  for (int q = 0; q < QN; ++q) {
    if (!on[q]) continue;
#pragma unroll
    for (int e = 0; e < 4; ++e) d[q][e] = live ? d[q][e] : 0.f;
    if (partial && a.gate) flush(2, c0[q], d[q][0] * nk[q][0], d[q][1] * nk[q][1], d[q][2] * nk[q][2], d[q][3] * nk[q][3]);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (DROP) d[q][e] = stays[q][e] ? d[q][e] * a.drop.scale : 0.f;
      d[q][e] *= par[2][c0[q] + e];
    }
    if (partial && a.w1) {
      float t[4];  // (dropped: nothing, whatever y is)
#pragma unroll
      for (int e = 0; e < 4; ++e) t[e] = DROP && !stays[q][e] ? 0.f : d[q][e] * hat1[q][e];
      flush(0, c0[q], t[0], t[1], t[2], t[3]);
    }
    if (partial && a.b1) flush(1, c0[q], d[q][0], d[q][1], d[q][2], d[q][3]);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      d[q][e] *= par[0][c0[q] + e];
      p1 = __builtin_fmaf(d[q][e], hat1[q][e], p1);
      p2 += d[q][e];
    }
  }
  if (!a.dy) return;
  if (a.kind1 == CL3D_NORM_NONE) {  // (y does not enter its own gradient, whatever it is)
    p1 = p2 = 0.f;
#pragma unroll
    for (int q = 0; q < QN; ++q)
#pragma unroll
      for (int e = 0; e < 4; ++e) hat1[q][e] = 0.f;
  } else {
    p1 = wave_sum<P>(p1, s[2], wave, lane, waves) * inv_c;
    p2 = a.kind1 == CL3D_NORM_LAYER ? wave_sum<P>(p2, s[3], wave, lane, waves) * inv_c : 0.f;
  }
  if (!live) return;
#pragma unroll
  for (int q = 0; q < QN; ++q) {
    if (!on[q]) continue;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      static_cast<S *>(a.dy)[at[q] + e * a.N] = T::put(st[1] * (d[q][e] - __builtin_fmaf(hat1[q][e], p1, p2)));
  }
}

// sums of the partial rows [row][which][C]: 16 columns a workgroup, 64 runs of rows side by side, joined in order
struct NormSums {
  const float *partial;
  void *out[5];
  int C, rows, chunks, gate_cloud, param_f32;
};
template <typename T>
__global__ __launch_bounds__(1024) void norm_sums_kernel(NormSums a) {
  __shared__ float s[64][17];
  const int which = blockIdx.y, col = threadIdx.x & 15, part = threadIdx.x >> 4, c = blockIdx.x * 16 + col;
  const bool cloud = which == 2 && a.gate_cloud;
  const int b = blockIdx.z;
  if (a.out[which] == nullptr || (!cloud && b > 0)) return;
  const int rows = cloud ? a.chunks : a.rows, first = cloud ? b * a.chunks : 0;
  float t = 0.f;
  if (c < a.C) {
#pragma unroll 4
    for (int r = part; r < rows; r += 64) t += a.partial[((long long)(first + r) * 5 + which) * a.C + c];
  }
  s[part][col] = t;
  __syncthreads();
  if (threadIdx.x >= 16 || c >= a.C) return;
  t = 0.f;
#pragma unroll
  for (int q = 0; q < 64; ++q) t += s[q][col];
  const long long at = (cloud ? (long long)b * a.C : 0) + c;
  if (a.param_f32) static_cast<float *>(a.out[which])[at] = t;
  else static_cast<typename T::storage *>(a.out[which])[at] = T::put(t);
}

// ---- host side -----------------------------------------------------------------------------------------------------
// up to kNormMaxC channels any number, up to kNormWideC multiples of 8 (the last stage of a backbone of width 288: 4608) in memory
// that starts on 16 bytes.  4096 x 4608 bf16, exit and next norm: 71 us forward, 180 backward (the wider variants hold a wave a SIMD;
// 4096 x 4096: 36 and 139)
constexpr int kNormMaxC = 4096, kNormWideC = 6144;

// workgroups of a cloud and rows of each
static void norm_grid(NormArgs &a, int rows_per_pass, int target) {
  long long want = ((long long)target + a.B - 1) / a.B;
  const long long passes = (a.N + rows_per_pass - 1) / rows_per_pass;
  if (want > passes) want = passes;
  if (want < 1) want = 1;
  const long long per = ((passes + want - 1) / want) * rows_per_pass;
  a.per = (int)per;
  a.chunks = (int)((a.N + per - 1) / per);
}

struct NormMap {
  int tpr, nv, v;
};
// lanes of a row and pieces of a lane: 16-byte pieces where C and the pointers allow, else single elements.  As few lanes as hold
// the row in one piece each (several rows a wave), the whole workgroup where 64 do not; a lane's pieces cost registers (a row's
// values and the sums of its columns: 23 per element backward), so there are variants for 1, 2, 4 ... of them.
static NormMap norm_map(int dtype, int C, bool aligned) {
  const int kv = dtype == CL3D_F32 ? 4 : 8;
  const int v = aligned && C % kv == 0 ? kv : 1;
  const int pieces = C / v, need = (pieces + 255) / 256;
  if (v > 1 && pieces <= 16) return {16, 1, v};
  if (v > 1 && pieces <= 32) return {32, 1, v};
  if (pieces <= 64) return {64, 1, v};
  if (need <= 2) return {256, need, v};
  if (C > kNormMaxC) return {256, kNormWideC / 256 / v, v};
  if (v > 1 || need <= 4) return {256, 4, v};
  return {256, need <= 10 ? 10 : 16, v};
}

template <typename T, int TPR, int NV, int V> static void norm_run(bool backward, const NormArgs &a, hipStream_t st) {
  const dim3 grid((unsigned)((long long)a.B * a.chunks));
  const bool bias = V == 1 || a.b1 || a.b2;  // (single elements: one variant)
  if (!backward) {
    if (a.has_drop) hipLaunchKernelGGL((norm_fwd_kernel<T, TPR, NV, V, true>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((norm_fwd_kernel<T, TPR, NV, V, false>), grid, dim3(256), 0, st, a);
  } else if (bias) {
    if (a.has_drop) hipLaunchKernelGGL((norm_bwd_kernel<T, TPR, NV, V, true, true>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((norm_bwd_kernel<T, TPR, NV, V, false, true>), grid, dim3(256), 0, st, a);
  } else if constexpr (V > 1) {
    if (a.has_drop) hipLaunchKernelGGL((norm_bwd_kernel<T, TPR, NV, V, true, false>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((norm_bwd_kernel<T, TPR, NV, V, false, false>), grid, dim3(256), 0, st, a);
  }
}
template <typename T> static void norm_pick(const NormMap &m, bool backward, const NormArgs &a, hipStream_t st) {
  constexpr int V = T::kVec;
  if (m.v == 1) {
    if (m.tpr == 64) return norm_run<T, 64, 1, 1>(backward, a, st);
    if (m.nv == 1) return norm_run<T, 256, 1, 1>(backward, a, st);
    if (m.nv == 2) return norm_run<T, 256, 2, 1>(backward, a, st);
    if (m.nv == 4) return norm_run<T, 256, 4, 1>(backward, a, st);
    if (m.nv == 10) return norm_run<T, 256, 10, 1>(backward, a, st);
    return norm_run<T, 256, 16, 1>(backward, a, st);
  }
  if (m.tpr == 16) return norm_run<T, 16, 1, V>(backward, a, st);
  if (m.tpr == 32) return norm_run<T, 32, 1, V>(backward, a, st);
  if (m.tpr == 64) return norm_run<T, 64, 1, V>(backward, a, st);
  if (m.nv == 1) return norm_run<T, 256, 1, V>(backward, a, st);
  if (m.nv == 2) return norm_run<T, 256, 2, V>(backward, a, st);
  if constexpr (V == 4) if (m.nv == 4) return norm_run<T, 256, 4, V>(backward, a, st);  // (16-bit: two pieces hold kNormMaxC)
  norm_run<T, 256, kNormWideC / 256 / V, V>(backward, a, st);
}
static void norm_launch(int dtype, const NormMap &m, bool backward, const NormArgs &a, hipStream_t st) {
  if (dtype == CL3D_F32) norm_pick<F32>(m, backward, a, st);
  else if (dtype == CL3D_BF16) norm_pick<Bf16>(m, backward, a, st);
  else norm_pick<F16>(m, backward, a, st);
}

struct CmMap {
  int points, quads;  // P, QN
};
// points of a workgroup: as many as leave the channels to sixteen waves, fewer where the clouds would not fill the chip with
// workgroups or have no more points.  Exit with dropout and its gradients, 64 / 16 points: 16 x 144 x 16 f32 16 / 11 us, 1 x 72 x 2500
// 12.1 / 11.4, 2000 x 64 x 8 37 / 19, but 4 x 72 x 10 000 29 / 41, 16 x 144 x 1024 bf16 21 / 28 (short runs of a channel)
static CmMap cm_map(int B, int N, int C) {
  int p = C <= 256 ? 64 : C <= 512 ? 32 : 16;
  while (p > 16 && (p / 2 >= N || (long long)B * ceil_div(N, p) < 256)) p /= 2;
  return {p, C <= 2 * 4 * kCmWaves * 64 / p ? 2 : 4};  // (as few channels a lane as sixteen waves allow)
}
static int cm_waves(const CmMap &m, int C) { return ceil_div(ceil_div(C / 4, m.quads), 64 / m.points); }
static bool norm_cm(int order, int B, int N, int C) {
  if (order != CL3D_CHANNEL_MAJOR || N <= 1 || C % 4 != 0 || C > kCmMaxC) return false;
  const CmMap m = cm_map(B, N, C);
  return (long long)B * ceil_div(N, m.points) * 64 * cm_waves(m, C) <= 0xffffffffll;  // (threads that a grid counts)
}

template <typename T, int P, int QN> static void norm_cm_run(bool backward, const NormArgs &a, const CmMap &m, hipStream_t st) {
  const dim3 grid((unsigned)((long long)a.B * a.chunks)), block(64 * cm_waves(m, a.C));
  const size_t lds = cm_lds_bytes(cm_waves(m, a.C), a.C);
  if (backward) {
    if (a.has_drop) hipLaunchKernelGGL((norm_cm_bwd_kernel<T, P, QN, true>), grid, block, lds, st, a);
    else hipLaunchKernelGGL((norm_cm_bwd_kernel<T, P, QN, false>), grid, block, lds, st, a);
  } else {
    if (a.has_drop) hipLaunchKernelGGL((norm_cm_fwd_kernel<T, P, QN, true>), grid, block, lds, st, a);
    else hipLaunchKernelGGL((norm_cm_fwd_kernel<T, P, QN, false>), grid, block, lds, st, a);
  }
}
template <typename T> static void norm_cm_pick(bool backward, const NormArgs &a, hipStream_t st) {
  const CmMap m = cm_map(a.B, (int)a.N, a.C);
  if (m.points == 64) return m.quads == 2 ? norm_cm_run<T, 64, 2>(backward, a, m, st) : norm_cm_run<T, 64, 4>(backward, a, m, st);
  if (m.points == 32) return m.quads == 2 ? norm_cm_run<T, 32, 2>(backward, a, m, st) : norm_cm_run<T, 32, 4>(backward, a, m, st);
  return m.quads == 2 ? norm_cm_run<T, 16, 2>(backward, a, m, st) : norm_cm_run<T, 16, 4>(backward, a, m, st);
}
static void norm_cm_launch(int dtype, bool backward, const NormArgs &a, hipStream_t st) {
  if (dtype == CL3D_F32) norm_cm_pick<F32>(backward, a, st);
  else if (dtype == CL3D_BF16) norm_cm_pick<Bf16>(backward, a, st);
  else norm_cm_pick<F16>(backward, a, st);
}

static bool params_aligned(const cl3d_norm_residual *p) {
  return aligned16(p->weight) && aligned16(p->bias) && aligned16(p->gate) && aligned16(p->next_weight) && aligned16(p->next_bias);
}

static int norm_checks(const cl3d_norm_residual *p, bool backward, const char *who) {
  CL3D_REQUIRE(p != nullptr, "%s: null argument block", who);
  CL3D_REQUIRE(p->dtype == CL3D_F32 || p->dtype == CL3D_BF16 || p->dtype == CL3D_F16, "%s: unknown element type %d", who, p->dtype);
  CL3D_REQUIRE(p->order == CL3D_POINT_MAJOR || p->order == CL3D_CHANNEL_MAJOR, "%s: unknown memory order %d", who, p->order);
  CL3D_REQUIRE(p->B >= 0 && p->N >= 0 && p->C > 0, "%s: bad sizes", who);
  CL3D_REQUIRE(p->kind >= CL3D_NORM_NONE && p->kind <= CL3D_NORM_LAYER && p->next_kind >= CL3D_NORM_NONE && p->next_kind <= CL3D_NORM_LAYER,
               "%s: unknown norm", who);
  CL3D_REQUIRE(p->y != nullptr || p->next_kind != CL3D_NORM_NONE, "%s: neither a block to leave nor a norm to enter", who);
  CL3D_REQUIRE(p->y != nullptr || (!p->weight && !p->bias && !p->gate && p->p == 0.0), "%s: a gate, dropout or norm of a block that is not there", who);
  if (p->C > kNormWideC || (p->C > kNormMaxC && p->C % 8 != 0) || (long long)p->B * p->N > 0x7fffff00ll)
    return fail(CL3D_E_UNSUPPORTED, "%s: more than %d channels (multiples of 8: %d), or points than 31 bits count", who, kNormMaxC, kNormWideC);
  if (p->C > kNormMaxC && !(params_aligned(p) && aligned16(p->x) && aligned16(p->y) && aligned16(p->out) && aligned16(p->next) && aligned16(p->dout) &&
                            aligned16(p->dnext) && aligned16(p->dx) && aligned16(p->dy)))
    return fail(CL3D_E_UNSUPPORTED, "%s: tensors of more than %d channels start on 16 bytes", who, kNormMaxC);
  if (p->gate_cloud && p->B > 65535) return fail(CL3D_E_UNSUPPORTED, "%s: a gate per cloud for more than 65535 clouds", who);
  return CL3D_OK;
}

static void norm_args(NormArgs &a, const cl3d_norm_residual *p) {
  a = NormArgs{};
  a.x = p->x; a.y = p->y;
  a.w1 = p->weight; a.b1 = p->bias; a.gate = p->gate; a.w2 = p->next_weight; a.b2 = p->next_bias;
  a.stats = p->stats;
  a.N = p->N; a.B = p->B; a.C = p->C;
  if (norm_cm(p->order, p->B, p->N, p->C)) a.chunks = ceil_div(a.N, cm_map(p->B, p->N, p->C).points);
  else if (!p->gate_cloud) { a.N *= a.B; a.B = 1; }  // nothing differs from cloud to cloud: one run of rows
  a.kind1 = p->kind; a.kind2 = p->next_kind;
  a.exit = p->y != nullptr; a.next = p->next_kind != CL3D_NORM_NONE;
  a.gate_cloud = p->gate_cloud; a.param_f32 = p->param_f32 || p->dtype == CL3D_F32;
  a.alpha = p->residual_scale; a.eps1 = p->eps; a.eps2 = p->next_eps;
  a.has_drop = p->p > 0.0;
}

// workgroups: as many as are resident with the registers of the 16-bit variants (four a CU forward, three backward); more would
// load their parameters again, one round too few leaves CUs idle (backward 81 920 x 288: 512 156 us, 768 125, 1024 167)
constexpr int kNormFwdGroups = 1024, kNormBwdGroups = 768;

// point-major copies of channel-major tensors, and back
struct NormCopies {
  const cl3d_norm_residual *p;
  Arena ar;
  hipStream_t st;
  bool copies;
  int rc = CL3D_OK;
  NormCopies(const cl3d_norm_residual *p_, void *ws, hipStream_t st_)
      : p(p_), ar(ws), st(st_), copies(p_->order == CL3D_CHANNEL_MAJOR && p_->N > 1 && p_->C > 1 && !norm_cm(p_->order, p_->B, p_->N, p_->C)) {}
  void *place() { return ar.take((size_t)p->B * p->N * p->C * elem_bytes(p->dtype)); }
  const void *in(const void *t) {
    if (!copies || !t) return t;
    void *d = place();
    if (d && rc == CL3D_OK) rc = transposed(p->dtype, t, p->B, p->C, p->N, d, st);
    return d;
  }
  void *out(void *t) { return copies && t ? place() : t; }
  void back(const void *rows, void *t) {
    if (copies && t && rc == CL3D_OK) rc = transposed(p->dtype, rows, p->B, p->N, p->C, t, st);
  }
};

size_t point_norm_workspace(int B, int N, int C, int flags) {
  // flags: element type | memory order << 2 | tensors to copy << 3 | parameter gradients << 8
  if (B <= 0 || N <= 0 || C <= 0) return 0;
  Arena ar(nullptr);
  const int order = (flags >> 2) & 1;
  if (norm_cm(order, B, N, C)) return (flags >> 8) & 1 ? (size_t)B * ceil_div(N, cm_map(B, N, C).points) * 5 * (size_t)C * sizeof(float) : 0;
  if (order == CL3D_CHANNEL_MAJOR && N > 1 && C > 1)
    for (int q = 0; q < ((flags >> 3) & 31); ++q) ar.take((size_t)B * N * C * elem_bytes(flags & 3));
  // partial rows of the backward pass: at most kNormBwdGroups + B workgroups
  if ((flags >> 8) & 1) ar.take(((size_t)kNormBwdGroups + B) * 5 * (size_t)C * sizeof(float));
  return ar.used;
}

}  // namespace cl3d

extern "C" int cl3d_norm_residual_fwd(const cl3d_norm_residual *p, cl3d_stream_t stream) {
  using namespace cl3d;
  int rc = norm_checks(p, false, "norm_residual_fwd");
  if (rc != CL3D_OK) return rc;
  NormArgs a;
  norm_args(a, p);
  rc = make_drop(a.drop, p->rng, p->p, "norm_residual_fwd");
  if (rc != CL3D_OK) return rc;
  if (p->B == 0 || p->N == 0) return CL3D_OK;
  CL3D_REQUIRE(p->x && (!a.exit || p->out) && (!a.next || p->next), "norm_residual_fwd: null pointer");
  CL3D_REQUIRE(aligned16(p->stats) && aligned16(p->ws), "norm_residual_fwd: stats and scratch start on 16 bytes");
  const hipStream_t st = (hipStream_t)stream;
  NormCopies need(p, nullptr, st), c(p, p->ws, st);
  need.in(p->x), need.in(p->y), need.out(p->out), need.out(p->next);
  if (need.ar.used && (!p->ws || p->ws_bytes < need.ar.used))
    return fail(CL3D_E_WORKSPACE, "norm_residual_fwd: %zu bytes of scratch, %zu needed", p->ws_bytes, need.ar.used);
  a.x = c.in(p->x); a.y = c.in(p->y);
  a.o = c.out(p->out); a.h = c.out(p->next);
  if (c.rc != CL3D_OK) return c.rc;
  if (norm_cm(p->order, p->B, p->N, p->C)) {
    norm_cm_launch(p->dtype, false, a, st);
    return check_launch("cl3d_norm_residual_fwd");
  }
  const NormMap m = norm_map(p->dtype, p->C, aligned16(a.x) && aligned16(a.y) && aligned16(a.o) && aligned16(a.h) && params_aligned(p));
  norm_grid(a, 256 / m.tpr, kNormFwdGroups);
  norm_launch(p->dtype, m, false, a, st);
  c.back(a.o, p->out), c.back(a.h, p->next);
  return c.rc != CL3D_OK ? c.rc : check_launch("cl3d_norm_residual_fwd");
}

extern "C" int cl3d_norm_residual_bwd(const cl3d_norm_residual *p, cl3d_stream_t stream) {
  using namespace cl3d;
  int rc = norm_checks(p, true, "norm_residual_bwd");
  if (rc != CL3D_OK) return rc;
  NormArgs a;
  norm_args(a, p);
  rc = make_drop(a.drop, p->rng, p->p, "norm_residual_bwd");
  if (rc != CL3D_OK) return rc;
  CL3D_REQUIRE(p->B > 0 && p->N > 0, "norm_residual_bwd: no points (their gradients are zeros: nothing to launch)");
  CL3D_REQUIRE(p->stats && (p->dout || p->dnext), "norm_residual_bwd: null pointer");
  CL3D_REQUIRE(!p->dnext || (a.next && p->x), "norm_residual_bwd: a gradient of a norm that was not formed");
  CL3D_REQUIRE(!p->dout || a.exit, "norm_residual_bwd: a gradient of a sum that was not formed");
  CL3D_REQUIRE((!p->dweight || p->weight) && (!p->dbias || p->bias) && (!p->dgate || p->gate) &&
                   (!p->dnext_weight || (a.next && p->next_weight)) && (!p->dnext_bias || (a.next && p->next_bias)),
               "norm_residual_bwd: a gradient of a parameter that is not there");
  const hipStream_t st = (hipStream_t)stream;
  const bool sums = p->dweight || p->dbias || p->dgate || p->dnext_weight || p->dnext_bias;
  const void *x = p->dnext ? p->x : nullptr;  // (without the entry's gradient x is not looked at)
  NormCopies need(p, nullptr, st), c(p, p->ws, st);
  need.in(x), need.in(p->y), need.in(p->dout), need.in(p->dnext), need.out(p->dx), need.out(p->dy);
  const NormMap m = norm_map(p->dtype, p->C, params_aligned(p) && (need.copies || (aligned16(x) && aligned16(p->y) && aligned16(p->dout) && aligned16(p->dnext) &&
                                                             aligned16(p->dx) && aligned16(p->dy))));
  const bool cm = norm_cm(p->order, p->B, p->N, p->C);
  if (!cm) norm_grid(a, 256 / m.tpr, kNormBwdGroups);
  const size_t partial_bytes = sums ? (size_t)a.B * a.chunks * 5 * a.C * sizeof(float) : 0;
  if (sums) need.ar.take(partial_bytes);
  if (need.ar.used && (!p->ws || p->ws_bytes < need.ar.used))
    return fail(CL3D_E_WORKSPACE, "norm_residual_bwd: %zu bytes of scratch, %zu needed", p->ws_bytes, need.ar.used);
  CL3D_REQUIRE(aligned16(p->stats) && aligned16(p->ws), "norm_residual_bwd: stats and scratch start on 16 bytes");
  a.x = c.in(x); a.y = c.in(p->y); a.dout = c.in(p->dout); a.dnext = c.in(p->dnext);
  a.dx = c.out(p->dx); a.dy = c.out(p->dy);
  if (sums) a.partial = static_cast<float *>(c.ar.take(partial_bytes));
  if (c.rc != CL3D_OK) return c.rc;
  if (cm) norm_cm_launch(p->dtype, true, a, st);
  else norm_launch(p->dtype, m, true, a, st);
  c.back(a.dx, p->dx), c.back(a.dy, p->dy);
  if (c.rc != CL3D_OK) return c.rc;
  if (sums) {
    NormSums s{a.partial, {a.exit ? p->dweight : nullptr, a.exit ? p->dbias : nullptr, a.exit ? p->dgate : nullptr, p->dnext_weight, p->dnext_bias},
               a.C, a.B * a.chunks, a.chunks, a.gate_cloud, a.param_f32};
    const dim3 grid(ceil_div(a.C, 16), 5, a.gate_cloud && p->dgate ? a.B : 1);
    if (p->dtype == CL3D_F32) hipLaunchKernelGGL(norm_sums_kernel<F32>, grid, dim3(1024), 0, st, s);
    else if (p->dtype == CL3D_BF16) hipLaunchKernelGGL(norm_sums_kernel<Bf16>, grid, dim3(1024), 0, st, s);
    else hipLaunchKernelGGL(norm_sums_kernel<F16>, grid, dim3(1024), 0, st, s);
  }
  return check_launch("cl3d_norm_residual_bwd");
}
