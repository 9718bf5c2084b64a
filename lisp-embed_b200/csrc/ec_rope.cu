// ec_rope.cu -- rotary positions on caller-owned device buffers.
//
// Pair i of a head is turned by the angle pos * f_i:
//   y0 = x0 c - x1 s,  y1 = x1 c + x0 s,
// with (x0, x1) = (x[i], x[i + rot/2]) (halves) or (x[2i], x[2i + 1])
// (interleaved) of the first `rot` elements; the rest of the head passes
// through.  The turn is orthogonal, so its gradient is the turn by -angle.
#include <cuda_fp16.h>

#include <cmath>

#include "ec_ops.h"

namespace ec {
namespace {

// ------------------------------------------------------------------ table --
struct TableArgs {
  float *cos_t, *sin_t;
  int64_t positions;
  int half;
  double theta;
  int scaling;
  double factor, p0, p1, original, amplitude;
};

// frequency of pair i (llama.lisp:124-135 without scaling)
__device__ double rope_freq(const TableArgs& a, int i) {
  const double f = pow(a.theta, -static_cast<double>(i) / a.half);
  const double two_pi = 6.283185307179586476925;
  if (a.scaling == EC_ROPE_LINEAR) return f / a.factor;
  if (a.scaling == EC_ROPE_LLAMA3) {
    // turns within the original context: below p0 scaled, above p1 kept
    const double keep = fmin(fmax((a.original * f / two_pi - a.p0) / (a.p1 - a.p0), 0.0), 1.0);
    return (1.0 - keep) * f / a.factor + keep * f;
  }
  if (a.scaling == EC_ROPE_YARN) {
    // pair index at which p0 (fast) / p1 (slow) turns fit the original context
    const double rot = 2.0 * a.half, lt = 2.0 * log(a.theta);
    const double low = fmax(floor(rot * log(a.original / (a.p0 * two_pi)) / lt), 0.0);
    const double high = fmin(ceil(rot * log(a.original / (a.p1 * two_pi)) / lt), rot - 1.0);
    const double ramp = fmin(fmax((i - low) / fmax(high - low, 1e-3), 0.0), 1.0);
    return f / a.factor * ramp + f * (1.0 - ramp);
  }
  return f;
}

// Thread (i, r): pair i of `run` consecutive positions.  The first angle and the
// step of one position are turned into cos and sin once; the rest follows by
// rotating in double, which drifts by a few 2^-53 a step (run <= 64: far below
// the fp32 result).  Computing every angle's cos and sin took 150 us more for
// 262144 x 32, which take 17 us now, 10 of them for the stores; no pipe is full
// (issue 41%): a thread's run is one chain of double products.
__global__ void rope_table_kernel(const TableArgs a, int run) {
  pdl_wait();
  pdl_trigger();
  const int64_t runs = (a.positions + run - 1) / run, n = runs * a.half;
  for (int64_t e = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; e < n;
       e += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int i = static_cast<int>(e % a.half);
    const int64_t p0 = e / a.half * run;
    const double f = rope_freq(a, i);
    double s, c, s1, c1;
    sincos(static_cast<double>(p0) * f, &s, &c);
    sincos(f, &s1, &c1);
    const int64_t end = min(p0 + run, a.positions);
    for (int64_t p = p0; p < end; ++p) {
      a.cos_t[p * a.half + i] = static_cast<float>(c * a.amplitude);
      a.sin_t[p * a.half + i] = static_cast<float>(s * a.amplitude);
      const double t = c * c1 - s * s1;
      s = s * c1 + c * s1;
      c = t;
    }
  }
}

// ------------------------------------------------------------------- turn --
struct RopeArgs {
  const void* x;
  void* y;
  int64_t xt, xh, yt, yh;  // strides in elements
  int64_t tokens, positions;
  int heads, half, tail;   // tail: elements past the turned part (0 in place)
  int inverse;
  const int32_t* pos;
  const float *cos_t, *sin_t;
};

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

// V elements, moved in pieces of 16 bytes at most: eight entries of a table are
// two of them, and a table need not be aligned to more
template <typename T, int V>
struct alignas(sizeof(T) * V < 16 ? sizeof(T) * V : 16) Vec {
  T e[V];
};

// One thread: V pairs (or V elements of the tail) of a token's heads h0 ..
// h0 + heads_per - 1.  The angle's cos and sin are read once for them, and the
// elements of up to four heads are under way together.  I: index type that
// holds the number of threads (64-bit divisions slow the others down).  Bounded
// by reading and writing the rows: 65536 tokens of 24 heads of 128 in 138 us,
// 93% of the copy rate.  The tail of a partly turned head is copied one head
// after the other, each load waiting for the store before it (x and y may be the
// same): 9001 tokens of 12 heads, 64 of 96 elements turned, take 25 us in fp32,
// 13 of them for the bytes.
template <typename T, int V, bool INTER, typename I>
__global__ void rope_kernel(const RopeArgs a, int per_head, int groups, int heads_per) {
  using VT = Vec<T, V>;
  using VF = Vec<float, V>;
  constexpr int B = 4;
  pdl_wait();
  pdl_trigger();
  const I n = static_cast<I>(a.tokens) * groups * per_head;
  for (I e = static_cast<I>(blockIdx.x) * blockDim.x + threadIdx.x; e < n; e += static_cast<I>(gridDim.x) * blockDim.x) {
    const int c = static_cast<int>(e % per_head);
    const I tg = e / per_head;
    const int g = static_cast<int>(tg % groups);
    const int64_t t = tg / groups;
    const int32_t p = a.pos[t];
    if (p < 0) continue;  // a row without a position stays as it is
    const int h0 = g * heads_per, h1 = min(h0 + heads_per, a.heads);
    const T* x = static_cast<const T*>(a.x) + t * a.xt;
    T* y = static_cast<T*>(a.y) + t * a.yt;
    if (c * V >= a.half) {
      const int i = a.half + c * V;
      for (int h = h0; h < h1; ++h)
        *reinterpret_cast<VT*>(y + h * a.yh + i) = *reinterpret_cast<const VT*>(x + h * a.xh + i);
      continue;
    }
    VF co, si;
    if (p < a.positions) {
      co = *reinterpret_cast<const VF*>(a.cos_t + static_cast<int64_t>(p) * a.half + c * V);
      si = *reinterpret_cast<const VF*>(a.sin_t + static_cast<int64_t>(p) * a.half + c * V);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) co.e[i] = si.e[i] = NAN;
    }
    if (a.inverse) {
#pragma unroll
      for (int i = 0; i < V; ++i) si.e[i] = -si.e[i];
    }
    const int first = INTER ? 2 * c * V : c * V, second = first + (INTER ? V : a.half);
    for (int hb = h0; hb < h1; hb += B) {
      VT u[B], w[B];
#pragma unroll
      for (int b = 0; b < B; ++b)
        if (hb + b < h1) {
          u[b] = *reinterpret_cast<const VT*>(x + (hb + b) * a.xh + first);
          w[b] = *reinterpret_cast<const VT*>(x + (hb + b) * a.xh + second);
        }
#pragma unroll
      for (int b = 0; b < B; ++b)
        if (hb + b < h1) {
          VT ru, rw;
#pragma unroll
          for (int i = 0; i < V; ++i) {
            if constexpr (INTER && V > 1) {
              // V consecutive pairs: elements 2i, 2i + 1 of the two vectors
              const VT& s = 2 * i < V ? u[b] : w[b];
              VT& r = 2 * i < V ? ru : rw;
              const int k = (2 * i) % V;
              const float x0 = to_f(s.e[k]), x1 = to_f(s.e[k + 1]);
              r.e[k] = from_f<T>(x0 * co.e[i] - x1 * si.e[i]);
              r.e[k + 1] = from_f<T>(x1 * co.e[i] + x0 * si.e[i]);
            } else {
              const float x0 = to_f(u[b].e[i]), x1 = to_f(w[b].e[i]);
              ru.e[i] = from_f<T>(x0 * co.e[i] - x1 * si.e[i]);
              rw.e[i] = from_f<T>(x1 * co.e[i] + x0 * si.e[i]);
            }
          }
          *reinterpret_cast<VT*>(y + (hb + b) * a.yh + first) = ru;
          *reinterpret_cast<VT*>(y + (hb + b) * a.yh + second) = rw;
        }
    }
  }
}

template <typename T, int V>
cudaError_t launch_rope(const RopeArgs& a, int interleaved, int num_sms, cudaStream_t st) {
  const int per_head = (a.half + a.tail) / V;
  // a head per thread while that does not fill the GPU, then several, so
  // that the angles are read once for them
  int heads_per = 1;
  while (heads_per < 8 && a.tokens * per_head * ((a.heads + 2 * heads_per - 1) / (2 * heads_per)) >=
                              static_cast<int64_t>(num_sms) * 2048)
    heads_per *= 2;
  const int groups = (a.heads + heads_per - 1) / heads_per;
  const int64_t n = a.tokens * groups * per_head;
  const int64_t want = (n + 255) / 256, most = static_cast<int64_t>(num_sms) * 64;
  const int grid = static_cast<int>(want < most ? want : most);
  auto run = [&](auto index) {
    using I = decltype(index);
    return launch_pdl(interleaved ? rope_kernel<T, V, true, I> : rope_kernel<T, V, false, I>, dim3(grid), dim3(256), 0, st,
                      a, per_head, groups, heads_per);
  };
  return n < (int64_t(1) << 31) ? run(uint32_t{}) : run(int64_t{});
}

template <typename T>
cudaError_t launch_rope_v(const RopeArgs& a, int interleaved, int num_sms, cudaStream_t st) {
  // widest vector (16 bytes at most) that divides the turned half, the tail
  // and every stride, and to which the buffers are aligned
  auto fits = [&](int v) {
    const size_t b = sizeof(T) * v, tb = v > 4 ? 16 : 4 * v;
    return a.half % v == 0 && a.tail % v == 0 && a.xt % v == 0 && a.xh % v == 0 && a.yt % v == 0 && a.yh % v == 0 &&
           op_aligned(a.x, b) && op_aligned(a.y, b) && op_aligned(a.cos_t, tb) && op_aligned(a.sin_t, tb);
  };
  static_assert(alignof(Vec<float, 8>) == 16 && alignof(Vec<float, 4>) == 16 && alignof(Vec<float, 2>) == 8,
                "tables are read through this type");
  if constexpr (sizeof(T) == 2) {
    if (fits(8)) return launch_rope<T, 8>(a, interleaved, num_sms, st);
  }
  if (fits(4)) return launch_rope<T, 4>(a, interleaved, num_sms, st);
  if (fits(2)) return launch_rope<T, 2>(a, interleaved, num_sms, st);
  return launch_rope<T, 1>(a, interleaved, num_sms, st);
}

}  // namespace
}  // namespace ec

using namespace ec;

extern "C" int ec_rope_table(float* cos_t, float* sin_t, int64_t positions, int rot_dim, double theta, int scaling,
                             double factor, double p0, double p1, double original, double amplitude, void* stream) {
  clear_error();
  if (positions < 0 || positions >= (int64_t(1) << 31)) return set_error(EC_EINVAL, "bad number of positions");
  if (rot_dim < 2 || rot_dim % 2 || rot_dim > 1024) return set_error(EC_EINVAL, "rot_dim %d: even, 2 .. 1024", rot_dim);
  if (!(theta > 1.0) || !std::isfinite(theta)) return set_error(EC_EINVAL, "theta must be a finite number above 1");
  if (scaling < EC_ROPE_NONE || scaling > EC_ROPE_YARN) return set_error(EC_EINVAL, "unknown rope scaling %d", scaling);
  if (scaling != EC_ROPE_NONE && (!(factor >= 1.0) || !std::isfinite(factor)))
    return set_error(EC_EINVAL, "rope scaling factor must be a finite number of 1 or more");
  if (scaling == EC_ROPE_LLAMA3 && !(p0 > 0.0 && p1 > p0 && std::isfinite(p1) && original > 0.0 && std::isfinite(original)))
    return set_error(EC_EINVAL, "llama3 scaling needs 0 < low factor < high factor and an original length");
  if (scaling == EC_ROPE_YARN && !(p1 > 0.0 && p0 >= p1 && std::isfinite(p0) && original > 0.0 && std::isfinite(original)))
    return set_error(EC_EINVAL, "yarn scaling needs beta_fast >= beta_slow > 0 and an original length");
  if (!std::isfinite(amplitude) || amplitude < 0.0) return set_error(EC_EINVAL, "amplitude must be finite and >= 0");
  if (positions == 0) return EC_OK;
  if (!cos_t || !sin_t) return set_error(EC_EINVAL, "cos or sin table is NULL");
  if (!op_aligned(cos_t, 4) || !op_aligned(sin_t, 4)) return set_error(EC_EINVAL, "tables must be 4-byte aligned");
  OpDevice dev;
  if (int rc = dev.enter({cos_t, sin_t})) return rc;
  if (amplitude == 0.0) amplitude = scaling == EC_ROPE_YARN ? 0.1 * std::log(factor) + 1.0 : 1.0;
  const TableArgs a{cos_t, sin_t, positions, rot_dim / 2, theta, scaling, factor, p0, p1, original, amplitude};
  // long runs while that leaves a few warps to every scheduler
  int run = 64;
  while (run > 4 && positions * a.half / run < static_cast<int64_t>(dev.num_sms()) * 512) run /= 2;
  const int64_t want = ((positions + run - 1) / run * a.half + 127) / 128, most = int64_t(1) << 20;
  return check_cuda(launch_pdl(rope_table_kernel, dim3(static_cast<int>(want < most ? want : most)), dim3(128), 0,
                               static_cast<cudaStream_t>(stream), a, run),
                    "rope table");
}

extern "C" int ec_rope(const void* x, int64_t x_token, int64_t x_head, void* y, int64_t y_token, int64_t y_head,
                       int dtype, int64_t tokens, int heads, int head_dim, int rot_dim, int interleaved, int inverse,
                       const int32_t* pos, const float* cos_t, const float* sin_t, int64_t positions, void* stream) {
  clear_error();
  const int es = op_elem_size(dtype);
  if (!es) return set_error(EC_EINVAL, "unsupported dtype %d", dtype);
  if (tokens < 0 || heads < 1 || heads > 65536 || head_dim < 2 || head_dim > 4096)
    return set_error(EC_EINVAL, "bad rope shape: %lld tokens, %d heads of %d", static_cast<long long>(tokens), heads, head_dim);
  if (rot_dim < 2 || rot_dim % 2 || rot_dim > head_dim)
    return set_error(EC_EINVAL, "rot_dim %d: even, 2 .. head_dim %d", rot_dim, head_dim);
  if (positions < 1 || positions >= (int64_t(1) << 31)) return set_error(EC_EINVAL, "bad number of positions");
  if (tokens >= (int64_t(1) << 38)) return set_error(EC_EINVAL, "too many tokens");
  if (tokens == 0) return EC_OK;
  if (!x || !y || !pos || !cos_t || !sin_t) return set_error(EC_EINVAL, "a rope buffer is NULL");
  if (!op_aligned(x, es) || !op_aligned(y, es) || !op_aligned(pos, 4) || !op_aligned(cos_t, 4) || !op_aligned(sin_t, 4))
    return set_error(EC_EINVAL, "a rope buffer is not aligned to its element");
  // the stride of a single token or head is never used
  if (heads == 1) x_head = y_head = 0;
  if (tokens == 1) x_token = y_token = 0;
  if ((heads > 1 && (x_head < head_dim || y_head < head_dim)) ||
      (tokens > 1 && (x_token < head_dim || y_token < head_dim)) || x_head < 0 || y_head < 0 || x_token < 0 || y_token < 0)
    return set_error(EC_EINVAL, "rope strides overlap heads of %d", head_dim);
  if (!op_rows_apart(y_token, y_head, tokens, heads, head_dim))
    return set_error(EC_EINVAL, "y's tokens overlap (strides %lld / %lld)", static_cast<long long>(y_token),
                     static_cast<long long>(y_head));
  const bool in_place = x == y;
  if (in_place && (x_token != y_token || x_head != y_head))
    return set_error(EC_EINVAL, "in place the strides of x and y must be equal");
  OpDevice dev;
  if (int rc = dev.enter({x, y, pos, cos_t, sin_t})) return rc;
  RopeArgs a{x, y, x_token, x_head, y_token, y_head, tokens, positions, heads, rot_dim / 2,
             in_place ? 0 : head_dim - rot_dim, inverse ? 1 : 0, pos, cos_t, sin_t};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int il = interleaved ? 1 : 0;
  const cudaError_t e = dtype == EC_F32    ? launch_rope_v<float>(a, il, dev.num_sms(), st)
                        : dtype == EC_BF16 ? launch_rope_v<__nv_bfloat16>(a, il, dev.num_sms(), st)
                                           : launch_rope_v<__half>(a, il, dev.num_sms(), st);
  return check_cuda(e, "rope");
}
