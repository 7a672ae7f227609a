// Rotary positions over up to three token axes for sm_100a, queries and keys in one launch.
//
//   angle(token, pair i of axis a) = position_a * f,   f = position_scale_a * theta_a^(-2 i / d_a)
//   (u, w) -> (u cos - w sin, u sin + w cos);   the gradient is the same with -angle.
//
// Angles: a far position times a frequency needs more than 24 bits before it is reduced to one turn, so
// position * (f / 2 pi) is formed and reduced in fp64 and only the fraction of a turn goes to the fp32
// sincospi. A block works the angles of its tokens out once, into shared memory, and uses them for all
// heads of queries and keys. The rest is a stream: every element is read once and written once.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>

#include "common.cuh"

namespace b200na {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxPairs = 128;   // head_dim <= 256

struct RotaryArgs {
  const void* in[2];
  void* out[2];
  int64_t stride[2][5];          // batch, token axes, head (elements)
  int heads[2];
  int ndim, B, D, axes;
  int shape[3];
  int64_t tokens;                // of all batch entries
  int first_pair[4];             // pairs before axis a
  double origin[3];
  double turns[kMaxPairs];       // frequency of each pair in turns per position, negated for the inverse
  const void* positions;
  int position_type, positions_batched;
};

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

template <class T, int kN>
struct alignas(sizeof(T) * kN) Pack {
  T v[kN];
};

// kVec: pairs that a thread turns at once. Halves: kVec channels of each half, interleaved: 2 kVec
// neighbours.
template <class T, int kVec, bool kInterleaved>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const __grid_constant__ RotaryArgs a,
                                                          int block_tokens) {
  extern __shared__ float2 cs[];                              // [block_tokens][pairs]
  __shared__ int64_t in_at[2][16], out_at[2][16];             // element offsets of the tokens' first head
  const int pairs = a.first_pair[a.axes];
  const int64_t token0 = (int64_t)blockIdx.x * block_tokens;
  const int count = (int)(a.tokens - token0 < block_tokens ? a.tokens - token0 : block_tokens);
  const int64_t per_batch = a.tokens / a.B;

  for (int i = threadIdx.x; i < count * pairs; i += kThreads) {
    const int tt = i / pairs, pair = i - tt * pairs;
    int axis = 0;
    while (axis + 1 < a.axes && pair >= a.first_pair[axis + 1]) ++axis;
    const int64_t token = token0 + tt;
    double at;
    if (a.positions) {
      const int64_t row = a.positions_batched ? token : token % per_batch;
      const int64_t e = row * a.axes + axis;
      at = a.position_type == 0   ? (double)static_cast<const int*>(a.positions)[e]
           : a.position_type == 1 ? (double)static_cast<const int64_t*>(a.positions)[e]
                                  : (double)static_cast<const float*>(a.positions)[e];
    } else {
      int64_t rest = token % per_batch;
      int x = 0;
      for (int d = a.ndim - 1; d >= axis; --d) {
        x = (int)(rest % a.shape[d]);
        rest /= a.shape[d];
      }
      at = a.origin[axis] + x;
    }
    const double turn = at * a.turns[pair];
    float s, c;
    sincospif(2.f * (float)(turn - rint(turn)), &s, &c);
    cs[i] = make_float2(c, s);
  }
  if ((int)threadIdx.x < count) {
    const int64_t token = token0 + threadIdx.x, b = token / per_batch;
    int64_t rest = token - b * per_batch;
    for (int w = 0; w < 2; ++w) {
      int64_t off = b * a.stride[w][0], r = rest;
      for (int d = a.ndim - 1; d >= 0; --d) {
        off += (r % a.shape[d]) * a.stride[w][1 + d];
        r /= a.shape[d];
      }
      in_at[w][threadIdx.x] = off;
      out_at[w][threadIdx.x] = token * a.heads[w] * a.D;
    }
  }
  __syncthreads();

  const int heads = a.heads[0] + a.heads[1];
  const int rows = count * heads;
  const int chunks = pairs / kVec;          // of the turned channels of a row
  for (int i = threadIdx.x; i < rows * chunks; i += kThreads) {
    const int row = i / chunks, pair = (i - row * chunks) * kVec;
    const int tt = row / heads;
    int h = row - tt * heads;
    const int w = h >= a.heads[0];
    if (w) h -= a.heads[0];
    const T* in = static_cast<const T*>(a.in[w]) + in_at[w][tt] + h * a.stride[w][a.ndim + 1];
    T* out = static_cast<T*>(a.out[w]) + out_at[w][tt] + (int64_t)h * a.D;
    const float2* t = cs + tt * pairs + pair;
    if (kInterleaved && kVec > 1) {
      Pack<T, 2 * kVec> x = *reinterpret_cast<const Pack<T, 2 * kVec>*>(in + 2 * pair);
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        const float u = to_f(x.v[2 * e]), v = to_f(x.v[2 * e + 1]);
        x.v[2 * e] = from_f<T>(u * t[e].x - v * t[e].y);
        x.v[2 * e + 1] = from_f<T>(u * t[e].y + v * t[e].x);
      }
      *reinterpret_cast<Pack<T, 2 * kVec>*>(out + 2 * pair) = x;
    } else {
      int axis = 0;
      while (axis + 1 < a.axes && pair >= a.first_pair[axis + 1]) ++axis;
      const int half = kInterleaved ? 1 : a.first_pair[axis + 1] - a.first_pair[axis];
      const int lo = kInterleaved ? 2 * pair : a.first_pair[axis] + pair;   // 2 first + (pair - first)
      Pack<T, kVec> x = *reinterpret_cast<const Pack<T, kVec>*>(in + lo);
      Pack<T, kVec> y = *reinterpret_cast<const Pack<T, kVec>*>(in + lo + half);
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        const float u = to_f(x.v[e]), v = to_f(y.v[e]);
        x.v[e] = from_f<T>(u * t[e].x - v * t[e].y);
        y.v[e] = from_f<T>(u * t[e].y + v * t[e].x);
      }
      *reinterpret_cast<Pack<T, kVec>*>(out + lo) = x;
      *reinterpret_cast<Pack<T, kVec>*>(out + lo + half) = y;
    }
  }
  // channels behind the last axis
  const int turned = 2 * pairs, rest = a.D - turned;
  for (int i = threadIdx.x; i < rows * rest; i += kThreads) {
    const int row = i / rest, ch = turned + i - row * rest;
    const int tt = row / heads;
    int h = row - tt * heads;
    const int w = h >= a.heads[0];
    if (w) h -= a.heads[0];
    static_cast<T*>(a.out[w])[out_at[w][tt] + (int64_t)h * a.D + ch] =
        static_cast<const T*>(a.in[w])[in_at[w][tt] + h * a.stride[w][a.ndim + 1] + ch];
  }
}

template <class T, bool kInterleaved>
int launch(const RotaryArgs& a, int vec, int sms, cudaStream_t stream) {
  const int pairs = a.first_pair[a.axes];
  // As many tokens to a block as leave every SM four blocks; 16 at most.
  int64_t per = a.tokens / ((int64_t)sms * 4);
  int block_tokens = (int)(per < 1 ? 1 : per > 16 ? 16 : per);
  const int64_t blocks = (a.tokens + block_tokens - 1) / block_tokens;
  if (blocks > 0x7fffffff) return B200NA_ERR_INVALID_ARGUMENT;
  const size_t smem = (size_t)block_tokens * pairs * sizeof(float2);
  switch (vec) {
    case 8: rotary_kernel<T, 8, kInterleaved><<<(unsigned)blocks, kThreads, smem, stream>>>(a, block_tokens); break;
    case 4: rotary_kernel<T, 4, kInterleaved><<<(unsigned)blocks, kThreads, smem, stream>>>(a, block_tokens); break;
    case 2: rotary_kernel<T, 2, kInterleaved><<<(unsigned)blocks, kThreads, smem, stream>>>(a, block_tokens); break;
    default: rotary_kernel<T, 1, kInterleaved><<<(unsigned)blocks, kThreads, smem, stream>>>(a, block_tokens); break;
  }
  B200NA_CUDA_TRY(cudaGetLastError());
  return B200NA_OK;
}

}  // namespace
}  // namespace b200na

extern "C" B200NA_API int b200na_rotary(
    const void* query, const void* key, void* query_out, void* key_out, int ndim, const int* shape, int B,
    int Hq, int Hkv, int D, int dtype, const int64_t* query_strides, const int64_t* key_strides, int axes,
    const int* axis_dims, const double* theta, const double* position_scale, const int64_t* origin,
    const void* positions, int position_type, int positions_batched, int interleaved, int inverse,
    b200na_stream_t stream) {
  using namespace b200na;
  if (ndim < 1 || ndim > 3 || !shape || axes < 1 || axes > 3 || !axis_dims || !theta || !position_scale ||
      !query_strides || B < 0 || Hq < 1 || Hkv < 0 || D < 1 ||
      Hq > 65536 || Hkv > 65536)
    return B200NA_ERR_INVALID_ARGUMENT;
  if (D > 2 * kMaxPairs) return B200NA_ERR_UNSUPPORTED;
  if (dtype != B200NA_F32 && dtype != B200NA_F16 && dtype != B200NA_BF16) return B200NA_ERR_UNSUPPORTED;
  if (positions ? position_type < 0 || position_type > 2 : axes != ndim || !origin)
    return B200NA_ERR_INVALID_ARGUMENT;
  if (Hkv > 0 && !key_strides) return B200NA_ERR_INVALID_ARGUMENT;
  RotaryArgs a{};
  a.ndim = ndim;
  a.axes = axes;
  a.B = B;
  a.D = D;
  a.heads[0] = Hq;
  a.heads[1] = Hkv;
  a.tokens = B;
  for (int d = 0; d < ndim; ++d) {
    if (shape[d] < 0) return B200NA_ERR_INVALID_ARGUMENT;
    if (shape[d] > 0 && a.tokens > ((int64_t)1 << 40) / shape[d]) return B200NA_ERR_INVALID_ARGUMENT;
    a.shape[d] = shape[d];
    a.tokens *= shape[d];
  }
  const int elem = dtype == B200NA_F32 ? 4 : 2;
  // pairs a thread turns at once: 16 bytes of every stream where sizes, strides and addresses allow
  int vec = 16 / elem / (interleaved ? 2 : 1);
  for (int d = 0; d < axes; ++d) {
    if (axis_dims[d] < 0 || axis_dims[d] % 2 || !(theta[d] > 0) || !std::isfinite(theta[d]) ||
        !std::isfinite(position_scale[d]))
      return B200NA_ERR_INVALID_ARGUMENT;
    const int n = axis_dims[d] / 2;
    a.first_pair[d + 1] = a.first_pair[d] + n;
    if (a.first_pair[d + 1] > D / 2) return B200NA_ERR_INVALID_ARGUMENT;
    while (n % vec) vec /= 2;
    for (int i = 0; i < n; ++i)
      a.turns[a.first_pair[d] + i] = (inverse ? -1.0 : 1.0) * position_scale[d] *
                                     std::pow(theta[d], -2.0 * i / axis_dims[d]) / 6.283185307179586476925286766559;
    a.origin[d] = origin ? (double)origin[d] : 0.0;
  }
  if (a.tokens == 0) return B200NA_OK;
  if (!query || !query_out || (Hkv > 0 && (!key || !key_out))) return B200NA_ERR_INVALID_ARGUMENT;
  a.in[0] = query;
  a.in[1] = key;
  a.out[0] = query_out;
  a.out[1] = key_out;
  for (int w = 0; w < (Hkv > 0 ? 2 : 1); ++w) {
    const int64_t* s = w ? key_strides : query_strides;
    for (int i = 0; i < ndim + 2; ++i) {
      const int64_t extent = i == 0 ? B : i <= ndim ? shape[i - 1] : a.heads[w];
      a.stride[w][i] = extent > 1 ? s[i] : 0;
    }
    const auto fits = [&](int v) {
      const int n = interleaved ? 2 * v : v;
      if ((reinterpret_cast<uintptr_t>(a.in[w]) | reinterpret_cast<uintptr_t>(a.out[w])) % (n * elem)) return false;
      for (int i = 0; i < ndim + 2; ++i)
        if (a.stride[w][i] % n) return false;
      return D % n == 0;
    };
    while (vec > 1 && !fits(vec)) vec /= 2;   // one pair at a time has no alignment to keep
  }
  a.positions = positions;
  a.position_type = position_type;
  a.positions_batched = positions_batched;
  int sms = 0;
  const int rc = sm_count_of_current_device(&sms);
  if (rc != B200NA_OK) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  switch (dtype) {
    case B200NA_F32: return interleaved ? launch<float, true>(a, vec, sms, st) : launch<float, false>(a, vec, sms, st);
    case B200NA_F16: return interleaved ? launch<__half, true>(a, vec, sms, st) : launch<__half, false>(a, vec, sms, st);
    default:
      return interleaved ? launch<__nv_bfloat16, true>(a, vec, sms, st)
                         : launch<__nv_bfloat16, false>(a, vec, sms, st);
  }
}
