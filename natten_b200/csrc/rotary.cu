// Rotary positions over up to three token axes for sm_100a, queries and keys in one launch.
//
//   angle(token, pair i of axis a) = position_a * f,   f = position_scale_a * theta_a^(-2 i / d_a)
//   (u, w) -> (u cos - w sin, u sin + w cos);   the gradient is the same with -angle.
//
// Angles: a far position times a frequency needs more than 24 bits before it is reduced to one turn, so
// position * (f / 2 pi) is formed and reduced in fp64 and only the fraction of a turn goes to the fp32
// sincospi. An angle is off by 2e-15 of itself at most (the frequency's rounding and the product's): nothing in fp32 up
// to about 2^25, 1e-5 at 2^32. A block works the angles of its tokens out once, into shared memory, and its threads keep their
// columns' cosines and sines while they go through the heads of queries and keys, of several batch entries where
// these stand at the same places. The rest is a stream: every element is read once and written once.
#include <algorithm>
#include <cmath>

#include "paged.cuh"

namespace b200na {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxPairs = 128;   // head_dim <= 256
constexpr int kMostTokens = 64;  // of a block

struct RotaryArgs {
  const void* in[2];
  void* out[2];
  int64_t stride[2][5];          // batch, token axes, head (elements)
  int heads[2];
  int ndim, B, D, axes;
  int shape[3];
  int64_t batch_tokens;          // of a batch entry
  int block_tokens, block_batches, tiles;   // of a block; blocks of a batch entry's tokens
  int first_pair[4];             // pairs before axis a
  double origin[3];
  double turns[kMaxPairs];       // frequency of each pair in turns per position, negated for the inverse
  const void* positions;
  int position_type, positions_batched;
};

// kVec: pairs that a thread turns at once. Halves: kVec channels of each half, interleaved: 2 kVec
// neighbours. A thread keeps its column of the rows, so that what depends on it is worked out once.
template <class T, int kVec, bool kInterleaved>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const __grid_constant__ RotaryArgs a) {
  // Rows that a thread has under way: about 96 bytes. Both launches of a training step on 15 x 30 x 52 tokens of 12 + 12
  // heads, as a replayed graph, with 1, 2, 3, 4, 6 rows of 16 bytes: 78, 64, 67, 68, 60 us (58 now; calls from the host
  // take 73 to 77, autograd's pace). A video of 32 x 48 x 80 tokens, 24 + 24 heads of 128 channels, 3.0 GB: 462 us, the
  // copy rate; 12 + 12 heads in fp32, the same bytes: 460 us.
  constexpr int kRowBytes = 2 * kVec * (int)sizeof(T), kUnroll = kRowBytes >= 32 ? 3 : 6;
  extern __shared__ __align__(16) float cs[];                 // [block_tokens][cosines, sines][stride]
  __shared__ int64_t in_at[2][kMostTokens], out_at[2][kMostTokens];   // offsets of the tokens' first head
  __shared__ double place[kMostTokens][3];
  const int pairs = a.first_pair[a.axes], stride = (pairs + 3) / 4 * 4;
  const int block_tokens = a.block_tokens, group = blockIdx.x / a.tiles;
  const int64_t token0 = (int64_t)(blockIdx.x - group * a.tiles) * block_tokens;
  const int b0 = group * a.block_batches, batches = min(a.block_batches, a.B - b0);
  const int count = (int)(a.batch_tokens - token0 < block_tokens ? a.batch_tokens - token0 : block_tokens);

  // For the angles a thread keeps its pair: a launch parameter that every lane reads elsewhere is read one lane
  // after the other, so it is read once.
  const int at_once = pairs > 0 ? kThreads / pairs : 0, my_token = pairs > 0 ? threadIdx.x / pairs : 0;
  const int my_pair = threadIdx.x - my_token * pairs;
  const int my_axis = (my_pair >= a.first_pair[1] && a.axes > 1) + (my_pair >= a.first_pair[2] && a.axes > 2);
  const double my_turns = my_token < at_once ? a.turns[my_pair] : 0.0;

  if ((int)threadIdx.x < count) {
    const int tt = threadIdx.x;
    const int64_t token = token0 + tt, whole = b0 * a.batch_tokens + token;
    int64_t off[2] = {b0 * a.stride[0][0], b0 * a.stride[1][0]};
    uint64_t r = token;
    for (int d = a.ndim - 1; d >= 0; --d) {
      uint64_t up = 0;
      uint32_t x = (uint32_t)r;
      if (d > 0) {
        up = r >> 32 ? r / a.shape[d] : (uint32_t)r / (uint32_t)a.shape[d];
        x = (uint32_t)(r - up * a.shape[d]);
      }
      r = up;
      off[0] += x * a.stride[0][1 + d];
      off[1] += x * a.stride[1][1 + d];
      if (!a.positions) place[tt][d] = a.origin[d] + (double)x;
    }
    if (a.positions) {
      const int64_t e = (a.positions_batched ? whole : token) * a.axes;
      for (int axis = 0; axis < a.axes; ++axis)
        place[tt][axis] = a.position_type == 0   ? (double)static_cast<const int*>(a.positions)[e + axis]
                          : a.position_type == 1 ? (double)static_cast<const int64_t*>(a.positions)[e + axis]
                                                 : (double)static_cast<const float*>(a.positions)[e + axis];
    }
    for (int w = 0; w < 2; ++w) {
      in_at[w][tt] = off[w];
      out_at[w][tt] = whole * a.heads[w] * a.D;
    }
  }
  __syncthreads();
  if (at_once > 0 && my_token < at_once) {
    for (int t = my_token; t < count; t += at_once) {
      const double turn = place[t][my_axis] * my_turns;
      float s, c;
      sincospif(2.f * (float)(turn - rint(turn)), &s, &c);
      cs[2 * t * stride + my_pair] = c;
      cs[(2 * t + 1) * stride + my_pair] = s;
    }
  }
  __syncthreads();

  // A thread keeps its token and its column: the cosines and sines stay in registers while it goes through
  // the heads, kUnroll of them at a time so that their loads are under way together.
  const int chunks = pairs / kVec;
  const int slot = chunks > 0 ? threadIdx.x / chunks : 0;
  const int per_token = chunks > 0 ? max(1, kThreads / chunks / block_tokens) : 0;   // threads of a column
  const int tt = chunks > 0 ? slot % block_tokens : 0, first = slot / block_tokens;
  if (tt < count && first < per_token) {
    const int pair = (threadIdx.x - slot * chunks) * kVec;
    const int axis = (pair >= a.first_pair[1] && a.axes > 1) + (pair >= a.first_pair[2] && a.axes > 2);
    const int half = kInterleaved ? 1 : a.first_pair[axis + 1] - a.first_pair[axis];
    const int lo = kInterleaved ? 2 * pair : a.first_pair[axis] + pair;     // 2 first + (pair - first)
    alignas(16) float cosine[kVec], sine[kVec];
    constexpr int kLoad = kVec < 4 ? kVec : 4;
#pragma unroll
    for (int e = 0; e < kVec; e += kLoad) {
      *reinterpret_cast<Elements<float, kLoad>*>(cosine + e) = *reinterpret_cast<const Elements<float, kLoad>*>(cs + 2 * tt * stride + pair + e);
      *reinterpret_cast<Elements<float, kLoad>*>(sine + e) = *reinterpret_cast<const Elements<float, kLoad>*>(cs + (2 * tt + 1) * stride + pair + e);
    }
    for (int z = 0; z < 2 * batches; ++z) {       // queries, then keys, of one batch entry after the other
      const int w = z >= batches, bi = z - w * batches;
      const int64_t head_stride = a.stride[w][a.ndim + 1];
      const T* src = static_cast<const T*>(a.in[w]) + in_at[w][tt] + bi * a.stride[w][0] + first * head_stride + lo;
      T* dst = static_cast<T*>(a.out[w]) + out_at[w][tt] + bi * a.batch_tokens * a.heads[w] * a.D + first * a.D + lo;
      const int64_t in_step = per_token * head_stride;
      const int out_step = per_token * a.D;
      for (int h = first; h < a.heads[w]; h += kUnroll * per_token) {
        constexpr int kWide = kInterleaved && kVec > 1 ? 2 * kVec : kVec;
        using Piece = Raw<T, kWide>;
        Piece x[kUnroll], y[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
          if (h + u * per_token < a.heads[w]) {
            x[u] = *reinterpret_cast<const Piece*>(src + u * in_step);
            if (kWide == kVec) y[u] = *reinterpret_cast<const Piece*>(src + u * in_step + half);
          }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
          if (h + u * per_token >= a.heads[w]) continue;
          T* const to = dst + u * out_step;
          if constexpr (kWide == kVec) {
            float p[kVec], q[kVec];
            to_floats<T, kVec>(x[u], p);
            to_floats<T, kVec>(y[u], q);
#pragma unroll
            for (int e = 0; e < kVec; ++e) {
              const float v = p[e];
              p[e] = v * cosine[e] - q[e] * sine[e];
              q[e] = v * sine[e] + q[e] * cosine[e];
            }
            *reinterpret_cast<Piece*>(to) = from_floats<T, kVec>(p);
            *reinterpret_cast<Piece*>(to + half) = from_floats<T, kVec>(q);
          } else {
            float p[kWide];
            to_floats<T, kWide>(x[u], p);
#pragma unroll
            for (int e = 0; e < kVec; ++e) {
              const float v = p[2 * e], z = p[2 * e + 1];
              p[2 * e] = v * cosine[e] - z * sine[e];
              p[2 * e + 1] = v * sine[e] + z * cosine[e];
            }
            *reinterpret_cast<Piece*>(to) = from_floats<T, kWide>(p);
          }
        }
        src += kUnroll * in_step;
        dst += kUnroll * out_step;
      }
    }
  }
  // channels behind the last axis
  const int heads = a.heads[0] + a.heads[1], rows = batches * count * heads;
  const int turned = 2 * pairs, rest = a.D - turned;
  for (int i = threadIdx.x; i < rows * rest; i += kThreads) {
    const int row = i / rest, ch = turned + i - row * rest;
    const int token = row / heads, bi = token / count, t = token - bi * count;
    int h = row - token * heads;
    const int w = h >= a.heads[0];
    if (w) h -= a.heads[0];
    static_cast<T*>(a.out[w])[out_at[w][t] + bi * a.batch_tokens * a.heads[w] * a.D + h * a.D + ch] =
        static_cast<const T*>(a.in[w])[in_at[w][t] + bi * a.stride[w][0] + h * a.stride[w][a.ndim + 1] + ch];
  }
}

template <class T, bool kInterleaved, int kVec>
void launch_vec(const RotaryArgs& a, int vec, unsigned blocks, size_t smem, cudaStream_t stream) {
  if constexpr (kVec > 1) {
    if (vec < kVec) return launch_vec<T, kInterleaved, kVec / 2>(a, vec, blocks, smem, stream);
  }
  rotary_kernel<T, kVec, kInterleaved><<<blocks, kThreads, smem, stream>>>(a);
}

template <class T, bool kInterleaved>
int launch(RotaryArgs a, int vec, int sms, cudaStream_t stream) {
  const int pairs = a.first_pair[a.axes], heads = a.heads[0] + a.heads[1];
  // Tokens of a block, a power of two so that a token's columns fill whole warps: as many as give each of its
  // threads a row, while every SM has a block; more, as long as every SM has eight. (21 x 31 x 96 tokens of 4 + 2
  // heads with at most 8, 16, 32 tokens: 88, 60, 53 us; 44 now.)
  const int64_t tokens = a.B * a.batch_tokens, per = tokens / ((int64_t)sms * 8);
  const int slots = pairs >= vec ? kThreads / (pairs / vec) : kMostTokens;
  const int most = std::min(std::min(slots, kMostTokens), 32 * 1024 / (8 * std::max(pairs, 1)));
  a.block_tokens = 1;
  while (a.block_tokens * 2 <= most && a.block_tokens < a.batch_tokens &&
         (a.block_tokens * 2 <= per ||
          (a.block_tokens * std::max(a.heads[0], a.heads[1]) < slots && a.block_tokens * 2 <= per * 8)))
    a.block_tokens *= 2;
  // Batch entries whose tokens stand at the same places share the angles: up to 32 rows of a token together.
  // (16 videos of 6 + 3 heads 214 -> 195 us, 184 with the
  // frequencies read once.)
  a.block_batches = 1;
  if (!a.positions || !a.positions_batched)
    while (a.block_batches < a.B && a.block_batches * 2 * heads <= 32 && a.block_batches * 2 * a.block_tokens <= per)
      a.block_batches *= 2;
  const int64_t tiles = (a.batch_tokens + a.block_tokens - 1) / a.block_tokens;
  const int64_t blocks = tiles * ((a.B + a.block_batches - 1) / a.block_batches);
  if (blocks > 0x7fffffff) return B200NA_ERR_INVALID_ARGUMENT;
  a.tiles = (int)tiles;
  const size_t smem = (size_t)a.block_tokens * 2 * ((pairs + 3) / 4 * 4) * sizeof(float);
  launch_vec<T, kInterleaved, 16 / (int)sizeof(T) / (kInterleaved ? 2 : 1)>(a, vec, (unsigned)blocks, smem, stream);
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
  int64_t tokens = B;
  for (int d = 0; d < ndim; ++d) {
    if (shape[d] < 0) return B200NA_ERR_INVALID_ARGUMENT;
    if (shape[d] > 0 && tokens > ((int64_t)1 << 40) / shape[d]) return B200NA_ERR_INVALID_ARGUMENT;
    a.shape[d] = shape[d];
    tokens *= shape[d];
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
    // theta^(-2 i / d) / 2 pi: every eighth one by itself, the others by a product with the first ones (1e-15)
    const double front = (inverse ? -1.0 : 1.0) * position_scale[d] / 6.283185307179586476925286766559;
    const double step = n > 1 ? std::pow(theta[d], -2.0 / axis_dims[d]) : 1.0;
    double* const turns = a.turns + a.first_pair[d];
    for (int i = 0; i < n; ++i)
      turns[i] = i % 8 ? turns[i - 1] * step : front * (i ? std::pow(theta[d], -2.0 * i / axis_dims[d]) : 1.0);
    a.origin[d] = origin ? (double)origin[d] : 0.0;
  }
  if (tokens == 0) return B200NA_OK;
  a.batch_tokens = tokens / B;
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
