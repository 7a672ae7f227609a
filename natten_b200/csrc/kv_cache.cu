// Writing tokens into the paged key/value cache and reading them back, for sm_100a.
//
// Both are streams of rows (one token's channels of one head): a row is read once and written once,
// keys and values in one launch. A group of lanes holds a whole row in registers, 16 bytes a lane and
// access, so the largest magnitude of a row (for its 8-bit scale) is a few shuffles away and the row is
// not read again. A block works on consecutive tokens of one sequence, so that a sequence's start and
// count are read once a block and places need 32-bit arithmetic only. One row of keys and one of values to a
// lane at a time: reading 8-bit prefixes (355 MB) takes 66 us so, 69 with two, 92 with three, 121 with four rows
// in flight, whose registers cost more threads than they give; writing 8-bit prompts (63 MB) 16.7 us, 18.4 with two.
#include <algorithm>

#include "paged.cuh"

namespace b200na {
namespace {

constexpr int kThreads = 256;
// Accesses of a row that a lane makes at least: two where the row has a scale, whose work is then shared by
// twice as many elements.
__host__ __device__ constexpr int lane_share(bool scaled, int vec) { return scaled && vec > 1 ? 2 : 1; }

struct MoveArgs {
  PagedPool pool[2];             // keys, values
  bool same_strides;             // of the two
  PageTable table;
  void* data[2];                 // [B, T, heads, D]: given to the write, filled (contiguous) by the read
  int64_t batch[2], token[2], head[2];   // its strides (elements)
  bool narrow;                   // those of tokens and heads fit 31 bits
  const int* start;
  const int* counts;
  int B, T, heads, D;
  uint32_t heads_magic;          // ceil(2^32 / heads): x / heads = x * magic >> 32 for x * heads < 2^32
  int tokens;                    // of a block
  int tiles;                     // blocks of a sequence
};

// The largest magnitude of a piece as bits: magnitudes of floats are ordered like their bits, infinities and
// NaNs come after all finite ones. 16-bit types: two maxima side by side.
template <class T, int kVec> __device__ __forceinline__ uint32_t largest_bits(const Raw<T, kVec>& x, uint32_t most) {
  if constexpr (sizeof(T) * kVec == 2) {
    return __vmaxu2(most, (uint32_t)x & 0x7fffu);
  } else {
    uint32_t w[sizeof(T) * kVec / 4];
    memcpy(w, &x, sizeof(w));
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) * kVec / 4); ++i)
      most = sizeof(T) == 2 ? __vmaxu2(most, w[i] & 0x7fff7fffu) : max(most, w[i] & 0x7fffffffu);
    return most;
  }
}

// The bytes of x / scale as the definition has them: a 32-bit division, then the rounding to e4m3. (A product with
// the rounded reciprocal may leave the middle of two e4m3 numbers and end at the other one.) Two values an instruction.
//  - 16-bit values: a product with the reciprocal in two parts, rounded once, 2^-45 off before that. The bytes are the
//    division's for every pair of a 16-bit value and the largest magnitude of its row (all mantissas of fp16 and bf16,
//    and the exponents at both ends of the range, were gone through).
//  - fp32: the correctly rounded quotient by a product with the reciprocal and Markstein's correction by its remainder.
//    Small scales and their rows are multiplied by 2^64 first, so that the remainders of all quotients that e4m3 does
//    not round to zero are representable.
// Writing 8-bit prompts out of 16-bit values (63 MB) takes 16.6 us so, as with the rounded reciprocal alone, and 17.1
// with Markstein's correction; out of fp32 values (105 MB) 30.6 us, 28.9 with the reciprocal alone.
template <class T> struct Quotient {
  float2 up, over, factor;
  __device__ __forceinline__ explicit Quotient(float scale) {
    if constexpr (sizeof(T) == 2) {
      const float r = __frcp_rd(scale), rest = __fmaf_rn(-scale, r, 1.f) * r;      // (never negative: -0 stays -0)
      factor = make_float2(r, r);
      up = make_float2(rest, rest);
    } else {
      const float u = scale < 0x1p-64f ? 0x1p64f : 1.f, r = __frcp_rn(scale * u);
      up = make_float2(-u, -u);
      over = make_float2(scale * u, scale * u);
      factor = make_float2(-r, -r);
    }
  }
  __device__ __forceinline__ float2 operator()(float2 x) const {
    if constexpr (sizeof(T) == 2) return __ffma2_rn(x, factor, __fmul2_rn(x, up));
    const float2 v = __fmul2_rn(x, up), q = __fmul2_rn(v, factor);                  // -x, x / scale
    return __ffma2_rn(__ffma2_rn(over, q, v), factor, q);
  }
  template <int kN> __device__ __forceinline__ void divide(float (&x)[kN]) const {
#pragma unroll
    for (int e = 0; e < kN; e += 2) {
      const float2 y = (*this)(make_float2(x[e], e + 1 < kN ? x[e + 1] : 0.f));
      x[e] = y.x;
      if (e + 1 < kN) x[e + 1] = y.y;
    }
  }
};

// Lanes per row: a power of two that holds D / kVec accesses, 32 at most (then several each).
template <class T, class P, int kVec, bool kWrite>
__global__ void __launch_bounds__(kThreads) move_kernel(const __grid_constant__ MoveArgs a, int lanes_log2) {
  constexpr bool kScaled = std::is_same<P, __nv_fp8_e4m3>::value;
  constexpr int kMost = (kVec >= 8 ? 1 : kVec >= 4 ? 2 : 8) * lane_share(kScaled, kVec);   // accesses of one row, D <= 256
  using In = Raw<T, kVec>;
  using Cached = Raw<P, kVec>;
  const int lane = threadIdx.x & ((1 << lanes_log2) - 1);
  const int group = threadIdx.x >> lanes_log2, groups = kThreads >> lanes_log2;
  const int b = blockIdx.x / a.tiles, t0 = (blockIdx.x - b * a.tiles) * a.tokens;
  const int count = a.counts ? max(min(a.counts[b], a.T), 0) : a.T;  // tokens that are moved
  const int here = min(a.tokens, (kWrite ? count : a.T) - t0);       // rows of tokens t0 + [0, here)
  if (here <= 0) return;
  const int64_t start = a.start ? a.start[b] : 0;
  const int* const entries = a.table.entry + b * a.table.stride;
  const int accesses = a.D / kVec, rows = here * a.heads;
  const bool my[2] = {lane < accesses, lane + (1 << lanes_log2) < accesses};
  const auto mine = [&](int i) { return i < 2 ? my[i] : lane + (i << lanes_log2) < accesses; };
  // this lane's piece of the first row
  T* data[2];
#pragma unroll
  for (int w = 0; w < 2; ++w)
    data[w] = static_cast<T*>(a.data[w]) + b * a.batch[w] + t0 * a.token[w] + lane * kVec;
  const int step = kVec << lanes_log2;                               // elements between a lane's accesses
  // (every lane of a warp takes part in every round: the shuffles below need them all)
  for (int row0 = 0; row0 < rows; row0 += groups) {
    const int row = row0 + group;
    const bool live = row < rows;
    const int tt = a.heads == 1 ? row : (int)__umulhi(row, a.heads_magic), h = row - tt * a.heads;
    In x[2][kMost];
    T* at[2];
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      at[w] = data[w] + (!kWrite ? (int64_t)row * a.D
                         : a.narrow ? (int64_t)tt * (int)a.token[w] + (int64_t)h * (int)a.head[w]
                                    : tt * a.token[w] + h * a.head[w]);
      if (kWrite) {
#pragma unroll
        for (int i = 0; i < kMost; ++i) {
          x[w][i] = In{};
          if (live && mine(i)) x[w][i] = *reinterpret_cast<const In*>(at[w] + i * step);
        }
      }
    }
    int page = -1, slot = 0;
    const int64_t p = start + t0 + tt;
    if (live && t0 + tt < count && p >= 0) {
      uint32_t index = (uint32_t)p;                                  // (start and t are 31 bits each)
      if (a.table.shift >= 0) {
        index >>= a.table.shift;
        slot = (uint32_t)p & (a.table.page_size - 1);
      } else {
        index /= (uint32_t)a.table.page_size;
        slot = (uint32_t)p - index * a.table.page_size;
      }
      if (index < (uint32_t)a.table.max_pages) page = entries[index];
      if ((uint32_t)page >= (uint32_t)a.table.pages) page = -1;
    }
    const bool there = page >= 0;
    Cached y[2][kMost];
    float scale[2] = {0.f, 0.f};
    int64_t off[2] = {0, 0}, scale_at[2] = {0, 0};
    P* cached[2];
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const PagedPool& pool = a.pool[w];
      if (w && a.same_strides) {
        off[1] = off[0];
        scale_at[1] = scale_at[0];
      } else if (there) {
        off[w] = pool.at(page, slot) + pool.head_at(h) + lane * kVec;
        if (kScaled) scale_at[w] = pool.scale_at(page, slot) + pool.scale_head_at(h);
      }
      cached[w] = static_cast<P*>(pool.base) + off[w];
      if (!kWrite) {
        if (kScaled && there) scale[w] = pool.scale[scale_at[w]];
#pragma unroll
        for (int i = 0; i < kMost; ++i) {
          y[w][i] = Cached{};
          if (there && mine(i)) y[w][i] = *reinterpret_cast<const Cached*>(cached[w] + i * step);
        }
      }
    }
    if constexpr (kWrite && kScaled) {
      uint32_t most[2] = {0, 0};
#pragma unroll
      for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int i = 0; i < kMost; ++i) most[w] = largest_bits<T, kVec>(x[w][i], most[w]);
      if constexpr (sizeof(T) == 2) {
        // keys in the low half, values in the high one
        uint32_t both = __vmaxu2(__byte_perm(most[0], most[1], 0x5410), __byte_perm(most[0], most[1], 0x7632));
        for (int o = 1; o < 1 << lanes_log2; o <<= 1) both = __vmaxu2(both, __shfl_xor_sync(0xffffffffu, both, o));
        scale[0] = as_float(bits_as<T>((uint16_t)both));
        scale[1] = as_float(bits_as<T>((uint16_t)(both >> 16)));
      } else {
        for (int o = 1; o < 1 << lanes_log2; o <<= 1)
#pragma unroll
          for (int w = 0; w < 2; ++w) most[w] = max(most[w], __shfl_xor_sync(0xffffffffu, most[w], o));
        scale[0] = __int_as_float(most[0]);
        scale[1] = __int_as_float(most[1]);
      }
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        // most / 448, correctly rounded (a product and Markstein's correction by its remainder); a row that
        // is not finite reads back as NaN
        const float m = scale[w], q = m * (1.f / kE4m3Max);
        const float s = fmaxf(__fmaf_rn(__fmaf_rn(-kE4m3Max, q, m), 1.f / kE4m3Max, q), kSmallestScale);
        scale[w] = m < INFINITY ? s : __int_as_float(0x7fc00000);
        if (there && lane == 0) a.pool[w].scale[scale_at[w]] = scale[w];
      }
    }
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const float factor = scale[w];
      const Quotient<T> by(scale[w]);
#pragma unroll
      for (int i = 0; i < kMost; ++i) {
        if constexpr (kWrite) {
          if (!there || !mine(i)) continue;
          if constexpr (kScaled) {
            float f[kVec];
            to_floats<T, kVec>(x[w][i], f);
            by.divide(f);
            y[w][i] = from_floats<P, kVec>(f);
          } else {
            y[w][i] = x[w][i];
          }
          *reinterpret_cast<Cached*>(cached[w] + i * step) = y[w][i];
        } else {
          if (!live || !mine(i)) continue;
          if constexpr (kScaled) {
            x[w][i] = In{};
            if (there) {
              float f[kVec];
              to_floats<P, kVec>(y[w][i], f);
#pragma unroll
              for (int e = 0; e < kVec; ++e) f[e] *= factor;
              x[w][i] = from_floats<T, kVec>(f);
            }
          } else {
            x[w][i] = y[w][i];
          }
          *reinterpret_cast<In*>(at[w] + i * step) = x[w][i];
        }
      }
    }
  }
}

template <class T, class P, bool kWrite>
int launch(MoveArgs a, cudaStream_t stream) {
  constexpr int kWide = 16 / (int)sizeof(T);
  // whole 16-byte accesses where sizes, strides and addresses of both sides allow
  bool wide = a.D % kWide == 0;
  for (int w = 0; w < 2; ++w) {
    const PagedPool& p = a.pool[w];
    wide = wide && reinterpret_cast<uintptr_t>(a.data[w]) % 16 == 0 &&
           reinterpret_cast<uintptr_t>(p.base) % (kWide * sizeof(P)) == 0 &&
           (a.batch[w] | a.token[w] | a.head[w] | p.page | p.token | p.head) % kWide == 0;
  }
  const int accesses = wide ? a.D / kWide : a.D;
  int lanes_log2 = 0;
  constexpr bool kScaled = std::is_same<P, __nv_fp8_e4m3>::value;
  const int share = lane_share(kScaled, wide ? kWide : 1);
  while (lanes_log2 < 5 && (share << lanes_log2) < accesses) ++lanes_log2;
  // Tokens of a block: rounds of its threads' rows, at least one token. More rounds (8 at most) share the wait
  // for the sequence's count and start, as long as every SM keeps eight blocks.
  int sms = 0;
  const int rc = sm_count_of_current_device(&sms);
  if (rc != B200NA_OK) return rc;
  const int64_t round = kThreads >> lanes_log2, all = (int64_t)a.B * a.T * a.heads / round;
  const int64_t rows = round * std::max<int64_t>(1, std::min<int64_t>(8, all / (8 * sms)));
  a.tokens = rows > a.heads ? (int)rows / a.heads : 1;
  a.tiles = (int)(((int64_t)a.T + a.tokens - 1) / a.tokens);
  a.narrow = true;
  for (int w = 0; w < 2; ++w)
    for (int64_t stride : {a.token[w], a.head[w]}) a.narrow = a.narrow && stride >= 0 && stride <= 0x7fffffff;
  a.heads_magic = a.heads == 1 ? 0 : (uint32_t)(((uint64_t)1 << 32) / a.heads) + (((uint64_t)1 << 32) % a.heads != 0);
  a.same_strides = a.pool[0].page == a.pool[1].page && a.pool[0].token == a.pool[1].token &&
                   a.pool[0].head == a.pool[1].head && a.pool[0].s_page == a.pool[1].s_page &&
                   a.pool[0].s_token == a.pool[1].s_token && a.pool[0].s_head == a.pool[1].s_head;
  const int64_t blocks = (int64_t)a.B * a.tiles;
  if (blocks > 0x7fffffff) return B200NA_ERR_INVALID_ARGUMENT;
  if (wide) move_kernel<T, P, kWide, kWrite><<<(unsigned)blocks, kThreads, 0, stream>>>(a, lanes_log2);
  else move_kernel<T, P, 1, kWrite><<<(unsigned)blocks, kThreads, 0, stream>>>(a, lanes_log2);
  B200NA_CUDA_TRY(cudaGetLastError());
  return B200NA_OK;
}

template <bool kWrite>
int dispatch(const MoveArgs& a, int dtype, int cache_dtype, cudaStream_t s) {
  if (cache_dtype == B200NA_E4M3) {
    switch (dtype) {
      case B200NA_F32: return launch<float, __nv_fp8_e4m3, kWrite>(a, s);
      case B200NA_F16: return launch<__half, __nv_fp8_e4m3, kWrite>(a, s);
      default: return launch<__nv_bfloat16, __nv_fp8_e4m3, kWrite>(a, s);
    }
  }
  switch (dtype) {
    case B200NA_F32: return launch<float, float, kWrite>(a, s);
    case B200NA_F16: return launch<__half, __half, kWrite>(a, s);
    default: return launch<__nv_bfloat16, __nv_bfloat16, kWrite>(a, s);
  }
}

int fill(MoveArgs& a, const b200na_kv_cache* cache, int B, int T, int dtype, const int* table,
         int64_t table_stride, int max_pages, const int* start, const int* counts) {
  const int rc = check_cache(cache, table, table_stride, max_pages, dtype, B);
  if (rc != B200NA_OK) return rc;
  if (T < 0) return B200NA_ERR_INVALID_ARGUMENT;
  a.pool[0] = paged_pool(*cache, false);
  a.pool[1] = paged_pool(*cache, true);
  a.table = page_table(*cache, table, table_stride, max_pages);
  a.B = B;
  a.T = T;
  a.heads = cache->heads;
  a.D = cache->head_dim;
  a.start = start;
  a.counts = counts;
  return B200NA_OK;
}

}  // namespace
}  // namespace b200na

extern "C" B200NA_API int b200na_kv_cache_write(const b200na_kv_cache* cache, const void* key, const void* value,
                                                int B, int T, int dtype, const int64_t* key_strides,
                                                const int64_t* value_strides, const int* table,
                                                int64_t table_stride, int max_pages, const int* start,
                                                const int* counts, b200na_stream_t stream) {
  using namespace b200na;
  MoveArgs a{};
  const int rc = fill(a, cache, B, T, dtype, table, table_stride, max_pages, start, counts);
  if (rc != B200NA_OK) return rc;
  if (!key_strides || !value_strides) return B200NA_ERR_INVALID_ARGUMENT;
  if (B == 0 || T == 0 || cache->pages == 0 || max_pages == 0) return B200NA_OK;
  if (!key || !value) return B200NA_ERR_INVALID_ARGUMENT;
  a.data[0] = const_cast<void*>(key);
  a.data[1] = const_cast<void*>(value);
  for (int w = 0; w < 2; ++w) {
    const int64_t* s = w ? value_strides : key_strides;
    a.batch[w] = B > 1 ? s[0] : 0;
    a.token[w] = T > 1 ? s[1] : 0;
    a.head[w] = cache->heads > 1 ? s[2] : 0;
  }
  return dispatch<true>(a, dtype, cache->dtype, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" B200NA_API int b200na_kv_cache_read(const b200na_kv_cache* cache, void* key, void* value, int B,
                                               int length, int dtype, const int* table, int64_t table_stride,
                                               int max_pages, const int* start, const int* counts,
                                               b200na_stream_t stream) {
  using namespace b200na;
  MoveArgs a{};
  const int rc = fill(a, cache, B, length, dtype, table, table_stride, max_pages, start, counts);
  if (rc != B200NA_OK) return rc;
  if (B == 0 || length == 0) return B200NA_OK;
  if (!key || !value) return B200NA_ERR_INVALID_ARGUMENT;
  a.data[0] = key;
  a.data[1] = value;
  for (int w = 0; w < 2; ++w) {
    a.head[w] = cache->head_dim;
    a.token[w] = (int64_t)cache->heads * cache->head_dim;
    a.batch[w] = a.token[w] * length;
  }
  return dispatch<false>(a, dtype, cache->dtype, reinterpret_cast<cudaStream_t>(stream));
}
