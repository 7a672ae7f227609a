// Writing tokens into the paged key/value cache and reading them back, for sm_100a.
//
// Both are streams of rows (one token's channels of one head): a row is read once and written once,
// keys and values in one launch. A group of lanes holds a whole row in registers, 16 bytes a lane and
// access, so the largest magnitude of a row (for its 8-bit scale) is a few shuffles away and the row is
// not read again. A block works on consecutive tokens of one sequence, so that a sequence's start and
// count are read once a block and places need 32-bit arithmetic only; a thread has kRows rows in flight.
#include "paged.cuh"

namespace b200na {
namespace {

constexpr int kThreads = 256;
constexpr int kRows = 4;         // rows of keys and of values that a thread has in flight

struct MoveArgs {
  PagedPool pool[2];             // keys, values
  PageTable table;
  void* data[2];                 // [B, T, heads, D]: given to the write, filled by the read
  int64_t batch[2], token[2], head[2];   // its strides (elements)
  const int* start;
  const int* counts;
  int B, T, heads, D;
  int tokens;                    // of a block
  int tiles;                     // blocks of a sequence
};

// Lanes per row: a power of two that holds D / kVec accesses, 32 at most (then several each).
template <class T, class P, int kVec, bool kWrite>
__global__ void __launch_bounds__(kThreads) move_kernel(const __grid_constant__ MoveArgs a, int lanes_log2) {
  constexpr int kMost = kVec >= 8 ? 1 : kVec >= 4 ? 2 : 8;    // accesses a lane makes of one row, D <= 256
  constexpr int kAtOnce = kMost == 8 ? 1 : kRows / (kMost * (int)sizeof(T) * kVec > 16 ? 2 : 1);
  constexpr bool kScaled = std::is_same<P, __nv_fp8_e4m3>::value;
  const int lanes = 1 << lanes_log2, lane = threadIdx.x & (lanes - 1);
  const int group = threadIdx.x >> lanes_log2, groups = kThreads >> lanes_log2;
  const int b = blockIdx.x / a.tiles, t0 = (blockIdx.x - b * a.tiles) * a.tokens;
  const int count = a.counts ? min(a.counts[b], a.T) : a.T;          // tokens that are moved
  const int here = min(a.tokens, (kWrite ? count : a.T) - t0);       // rows of tokens t0 + [0, here)
  if (here <= 0) return;
  const int64_t start = a.start ? a.start[b] : 0;
  const int accesses = a.D / kVec, rows = here * a.heads;
  // (every lane of a warp takes part in every round: the shuffles below need them all)
  for (int row0 = 0; row0 < rows; row0 += groups * kAtOnce) {
    using In = Raw<T, kVec>;
    using Cached = Raw<P, kVec>;
    In x[kAtOnce][2][kMost];
    bool live[kAtOnce];
    int t[kAtOnce], h[kAtOnce];
    int64_t page[kAtOnce];
    int slot[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const int row = row0 + u * groups + group;
      live[u] = row < rows;
      const int tt = live[u] ? (int)((uint32_t)row / (uint32_t)a.heads) : 0;
      h[u] = live[u] ? row - tt * a.heads : 0;
      t[u] = t0 + tt;
    }
    if (kWrite) {
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u)
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const T* data = static_cast<const T*>(a.data[w]) + b * a.batch[w] + t[u] * a.token[w] + h[u] * a.head[w];
#pragma unroll
          for (int i = 0; i < kMost; ++i)
            if (live[u] && lane + (i << lanes_log2) < accesses)
              x[u][w][i] = *reinterpret_cast<const In*>(data + (lane + (i << lanes_log2)) * kVec);
        }
    }
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      page[u] = -1;
      slot[u] = 0;
      const int64_t p = start + t[u];
      if (live[u] && t[u] < count && p >= 0) {
        int64_t index;
        a.table.split(p, &index, &slot[u]);
        page[u] = a.table.page_of(b, index);
      }
    }
    if (kWrite) {
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        const bool to = page[u] >= 0;
        float inverse[2] = {1.f, 1.f};
        if constexpr (kScaled) {
          float most[2] = {0.f, 0.f};
#pragma unroll
          for (int w = 0; w < 2; ++w)
#pragma unroll
            for (int i = 0; i < kMost; ++i)
              if (live[u] && lane + (i << lanes_log2) < accesses) {
                float f[kVec];
                to_floats<T, kVec>(x[u][w][i], f);
#pragma unroll
                for (int e = 0; e < kVec; ++e) {
                  const float m = fabsf(f[e]);
                  most[w] = fmaxf(most[w], m < INFINITY ? m : INFINITY);   // infinity also for a NaN
                }
              }
          for (int o = lanes / 2; o > 0; o >>= 1)
#pragma unroll
            for (int w = 0; w < 2; ++w) most[w] = fmaxf(most[w], __shfl_xor_sync(0xffffffffu, most[w], o));
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            // not finite: the whole row reads back as NaN
            const float scale = most[w] < INFINITY ? fmaxf(__fdiv_rn(most[w], kE4m3Max), kSmallestScale)
                                                   : __int_as_float(0x7fc00000);
            inverse[w] = __frcp_rn(scale);
            const PagedPool& pool = a.pool[w];
            if (to && lane == 0)
              pool.scale[page[u] * pool.s_page + slot[u] * pool.s_token + h[u] * pool.s_head] = scale;
          }
        }
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const PagedPool& pool = a.pool[w];
          P* const cached = static_cast<P*>(pool.base) + (to ? page[u] * pool.page + slot[u] * pool.token + h[u] * pool.head : 0);
#pragma unroll
          for (int i = 0; i < kMost; ++i)
            if (to && lane + (i << lanes_log2) < accesses) {
              Cached y;
              if constexpr (kScaled) {
                float f[kVec];
                to_floats<T, kVec>(x[u][w][i], f);
#pragma unroll
                for (int e = 0; e < kVec; ++e) f[e] *= inverse[w];
                y = from_floats<P, kVec>(f);
              } else {
                y = x[u][w][i];
              }
              *reinterpret_cast<Cached*>(cached + (lane + (i << lanes_log2)) * kVec) = y;
            }
        }
      }
    } else {
      Cached y[kAtOnce][2][kMost];
      float scale[kAtOnce][2];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u)
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const PagedPool& pool = a.pool[w];
          const bool from = page[u] >= 0;
          scale[u][w] = 0.f;
          if (kScaled && from)
            scale[u][w] = pool.scale[page[u] * pool.s_page + slot[u] * pool.s_token + h[u] * pool.s_head];
          const P* const cached = static_cast<const P*>(pool.base) + (from ? page[u] * pool.page + slot[u] * pool.token + h[u] * pool.head : 0);
#pragma unroll
          for (int i = 0; i < kMost; ++i) {
            y[u][w][i] = Cached{};
            if (from && lane + (i << lanes_log2) < accesses)
              y[u][w][i] = *reinterpret_cast<const Cached*>(cached + (lane + (i << lanes_log2)) * kVec);
          }
        }
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u)
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          T* const data = static_cast<T*>(a.data[w]) + b * a.batch[w] + t[u] * a.token[w] + h[u] * a.head[w];
#pragma unroll
          for (int i = 0; i < kMost; ++i)
            if (live[u] && lane + (i << lanes_log2) < accesses) {
              if constexpr (kScaled) {
                float f[kVec];
                to_floats<P, kVec>(y[u][w][i], f);
#pragma unroll
                for (int e = 0; e < kVec; ++e) f[e] *= scale[u][w];
                x[u][w][i] = from_floats<T, kVec>(f);
              } else {
                x[u][w][i] = y[u][w][i];
              }
              *reinterpret_cast<In*>(data + (lane + (i << lanes_log2)) * kVec) = x[u][w][i];
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
  while (lanes_log2 < 5 && (1 << lanes_log2) < accesses) ++lanes_log2;
  // tokens of a block: one round of its threads' rows, at least one token
  const int rows = (kThreads >> lanes_log2) * kRows;
  a.tokens = rows > a.heads ? rows / a.heads : 1;
  a.tiles = (a.T + a.tokens - 1) / a.tokens;
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
