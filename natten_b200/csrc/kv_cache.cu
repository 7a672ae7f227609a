// Writing tokens into the paged key/value cache and reading them back, for sm_100a.
//
// Both are streams of rows (one token's channels of one head): a row is read once and written once,
// keys and values in one launch. A group of lanes holds a whole row in registers, 16 bytes a lane and
// access, so the largest magnitude of a row (for its 8-bit scale) is a few shuffles away and the row is
// not read again.
#include <type_traits>

#include "paged.cuh"

namespace b200na {
namespace {

constexpr int kThreads = 256;

struct MoveArgs {
  PagedPool pool[2];             // keys, values
  PageTable table;
  void* data[2];                 // [B, T, heads, D]: given to the write, filled by the read
  int64_t batch[2], token[2], head[2];   // its strides (elements)
  const int* start;
  const int* counts;
  int B, T, heads, D;
};

// Lanes per row: a power of two that holds D / kVec accesses, 32 at most (then several each).
template <class T, class P, int kVec, bool kWrite>
__global__ void __launch_bounds__(kThreads) move_kernel(const __grid_constant__ MoveArgs a, int lanes) {
  constexpr int kMost = kVec >= 8 ? 1 : kVec >= 4 ? 2 : 8;    // accesses a lane makes of one row, D <= 256
  constexpr bool kScaled = std::is_same<P, __nv_fp8_e4m3>::value;
  const int lane = threadIdx.x & (lanes - 1);
  const int64_t per_step = (int64_t)gridDim.x * (kThreads / lanes);
  const int64_t rows = (int64_t)a.B * a.T * a.heads;
  const int accesses = a.D / kVec;
  // (every lane of a warp takes part in every round: the shuffles below need them all)
  const int64_t first = (int64_t)blockIdx.x * (kThreads / lanes) + threadIdx.x / lanes;
  for (int64_t round = first - threadIdx.x / lanes; round < rows; round += per_step) {
    const int64_t row = round + threadIdx.x / lanes;
    bool live = row < rows;
    const int64_t token = live ? row / a.heads : 0;
    const int h = live ? (int)(row - token * a.heads) : 0;
    const int b = (int)(token / a.T), t = (int)(token - (int64_t)b * a.T);
    const bool inside = live && (!a.counts || t < a.counts[b]);
    int64_t page = -1;
    int slot = 0;
    if (inside) {
      const int64_t p = (a.start ? (int64_t)a.start[b] : 0) + t;
      int64_t index;
      if (p >= 0) {
        a.table.split(p, &index, &slot);
        page = a.table.page_of(b, index);
      }
    }
    if (kWrite) live = page >= 0;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const PagedPool& pool = a.pool[w];
      P* cached = static_cast<P*>(pool.base) + page * pool.page + (int64_t)slot * pool.token + h * pool.head;
      T* data = static_cast<T*>(a.data[w]) + b * a.batch[w] + (int64_t)t * a.token[w] + h * a.head[w];
      float* scale_at = kScaled ? pool.scale + page * pool.s_page + (int64_t)slot * pool.s_token + h * pool.s_head
                                : nullptr;
      if (kWrite) {
        Elements<T, kVec> x[kMost];
        float most = 0.f;
#pragma unroll
        for (int i = 0; i < kMost; ++i) {
          const int at = lane + i * lanes;
          if (live && at < accesses) {
            x[i] = *reinterpret_cast<const Elements<T, kVec>*>(data + at * kVec);
            if (kScaled) {
#pragma unroll
              for (int e = 0; e < kVec; ++e) {
                const float m = fabsf(as_float(x[i].v[e]));
                most = fmaxf(most, m < INFINITY ? m : INFINITY);   // infinity also for a NaN
              }
            }
          }
        }
        float inverse = 1.f;
        if (kScaled) {
          for (int o = lanes / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
          // not finite: the whole row reads back as NaN
          const float scale = most < INFINITY ? fmaxf(__fdiv_rn(most, kE4m3Max), kSmallestScale)
                                              : __int_as_float(0x7fc00000);
          inverse = __frcp_rn(scale);
          if (live && lane == 0) *scale_at = scale;
        }
#pragma unroll
        for (int i = 0; i < kMost; ++i) {
          const int at = lane + i * lanes;
          if (live && at < accesses) {
            Elements<P, kVec> y;
#pragma unroll
            for (int e = 0; e < kVec; ++e) {
              if constexpr (kScaled) y.v[e] = from_float<P>(as_float(x[i].v[e]) * inverse);
              else y.v[e] = x[i].v[e];
            }
            *reinterpret_cast<Elements<P, kVec>*>(cached + at * kVec) = y;
          }
        }
      } else {
        const float scale = kScaled && page >= 0 ? *scale_at : 0.f;
#pragma unroll
        for (int i = 0; i < kMost; ++i) {
          const int at = lane + i * lanes;
          if (live && at < accesses) {
            Elements<T, kVec> y;
            if (page >= 0) {
              const Elements<P, kVec> x = *reinterpret_cast<const Elements<P, kVec>*>(cached + at * kVec);
#pragma unroll
              for (int e = 0; e < kVec; ++e) {
                if constexpr (kScaled) y.v[e] = from_float<T>(as_float(x.v[e]) * scale);
                else y.v[e] = x.v[e];
              }
            } else {
#pragma unroll
              for (int e = 0; e < kVec; ++e) y.v[e] = from_float<T>(0.f);
            }
            *reinterpret_cast<Elements<T, kVec>*>(data + at * kVec) = y;
          }
        }
      }
    }
  }
}

template <class T, class P, bool kWrite>
int launch(const MoveArgs& a, cudaStream_t stream) {
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
  int lanes = 1;
  while (lanes < 32 && lanes < accesses) lanes *= 2;
  int sms = 0;
  const int rc = sm_count_of_current_device(&sms);
  if (rc != B200NA_OK) return rc;
  const int64_t rows = (int64_t)a.B * a.T * a.heads, per_block = kThreads / lanes;
  int64_t blocks = (rows + per_block - 1) / per_block;
  if (blocks > (int64_t)sms * 64) blocks = (int64_t)sms * 64;
  if (wide) move_kernel<T, P, kWide, kWrite><<<(unsigned)blocks, kThreads, 0, stream>>>(a, lanes);
  else move_kernel<T, P, 1, kWrite><<<(unsigned)blocks, kThreads, 0, stream>>>(a, lanes);
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
