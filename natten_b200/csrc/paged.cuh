// Addresses and rows of the paged key/value cache (see b200na_kv_cache in the C header), shared by the
// kernels that write it, read it back and attend over it.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cstring>
#include <type_traits>

#include "common.cuh"

namespace b200na {

// e4m3 rows: value * scale. The largest magnitude of a row becomes 448, the type's largest value.
constexpr float kE4m3Max = 448.f;
constexpr float kSmallestScale = 1.17549435e-38f;   // 2^-126: its reciprocal is finite

struct PagedPool {
  void* base;
  float* scale;                 // fp32 per token and head; nullptr when the pool is not 8-bit
  int64_t page, token, head;    // strides in elements
  int64_t s_page, s_token, s_head;
  bool narrow;                  // all of them fit 31 bits: one multiply-add each

  __device__ __forceinline__ int64_t at(int pg, int slot) const {
    if (narrow) return (int64_t)pg * (int)page + (int64_t)slot * (int)token;
    return pg * page + slot * token;
  }
  __device__ __forceinline__ int64_t scale_at(int pg, int slot) const {
    if (narrow) return (int64_t)pg * (int)s_page + (int64_t)slot * (int)s_token;
    return pg * s_page + slot * s_token;
  }
  __device__ __forceinline__ int64_t head_at(int h) const { return narrow ? (int64_t)h * (int)head : h * head; }
  __device__ __forceinline__ int64_t scale_head_at(int h) const { return narrow ? (int64_t)h * (int)s_head : h * s_head; }
};

struct PageTable {
  const int* entry;             // [B, max_pages], rows `stride` entries apart
  int64_t stride;
  int max_pages, page_size, shift;   // shift: log2(page_size), -1 when that is no power of two
  int64_t pages;

  // Page and slot of logical token `p` >= 0 of sequence `b`; page -1 when there is none.
  __device__ __forceinline__ void split(int64_t p, int64_t* index, int* slot) const {
    if (shift >= 0) {
      *index = p >> shift;
      *slot = (int)(p & (page_size - 1));
    } else {
      *index = p / page_size;
      *slot = (int)(p - *index * page_size);
    }
  }
  __device__ __forceinline__ int64_t page_of(int b, int64_t index) const {
    if (index < 0 || index >= max_pages) return -1;
    const int e = entry[b * stride + index];
    return e >= 0 && e < pages ? e : -1;
  }
};

// A stride of an axis of one entry means nothing and is not looked at.
inline PagedPool paged_pool(const b200na_kv_cache& c, bool value) {
  const int64_t* s = value ? c.value_stride : c.key_stride;
  const int64_t* f = value ? c.value_scale_stride : c.key_scale_stride;
  const bool one[3] = {c.pages <= 1, c.page_size <= 1, c.heads <= 1};
  PagedPool p{};
  p.base = value ? c.value : c.key;
  p.page = one[0] ? 0 : s[0];
  p.token = one[1] ? 0 : s[1];
  p.head = one[2] ? 0 : s[2];
  if (c.dtype == B200NA_E4M3) {
    p.scale = value ? c.value_scale : c.key_scale;
    p.s_page = one[0] ? 0 : f[0];
    p.s_token = one[1] ? 0 : f[1];
    p.s_head = one[2] ? 0 : f[2];
  }
  p.narrow = true;
  for (int64_t stride : {p.page, p.token, p.head, p.s_page, p.s_token, p.s_head})
    p.narrow = p.narrow && stride >= 0 && stride <= 0x7fffffff;
  return p;
}

inline PageTable page_table(const b200na_kv_cache& c, const int* table, int64_t stride, int max_pages) {
  PageTable t{table, stride, max_pages, c.page_size, -1, c.pages};
  for (int i = 0; i < 31; ++i)
    if (c.page_size == 1 << i) t.shift = i;
  return t;
}

inline int check_cache(const b200na_kv_cache* c, const int* table, int64_t table_stride, int max_pages,
                       int dtype, int B) {
  if (!c || c->pages < 0 || c->pages > 0x7fffffff || c->page_size < 1 || c->heads < 1 || c->heads > 32768 || c->head_dim < 1 ||
      max_pages < 0 || B < 0 || (B > 1 && table_stride < 0))
    return B200NA_ERR_INVALID_ARGUMENT;
  if (c->head_dim > 256) return B200NA_ERR_UNSUPPORTED;
  if (dtype != B200NA_F32 && dtype != B200NA_F16 && dtype != B200NA_BF16) return B200NA_ERR_UNSUPPORTED;
  if (c->dtype == B200NA_E4M3) {
    if (c->pages > 0 && (!c->key_scale || !c->value_scale)) return B200NA_ERR_INVALID_ARGUMENT;
  } else if (c->dtype != dtype) {
    return B200NA_ERR_INVALID_ARGUMENT;
  }
  if (c->pages > 0 && (!c->key || !c->value)) return B200NA_ERR_INVALID_ARGUMENT;
  // a place before the pool's first one would be taken for one that is not there
  for (bool value : {false, true}) {
    const PagedPool p = paged_pool(*c, value);
    for (int64_t stride : {p.page, p.token, p.head, p.s_page, p.s_token, p.s_head})
      if (stride < 0) return B200NA_ERR_INVALID_ARGUMENT;
  }
  if (B > 0 && max_pages > 0 && !table) return B200NA_ERR_INVALID_ARGUMENT;
  return B200NA_OK;
}

// ---- elements -----------------------------------------------------------------------------------------
__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float as_float(__nv_fp8_e4m3 v) { return static_cast<float>(v); }
template <class T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <> __device__ __forceinline__ __nv_fp8_e4m3 from_float<__nv_fp8_e4m3>(float v) {
  return __nv_fp8_e4m3(v);
}

template <class T, int kN>
struct alignas(sizeof(T) * kN) Elements {
  T v[kN];
};

// The bits of `x` as another type of the same size.
template <class To, class From> __device__ __forceinline__ To bits_as(const From& x) {
  static_assert(sizeof(To) == sizeof(From), "sizes differ");
  To y;
  memcpy(&y, &x, sizeof(To));
  return y;
}

// kBytes as one access.
template <int kBytes> struct RawOf;
template <> struct RawOf<1> { using type = uint8_t; };
template <> struct RawOf<2> { using type = uint16_t; };
template <> struct RawOf<4> { using type = uint32_t; };
template <> struct RawOf<8> { using type = uint2; };
template <> struct RawOf<16> { using type = uint4; };
template <class T, int kN> using Raw = typename RawOf<(int)sizeof(T) * kN>::type;

// kN elements out of their bits and back. 8 bits: two values an instruction.
template <class T, int kN> __device__ __forceinline__ void to_floats(const Raw<T, kN>& bits, float (&y)[kN]) {
  if constexpr (std::is_same<T, __nv_fp8_e4m3>::value && kN % 2 == 0) {
    __nv_fp8x2_storage_t x[kN / 2];
    memcpy(x, &bits, kN);
#pragma unroll
    for (int e = 0; e < kN / 2; ++e) {
      const float2 f = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(x[e], __NV_E4M3)));
      y[2 * e] = f.x;
      y[2 * e + 1] = f.y;
    }
  } else {
    T x[kN];
    memcpy(x, &bits, sizeof(x));
#pragma unroll
    for (int e = 0; e < kN; ++e) y[e] = as_float(x[e]);
  }
}
template <class T, int kN> __device__ __forceinline__ Raw<T, kN> from_floats(const float (&x)[kN]) {
  Raw<T, kN> bits;
  if constexpr (std::is_same<T, __nv_fp8_e4m3>::value && kN % 2 == 0) {
    __nv_fp8x2_storage_t y[kN / 2];
#pragma unroll
    for (int e = 0; e < kN / 2; ++e)
      y[e] = __nv_cvt_float2_to_fp8x2(make_float2(x[2 * e], x[2 * e + 1]), __NV_SATFINITE, __NV_E4M3);
    memcpy(&bits, y, kN);
  } else {
    T y[kN];
#pragma unroll
    for (int e = 0; e < kN; ++e) y[e] = from_float<T>(x[e]);
    memcpy(&bits, y, sizeof(y));
  }
  return bits;
}

}  // namespace b200na
