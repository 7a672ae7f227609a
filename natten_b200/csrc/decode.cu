// Attention of the newest tokens of every sequence over a paged key/value cache (causal 1-D neighborhood
// attention, stride 1, as serving needs it) for sm_100a.
//
//   s_j = scale * q . k_j,   out = sum_j exp(s_j - m) v_j / l,   m = max_j s_j,   l = sum_j exp(s_j - m)
//
// over the attended tokens j of one query row. Every attended key and value row is read once for all query
// heads that share it and does about two products a byte and row: the memory's rate bounds it, so what
// counts is that all SMs read all the time, whatever the sequences' lengths are.
//
// Work: an item is one sequence, one key/value head and up to 16 (CUDA cores: 8) rows, which are the heads
// of the group times neighbouring query tokens. Its keys are cut into units of 64. The units of all items
// in a row are cut into as many equal ranges as there are blocks; lengths are read on the device, so the
// host waits for nothing and a captured launch follows them. A block keeps the running maximum and sum of
// each row over its range of an item and either writes the result (it had the whole item) or leaves a part
// (at most two per block: the end of one item and the beginning of another). The second launch joins parts.
#include <type_traits>

#include "paged.cuh"

namespace b200na {
namespace {

constexpr int kThreads = 128, kWarps = kThreads / 32;
constexpr int kUnit = 64;             // keys of a unit of work
constexpr int kMostParts = 2 * 148;   // blocks of the first launch: two per SM
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct DecodeArgs {
  const void* query;
  int64_t q_batch, q_token, q_head;
  void* out;
  float* lse;
  PagedPool key, value;
  PageTable table;
  const int* lengths;
  int64_t capacity;                   // tokens that a row of the table can name
  int B, T, Hq, heads, group, D;      // heads: of keys and values; group: query heads of each
  int64_t window;                     // tokens attended at most
  int dilation;
  float scale_log2;
  int item_tokens, item_heads;        // query tokens and heads of an item: its rows
  int token_blocks, head_blocks;
  int64_t items;                      // of one sequence
  int parts;
  int2* covered;                      // [B * items]: first block that worked on the item, how many
  float2* part_ml;                    // [2 * parts][rows]: maximum (of scale_log2 * q.k) and sum
  float* part_o;                      // [2 * parts][rows][D]
};

// What the blocks of a launch agree on: the units of a sequence (the same for each of its items).
__device__ __forceinline__ int64_t units_of(const DecodeArgs& a, int length) {
  int64_t n = length < 0 ? 0 : length;
  if (a.dilation > 1) n = n > 0 ? (n - 1) / a.dilation + 1 : 0;
  const int64_t widest = a.window + (a.dilation > 1 ? 0 : a.item_tokens - 1);
  n = n < a.capacity ? n : a.capacity;
  n = n < widest ? n : widest;
  return n > 0 ? (n + kUnit - 1) / kUnit : 1;   // an item without keys still has its rows written
}

struct Item {
  int64_t index;         // among the sequence's
  int b, head, t0, tokens, h0, heads;
  int64_t p0;            // position of token t0
  int64_t first, n;      // keys at first + dilation * i, i < n
};

__device__ __forceinline__ Item item_of(const DecodeArgs& a, int b, int64_t index, int length) {
  Item it;
  it.index = index;
  it.b = b;
  const int hb = (int)(index % a.head_blocks);
  const int64_t rest = index / a.head_blocks;
  const int tb = (int)(rest % a.token_blocks);
  it.head = (int)(rest / a.token_blocks);
  it.t0 = tb * a.item_tokens;
  it.tokens = min(a.item_tokens, a.T - it.t0);
  it.h0 = hb * a.item_heads;
  it.heads = min(a.item_heads, a.group - it.h0);
  const int64_t len = length < 0 ? 0 : length;
  it.p0 = len - a.T + it.t0;
  const int64_t last = it.p0 + it.tokens - 1;
  it.first = 0;
  it.n = 0;
  if (last < 0) return it;
  if (a.dilation > 1) {                       // one token an item
    int64_t count = last / a.dilation + 1;
    count = count < a.window ? count : a.window;
    it.first = last - (count - 1) * a.dilation;
    const int64_t there = it.first < a.capacity ? (a.capacity - 1 - it.first) / a.dilation + 1 : 0;
    it.n = count < there ? count : there;
  } else {
    const int64_t from = (it.p0 > 0 ? it.p0 : 0) - a.window + 1;
    it.first = from > 0 ? from : 0;
    const int64_t end = (last < a.capacity ? last : a.capacity - 1) + 1;
    it.n = end > it.first ? end - it.first : 0;
  }
  return it;
}

__device__ __forceinline__ int64_t range_begin(int64_t units, int part, int parts) {
  return units * part / parts;
}

// The block's range of units and the sequence in which it begins. With fewer units than blocks the last
// blocks have nothing to do: a block between an item's first and last one always has a unit of it.
struct Range {
  int64_t begin, end, total;
  int parts;
  int b;                 // sequence of `begin`
  int64_t before;        // units of all sequences before it
};
__device__ Range my_range(const DecodeArgs& a) {
  __shared__ int64_t sums[kWarps];
  __shared__ int64_t found_before;
  __shared__ int found_b;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t total = 0;
  for (int b = threadIdx.x; b < a.B; b += kThreads) total += units_of(a, a.lengths[b]) * a.items;
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  if (lane == 0) sums[warp] = total;
  __syncthreads();
  Range r;
  r.total = 0;
  for (int w = 0; w < kWarps; ++w) r.total += sums[w];
  r.parts = (int)(r.total < a.parts ? r.total : a.parts);
  r.begin = r.end = r.b = 0;
  r.before = 0;
  if ((int)blockIdx.x >= r.parts) return r;
  r.begin = range_begin(r.total, blockIdx.x, r.parts);
  r.end = range_begin(r.total, blockIdx.x + 1, r.parts);
  int64_t before = 0;
  for (int b0 = 0; b0 < a.B; b0 += kThreads) {
    __syncthreads();
    const int b = b0 + threadIdx.x;
    const int64_t mine = b < a.B ? units_of(a, a.lengths[b]) * a.items : 0;
    int64_t incl = mine;
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += x;
    }
    if (lane == 31) sums[warp] = incl;
    __syncthreads();
    int64_t base = before, chunk = 0;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) base += sums[w];
      chunk += sums[w];
    }
    const int64_t lo = base + incl - mine;
    if (lo <= r.begin && r.begin < lo + mine) {
      found_b = b;
      found_before = lo;
    }
    before += chunk;
    if (r.begin < before) break;              // (the same for every thread)
  }
  __syncthreads();
  r.b = found_b;
  r.before = found_before;
  return r;
}

// How a segment (the block's part of an item) leaves: whole, or as part 0 (the item began in an earlier
// block) or 1 of the block. The block that has the item's first unit notes which blocks the join has to
// look at.
__device__ __forceinline__ int part_of(const DecodeArgs& a, const Range& r, int64_t item_begin,
                                       int64_t item_end, int64_t item_id) {
  if (item_begin >= r.begin && threadIdx.x == 0) {
    int last = blockIdx.x;
    if (item_end > r.end) {
      last = (int)((item_end - 1) * r.parts / r.total);
      while (range_begin(r.total, last + 1, r.parts) < item_end) ++last;
      while (range_begin(r.total, last, r.parts) >= item_end) --last;
    }
    a.covered[item_id] = make_int2(blockIdx.x, last - blockIdx.x + 1);
  }
  if (item_begin >= r.begin && item_end <= r.end) return -1;
  return item_begin < r.begin ? 0 : 1;
}

// Merges the warps' maxima, sums and outputs of the item's rows and writes them out. `o` holds the warps'
// unnormalised outputs [kWarps][rows_max][D], ml their (maximum, sum) [kWarps][rows_max].
template <class T>
__device__ __forceinline__ void leave(const DecodeArgs& a, const Item& it, int part, const float* o,
                                      const float2* ml, int rows_max) {
  const int rows = it.tokens * it.heads;
  for (int i = threadIdx.x; i < rows * a.D; i += kThreads) {
    const int row = i / a.D, d = i - row * a.D;
    float m = -INFINITY, l = 0.f, x = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) m = fmaxf(m, ml[w * rows_max + row].x);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float2 p = ml[w * rows_max + row];
      if (p.x == -INFINITY) continue;         // the warp met no key of this row
      const float f = exp2f(p.x - m);
      l += f * p.y;
      x += f * o[(w * rows_max + row) * a.D + d];
    }
    if (part < 0) {
      const int t = it.t0 + row / it.heads, h = it.head * a.group + it.h0 + row % it.heads;
      const int64_t at = ((int64_t)it.b * a.T + t) * a.Hq + h;
      static_cast<T*>(a.out)[at * a.D + d] = from_float<T>(m == -INFINITY ? 0.f : x / l);
      if (d == 0 && a.lse) a.lse[at] = m == -INFINITY ? -INFINITY : (m + log2f(l)) * kLn2;
    } else {
      const int64_t slot = (int64_t)(2 * blockIdx.x + part) * rows_max + row;
      a.part_o[slot * a.D + d] = x;
      if (d == 0) a.part_ml[slot] = make_float2(m, l);
    }
  }
}

// ---- CUDA cores: fp32, and layouts that 16-byte copies cannot read -------------------------------------
// A lane takes a key of a 32-key tile for the products with the queries, and every 32nd channel for the
// products with the values.
template <class T, class P, int kRows, int kD32, bool kWide>
__global__ void __launch_bounds__(kThreads) decode_simt_kernel(const __grid_constant__ DecodeArgs a) {
  constexpr bool kScaled = std::is_same<P, __nv_fp8_e4m3>::value;
  constexpr int kVec = kWide ? 16 / (int)sizeof(P) : 1;
  extern __shared__ float smem[];
  float* q = smem;                                      // [kRows][D]
  float* o = smem + kRows * a.D;                        // [kWarps][kRows][D]
  __shared__ float2 ml[kWarps * kRows];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Range r = my_range(a);
  int b = r.b;
  int64_t before = r.before;
  for (int64_t at = r.begin; at < r.end;) {
    const int length = a.lengths[b];
    const int64_t units = units_of(a, length);
    const int64_t index = (at - before) / units;
    if (index >= a.items) {
      before += units * a.items;
      ++b;
      continue;
    }
    const Item it = item_of(a, b, index, length);
    const int64_t item_begin = before + index * units, item_end = item_begin + units;
    const int64_t stop = item_end < r.end ? item_end : r.end;
    const int rows = it.tokens * it.heads;
    __syncthreads();                                    // (the last segment's buffers are read)
    for (int i = threadIdx.x; i < kRows * a.D; i += kThreads) {
      const int row = i / a.D, d = i - row * a.D;
      float x = 0.f;
      if (row < rows) {
        const int t = it.t0 + row / it.heads, h = it.head * a.group + it.h0 + row % it.heads;
        x = as_float(static_cast<const T*>(a.query)[b * a.q_batch + t * a.q_token + h * a.q_head + d]);
      }
      q[i] = x;
    }
    __syncthreads();
    float acc[kRows][kD32], m[kRows], l[kRows];
#pragma unroll
    for (int x = 0; x < kRows; ++x) {
      m[x] = -INFINITY;
      l[x] = 0.f;
#pragma unroll
      for (int e = 0; e < kD32; ++e) acc[x][e] = 0.f;
    }
    const int64_t begin = (at - item_begin) * kUnit;
    const int64_t end = min((stop - item_begin) * kUnit, it.n);
    for (int64_t i0 = begin + warp * 32; i0 < end; i0 += kWarps * 32) {
      const int64_t i = i0 + lane, j = it.first + i * a.dilation;
      int64_t page = -1;
      int slot = 0;
      if (i < end) {
        int64_t pi;
        a.table.split(j, &pi, &slot);
        page = a.table.page_of(b, pi);
      }
      const bool there = page >= 0;
      const P* k = static_cast<const P*>(a.key.base);
      int64_t v_at = 0;
      float k_scale = 1.f, v_scale = 1.f;
      if (there) {
        k += page * a.key.page + (int64_t)slot * a.key.token + it.head * a.key.head;
        v_at = page * a.value.page + (int64_t)slot * a.value.token + it.head * a.value.head;
        if (kScaled) {
          k_scale = a.key.scale[page * a.key.s_page + (int64_t)slot * a.key.s_token + it.head * a.key.s_head];
          v_scale = a.value.scale[page * a.value.s_page + (int64_t)slot * a.value.s_token + it.head * a.value.s_head];
        }
      }
      float s[kRows];
#pragma unroll
      for (int x = 0; x < kRows; ++x) s[x] = 0.f;
      if (there)
        for (int d = 0; d < a.D; d += kVec) {
          const Elements<P, kVec> kk = *reinterpret_cast<const Elements<P, kVec>*>(k + d);
#pragma unroll
          for (int e = 0; e < kVec; ++e)
#pragma unroll
            for (int x = 0; x < kRows; ++x) s[x] += as_float(kk.v[e]) * q[x * a.D + d + e];
        }
      uint32_t seen[kRows];
#pragma unroll
      for (int x = 0; x < kRows; ++x) {
        const int64_t p = it.p0 + (x < rows ? x / it.heads : 0);
        const bool on = there && x < rows && (a.dilation > 1 || (j <= p && j > p - a.window));
        seen[x] = __ballot_sync(0xffffffffu, on);
        s[x] = on ? s[x] * k_scale * a.scale_log2 : -INFINITY;
        float top = s[x];
        for (int f = 16; f > 0; f >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, f));
        const float next = fmaxf(m[x], top);
        // nothing seen yet: no difference of infinities. (A NaN logit is passed over by the maximum and
        // comes back in the exponential.)
        const float base = next == -INFINITY ? 0.f : next;
        const float keep = exp2f(m[x] - base);
        s[x] = on ? exp2f(s[x] - base) : 0.f;
        float sum = s[x];
        for (int f = 16; f > 0; f >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, f);
        l[x] = l[x] * keep + sum;
        m[x] = (seen[x] && next == -INFINITY && sum != sum) ? 0.f : next;   // only NaN logits: they count
#pragma unroll
        for (int e = 0; e < kD32; ++e) acc[x][e] *= keep;
        s[x] *= v_scale;
      }
      const int count = (int)min((int64_t)32, end - i0);
      for (int key = 0; key < count; ++key) {
        const int64_t off = __shfl_sync(0xffffffffu, v_at, key);
        const bool has = __shfl_sync(0xffffffffu, (int)there, key);
        if (!has) continue;
        const P* v = static_cast<const P*>(a.value.base) + off;
        float vv[kD32];
#pragma unroll
        for (int e = 0; e < kD32; ++e) vv[e] = lane + 32 * e < a.D ? as_float(v[lane + 32 * e]) : 0.f;
#pragma unroll
        for (int x = 0; x < kRows; ++x) {
          const float p = __shfl_sync(0xffffffffu, s[x], key);
          // a NaN or an infinity stays with the rows that attend its token
          if (seen[x] >> key & 1)
#pragma unroll
            for (int e = 0; e < kD32; ++e) acc[x][e] += p * vv[e];
        }
      }
    }
#pragma unroll
    for (int x = 0; x < kRows; ++x) {
      if (lane == 0) ml[warp * kRows + x] = make_float2(m[x], l[x]);
#pragma unroll
      for (int e = 0; e < kD32; ++e)
        if (lane + 32 * e < a.D) o[(warp * kRows + x) * a.D + lane + 32 * e] = acc[x][e];
    }
    __syncthreads();
    const int part = part_of(a, r, item_begin, item_end, (int64_t)b * a.items + index);
    leave<T>(a, it, part, o, ml, kRows);
    at = stop;
  }
}

// ---- the join --------------------------------------------------------------------------------------------
// A warp per row of an item; items that one block had are done.
template <class T>
__global__ void __launch_bounds__(kThreads) decode_join_kernel(const __grid_constant__ DecodeArgs a,
                                                               int rows_max) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31;
  const int64_t id = ((int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5)) / rows_max;
  const int row = (int)(((int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5)) - id * rows_max);
  if (id >= a.B * a.items) return;
  const int2 covered = a.covered[id];
  if (covered.y <= 1) return;
  const int b = (int)(id / a.items);
  const Item it = item_of(a, b, id - b * a.items, a.lengths[b]);
  if (row >= it.tokens * it.heads) return;
  // the first block's part is its second one (the item began there), the others' their first
  const auto slot = [&](int i) {
    return (int64_t)(2 * (covered.x + i) + (i == 0 ? 1 : 0)) * rows_max + row;
  };
  float m = -INFINITY;
  for (int i = lane; i < covered.y; i += 32) m = fmaxf(m, a.part_ml[slot(i)].x);
  for (int f = 16; f > 0; f >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, f));
  float l = 0.f, acc[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] = 0.f;
  for (int i = 0; i < covered.y; ++i) {
    const float2 p = a.part_ml[slot(i)];
    if (p.x == -INFINITY) continue;
    const float f = exp2f(p.x - m);
    l += f * p.y;
    const float* o = a.part_o + slot(i) * a.D;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (lane + 32 * e < a.D) acc[e] += f * o[lane + 32 * e];
  }
  const int t = it.t0 + row / it.heads, h = it.head * a.group + it.h0 + row % it.heads;
  const int64_t at = ((int64_t)b * a.T + t) * a.Hq + h;
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (lane + 32 * e < a.D)
      static_cast<T*>(a.out)[at * a.D + lane + 32 * e] = from_float<T>(m == -INFINITY ? 0.f : acc[e] / l);
  if (lane == 0 && a.lse) a.lse[at] = m == -INFINITY ? -INFINITY : (m + log2f(l)) * kLn2;
}

// ---- host --------------------------------------------------------------------------------------------------

struct Plan {
  int rows_max;             // rows of an item
  int item_tokens, item_heads, token_blocks, head_blocks, parts;
  int64_t items;
  int64_t covered_bytes, ml_bytes, o_bytes;
};

int64_t round_up(int64_t n) { return (n + 255) / 256 * 256; }

int make_plan(Plan* p, int B, int T, int Hq, const b200na_kv_cache* cache, int max_pages, int kernel,
              int dilation, int dtype) {
  const int rc = check_cache(cache, reinterpret_cast<const int*>(16), 0, max_pages, dtype, B);
  if (rc != B200NA_OK) return rc;
  if (T < 0 || Hq < 1 || Hq % cache->heads || Hq > 65536 || kernel < 0 || dilation < 1)
    return B200NA_ERR_INVALID_ARGUMENT;
  const int group = Hq / cache->heads;
  p->rows_max = group == 1 && (T <= 1 || dilation > 1) ? 1 : 8;
  p->item_heads = group < p->rows_max ? group : p->rows_max;
  p->head_blocks = (group + p->item_heads - 1) / p->item_heads;
  p->item_tokens = dilation > 1 ? 1 : p->rows_max / p->item_heads;
  if (p->item_tokens > T) p->item_tokens = T < 1 ? 1 : T;
  p->token_blocks = (T + p->item_tokens - 1) / p->item_tokens;
  p->items = (int64_t)cache->heads * p->token_blocks * p->head_blocks;
  if (B > 0 && p->items > ((int64_t)1 << 31) / B) return B200NA_ERR_INVALID_ARGUMENT;
  // units if every sequence were as long as the table allows
  int64_t most = (int64_t)max_pages * cache->page_size;
  if (kernel > 0 && most > (int64_t)kernel + p->item_tokens) most = (int64_t)kernel + p->item_tokens;
  const int64_t units = B * p->items * (most / kUnit + 1);
  if (most / kUnit + 1 > ((int64_t)1 << 52) / (B * p->items + 1)) return B200NA_ERR_INVALID_ARGUMENT;
  p->parts = (int)(units < kMostParts ? (units < 1 ? 1 : units) : kMostParts);
  p->covered_bytes = round_up(B * p->items * (int64_t)sizeof(int2));
  p->ml_bytes = round_up((int64_t)2 * p->parts * p->rows_max * sizeof(float2));
  p->o_bytes = round_up((int64_t)2 * p->parts * p->rows_max * cache->head_dim * sizeof(float));
  return B200NA_OK;
}

template <class K>
int opt_in(K kernel, size_t bytes) {
  if (bytes > 48 * 1024)
    B200NA_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
  return B200NA_OK;
}

template <class T, class P, int kRows, int kD32, bool kWide>
int launch_simt(const DecodeArgs& a, cudaStream_t s) {
  const size_t smem = (size_t)(1 + kWarps) * kRows * a.D * sizeof(float);
  const int rc = opt_in(decode_simt_kernel<T, P, kRows, kD32, kWide>, smem);
  if (rc != B200NA_OK) return rc;
  decode_simt_kernel<T, P, kRows, kD32, kWide><<<a.parts, kThreads, smem, s>>>(a);
  B200NA_CUDA_TRY(cudaGetLastError());
  return B200NA_OK;
}

template <class T, class P>
int run_simt(const DecodeArgs& a, int rows_max, cudaStream_t s) {
  constexpr int kVec = 16 / (int)sizeof(P);
  if constexpr (std::is_same<T, float>::value) {
    const bool wide = a.D % kVec == 0 && reinterpret_cast<uintptr_t>(a.key.base) % 16 == 0 &&
                      (a.key.page | a.key.token | a.key.head) % kVec == 0;
    if (wide) {
      if (rows_max == 1) return a.D <= 128 ? launch_simt<T, P, 1, 4, true>(a, s) : launch_simt<T, P, 1, 8, true>(a, s);
      return a.D <= 128 ? launch_simt<T, P, 8, 4, true>(a, s) : launch_simt<T, P, 8, 8, true>(a, s);
    }
  }
  if (rows_max == 1) return a.D <= 128 ? launch_simt<T, P, 1, 4, false>(a, s) : launch_simt<T, P, 1, 8, false>(a, s);
  return a.D <= 128 ? launch_simt<T, P, 8, 4, false>(a, s) : launch_simt<T, P, 8, 8, false>(a, s);
}

template <class T>
int run(const DecodeArgs& a, int cache_dtype, int rows_max, cudaStream_t s) {
  int rc = cache_dtype == B200NA_E4M3 ? run_simt<T, __nv_fp8_e4m3>(a, rows_max, s) : run_simt<T, T>(a, rows_max, s);
  if (rc != B200NA_OK) return rc;
  // The join's blocks may take their places while the first launch's last ones run (they wait for its end
  // before they read anything).
  cudaLaunchConfig_t cfg{};
  const int64_t warps = a.B * a.items * rows_max;
  const int64_t blocks = (warps + kWarps - 1) / kWarps;
  if (blocks > 0x7fffffff) return B200NA_ERR_INVALID_ARGUMENT;
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  B200NA_CUDA_TRY(cudaLaunchKernelEx(&cfg, decode_join_kernel<T>, a, rows_max));
  return B200NA_OK;
}

}  // namespace
}  // namespace b200na

extern "C" B200NA_API int64_t b200na_na1d_decode_workspace(int B, int T, int Hq, const b200na_kv_cache* cache,
                                                           int max_pages, int kernel, int dilation, int dtype) {
  b200na::Plan p;
  const int rc = b200na::make_plan(&p, B, T, Hq, cache, max_pages, kernel, dilation, dtype);
  return rc != B200NA_OK ? rc : p.covered_bytes + p.ml_bytes + p.o_bytes;
}

extern "C" B200NA_API int b200na_na1d_decode(const void* query, const int64_t* query_strides,
                                             const b200na_kv_cache* cache, void* out, float* lse, int B, int T,
                                             int Hq, int dtype, const int* table, int64_t table_stride,
                                             int max_pages, const int* lengths, int kernel, int dilation,
                                             float scale, void* workspace, b200na_stream_t stream) {
  using namespace b200na;
  Plan p;
  int rc = make_plan(&p, B, T, Hq, cache, max_pages, kernel, dilation, dtype);
  if (rc != B200NA_OK) return rc;
  rc = check_cache(cache, table, table_stride, max_pages, dtype, B);
  if (rc != B200NA_OK) return rc;
  if (!query_strides || !(scale > 0.f) || !(scale < INFINITY)) return B200NA_ERR_INVALID_ARGUMENT;
  if (B == 0 || T == 0) return B200NA_OK;
  if (!query || !out || !lengths || !workspace) return B200NA_ERR_INVALID_ARGUMENT;
  if (reinterpret_cast<uintptr_t>(workspace) % 16) return B200NA_ERR_ALIGNMENT;
  DecodeArgs a{};
  a.query = query;
  a.q_batch = B > 1 ? query_strides[0] : 0;
  a.q_token = T > 1 ? query_strides[1] : 0;
  a.q_head = Hq > 1 ? query_strides[2] : 0;
  a.out = out;
  a.lse = lse;
  a.key = paged_pool(*cache, false);
  a.value = paged_pool(*cache, true);
  a.table = page_table(*cache, table, table_stride, max_pages);
  a.lengths = lengths;
  a.capacity = (int64_t)max_pages * cache->page_size;
  a.B = B;
  a.T = T;
  a.Hq = Hq;
  a.heads = cache->heads;
  a.group = Hq / cache->heads;
  a.D = cache->head_dim;
  a.window = kernel > 0 ? kernel : 0x7fffffff;
  a.dilation = dilation;
  a.scale_log2 = scale * kLog2e;
  a.item_tokens = p.item_tokens;
  a.item_heads = p.item_heads;
  a.token_blocks = p.token_blocks;
  a.head_blocks = p.head_blocks;
  a.items = p.items;
  a.parts = p.parts;
  uint8_t* w = static_cast<uint8_t*>(workspace);
  a.covered = reinterpret_cast<int2*>(w);
  a.part_ml = reinterpret_cast<float2*>(w + p.covered_bytes);
  a.part_o = reinterpret_cast<float*>(w + p.covered_bytes + p.ml_bytes);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  switch (dtype) {
    case B200NA_F32: return run<float>(a, cache->dtype, p.rows_max, s);
    case B200NA_F16: return run<__half>(a, cache->dtype, p.rows_max, s);
    default: return run<__nv_bfloat16>(a, cache->dtype, p.rows_max, s);
  }
}
