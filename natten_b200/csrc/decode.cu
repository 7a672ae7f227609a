// Attention of the newest tokens of every sequence over a paged key/value cache (causal 1-D neighborhood
// attention, stride 1, as serving needs it) for sm_100a.
//
//   s_j = scale * q . k_j,   out = sum_j exp(s_j - m) v_j / l,   m = max_j s_j,   l = sum_j exp(s_j - m)
//
// over the attended tokens j of one query row. An attended key or value row is read once for the rows of an item
// (below: up to 16), and again, mostly out of L2, where the query heads that share it times the new tokens are more.
// It does about two products a byte and row: the memory's rate bounds it, so what counts is that all SMs read
// all the time, whatever the sequences' lengths are.
//
// Work: an item is one sequence, one key/value head and up to 16 (fp32 and CUDA cores: 8) rows, which are the heads
// of the group times neighbouring query tokens. Its keys are cut into units, a tile for each warp of a block.
// Lengths are read on the device, so the host waits for nothing and a captured launch follows them.
//  - Few units at most (a window, a short table): a cluster of 1, 2, 4 or 8 blocks has an item, and joins its
//    parts through distributed shared memory. One launch and no scratch.
//  - Otherwise the units of all items in a row are cut into as many equal ranges as there are blocks on the GPU,
//    whatever the sequences' lengths are. A block keeps the running maximum and sum of each row over its range
//    of an item and either writes the result (it had the whole item) or leaves a part in scratch (at most two
//    per block: the end of one item and the beginning of another). A second launch joins the parts.
#include <type_traits>

#include "paged.cuh"

namespace b200na {
namespace {

constexpr int kThreads = 128, kWarps = kThreads / 32;
constexpr int kMostParts = 2 * 148;   // blocks that the GPU holds: two per SM
constexpr int kClusterUnits = 40;     // units of an item that a block of a cluster takes at most (see make_plan)
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct DecodeArgs {
  const void* query;
  int64_t q_batch, q_token, q_head;
  bool q_wide;                        // query rows lie on 16 bytes
  void* out;
  float* lse;
  PagedPool key, value;
  bool same_strides;                  // of the pools of keys and values
  PageTable table;
  const int* lengths;
  int capacity;                       // tokens that a row of the table can name
  int B, T, Hq, heads, group, D;      // heads: of keys and values; group: query heads of each
  int64_t window;                     // tokens attended at most
  int dilation;
  float scale_log2;
  int item_tokens, item_heads;        // query tokens and heads of an item: its rows
  int token_blocks, head_blocks;
  uint32_t items;                     // of one sequence
  int cluster, cluster_log2;          // blocks that share an item; 0: ranges over all items, and the join
  int parts;                          // blocks of those ranges
  int step;                           // keys that the warps of a block take at once: a tile each
  int unit, unit_log2;                // keys of a unit of work, `step` times a power of two
  int2* covered;                      // [B * items]: first block that worked on the item, how many
  float2* part_ml;                    // [2 * parts][rows]: maximum (of scale_log2 * q.k) and sum
  float* part_o;                      // [2 * parts][rows][D]
};

// What the blocks of a launch agree on: the units of a sequence (the same for each of its items). (The host
// has seen to it that the units of all items together fit 31 bits.)
__device__ __forceinline__ uint32_t units_of(const DecodeArgs& a, int length) {
  int n = length < 0 ? 0 : length;
  if (a.dilation > 1) n = n > 0 ? (n - 1) / a.dilation + 1 : 0;
  const int64_t widest = a.window + (a.dilation > 1 ? 0 : a.item_tokens - 1);
  n = n < a.capacity ? n : a.capacity;
  n = n < widest ? n : (int)widest;
  return n > 0 ? ((uint32_t)n + a.unit - 1) >> a.unit_log2 : 1;   // an item without keys still has its rows written
}

struct Item {
  int b, head, t0, tokens, h0, heads;
  uint32_t heads_magic;  // row / heads = row * magic >> 16, for rows of an item
  int p0;                // position of token t0
  int first, n;          // keys at first + dilation * i, i < n
};

__device__ __forceinline__ int token_of(const Item& it, int row) { return row * it.heads_magic >> 16; }

// The rows of an item: they do not depend on the sequence's length.
__device__ __forceinline__ Item rows_of(const DecodeArgs& a, int b, uint32_t index) {
  Item it;
  it.b = b;
  uint32_t hb = 0, tb = 0, head = index;
  if (a.head_blocks > 1) {
    hb = head % a.head_blocks;
    head /= a.head_blocks;
  }
  if (a.token_blocks > 1) {
    tb = head % a.token_blocks;
    head /= a.token_blocks;
  }
  it.head = head;
  it.t0 = tb * a.item_tokens;
  it.tokens = min(a.item_tokens, a.T - it.t0);
  it.h0 = hb * a.item_heads;
  it.heads = min(a.item_heads, a.group - it.h0);
  it.heads_magic = 65536u / it.heads + 1;
  return it;
}

__device__ __forceinline__ Item item_of(const DecodeArgs& a, int b, uint32_t index, int length) {
  Item it = rows_of(a, b, index);
  const int len = length < 0 ? 0 : length;
  it.p0 = len - a.T + it.t0;
  const int last = it.p0 + it.tokens - 1;
  it.first = 0;
  it.n = 0;
  if (last < 0) return it;
  if (a.dilation > 1) {                       // one token an item
    const int there = last / a.dilation + 1;
    const int count = there < a.window ? there : (int)a.window;
    it.first = last - (count - 1) * a.dilation;
    const int known = it.first < a.capacity ? (a.capacity - 1 - it.first) / a.dilation + 1 : 0;
    it.n = count < known ? count : known;
  } else {
    const int64_t from = (it.p0 > 0 ? it.p0 : 0) - a.window + 1;
    it.first = from > 0 ? (int)from : 0;
    const int end = last < a.capacity ? last + 1 : a.capacity;
    it.n = end > it.first ? end - it.first : 0;
  }
  return it;
}

// The ranges of `parts` blocks over `total` units: equal to within one unit, the longer ones first.
struct Split {
  uint32_t base, extra;
  __device__ __forceinline__ Split(uint32_t total, uint32_t parts) : base(total / parts), extra(total - base * parts) {}
  __device__ __forceinline__ uint32_t begin(uint32_t part) const { return part * base + min(part, extra); }
  __device__ __forceinline__ uint32_t part_with(uint32_t unit) const {
    const uint32_t longer = extra * (base + 1);
    return unit < longer ? unit / (base + 1) : extra + (unit - longer) / base;
  }
};

// The block's range of units and the sequence in which it begins. With fewer units than blocks the last
// blocks have nothing to do: a block between an item's first and last one always has a unit of it.
struct Range {
  uint32_t begin, end, total;
  int parts;
  int b, length;         // sequence of `begin`
  uint32_t before;       // units of all sequences before it
};
__device__ __forceinline__ Range my_range(const DecodeArgs& a) {
  Range r;
  if (a.cluster) {
    // the block's share of its cluster's item, counted like the ranges below from the sequence's first unit
    const uint32_t id = blockIdx.x >> a.cluster_log2, rank = blockIdx.x & (a.cluster - 1);
    r.b = id / a.items;
    r.length = a.lengths[r.b];
    r.before = 0;
    const uint32_t units = units_of(a, r.length), first = (id - r.b * a.items) * units;
    r.begin = first + (units * rank >> a.cluster_log2);
    r.end = first + (units * (rank + 1) >> a.cluster_log2);
    r.total = r.parts = 0;
    return r;
  }
  __shared__ uint32_t sums[2][kWarps];
  __shared__ uint32_t found_before;
  __shared__ int found_b, found_length;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const auto scan = [&](uint32_t x) {         // inclusive, over the warp
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    return x;
  };
  // the first kThreads sequences, a thread each, and the sum of the others
  int length = (int)threadIdx.x < a.B ? a.lengths[threadIdx.x] : 0;
  uint32_t mine = (int)threadIdx.x < a.B ? units_of(a, length) * a.items : 0, incl = scan(mine), others = 0;
  for (int b = threadIdx.x + kThreads; b < a.B; b += kThreads) others += units_of(a, a.lengths[b]) * a.items;
  others = __reduce_add_sync(0xffffffffu, others);
  if (lane == 31) {
    sums[0][warp] = incl;
    sums[1][warp] = others;
  }
  __syncthreads();
  r.total = 0;
  uint32_t before = 0, chunk = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += sums[0][w];
    chunk += sums[0][w];
    r.total += sums[0][w] + sums[1][w];
  }
  r.parts = (int)min(r.total, (uint32_t)a.parts);
  r.begin = r.end = 0;
  r.b = r.length = 0;
  r.before = 0;
  if ((int)blockIdx.x >= r.parts) return r;
  const Split split(r.total, r.parts);
  r.begin = split.begin(blockIdx.x);
  r.end = split.begin(blockIdx.x + 1);
  for (int b0 = 0;;) {                        // the sequence with the range's first unit (always found)
    const uint32_t lo = before + incl - mine;
    if (lo <= r.begin && r.begin < lo + mine) {
      found_b = b0 + threadIdx.x;
      found_length = length;
      found_before = lo;
    }
    __syncthreads();
    b0 += kThreads;
    if (r.begin < chunk || b0 >= a.B) break;  // (the same for every thread)
    const int b = b0 + threadIdx.x;
    length = b < a.B ? a.lengths[b] : 0;
    mine = b < a.B ? units_of(a, length) * a.items : 0;
    incl = scan(mine);
    if (lane == 31) sums[0][warp] = incl;
    __syncthreads();
    before = chunk;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += sums[0][w];
      chunk += sums[0][w];
    }
  }
  r.b = found_b;
  r.length = found_length;
  r.before = found_before;
  return r;
}

// The join's blocks may take their places as blocks of this launch end (they wait for all of it before they read
// anything; every block of this launch has its place from the start).
__device__ __forceinline__ void allow_join(const DecodeArgs& a) {
  if (!a.cluster) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// How a segment (the block's part of an item) leaves: whole (-1), as part 0 of the block (the item began in an
// earlier one) or 1, or as the block's part of its cluster's item (2). The block that has the item's first unit
// notes which blocks the join has to look at.
__device__ __forceinline__ int part_of(const DecodeArgs& a, const Range& r, uint32_t item_begin,
                                       uint32_t item_end, int64_t item_id) {
  if (a.cluster) return a.cluster == 1 ? -1 : 2;
  const bool begins = item_begin >= r.begin, ends = item_end <= r.end;
  if (begins && threadIdx.x == 0)
    a.covered[item_id] = make_int2(
        blockIdx.x, ends ? 1 : (int)Split(r.total, r.parts).part_with(item_end - 1) - (int)blockIdx.x + 1);
  return begins && ends ? -1 : begins ? 1 : 0;
}

// Final values of kN channels of a row.
template <class T, int kN>
__device__ __forceinline__ void write_row(const DecodeArgs& a, const Item& it, int row, int d, float m, float l,
                                          const Elements<float, kN>& x) {
  const int tt = token_of(it, row), h = it.head * a.group + it.h0 + row - tt * it.heads;
  const int64_t at = ((int64_t)it.b * a.T + it.t0 + tt) * a.Hq + h;
  Elements<T, kN> y;
#pragma unroll
  for (int e = 0; e < kN; ++e) y.v[e] = from_float<T>(m == -INFINITY ? 0.f : x.v[e] / l);
  *reinterpret_cast<Elements<T, kN>*>(static_cast<T*>(a.out) + at * a.D + d) = y;
  if (d == 0 && a.lse) a.lse[at] = m == -INFINITY ? -INFINITY : (m + log2f(l)) * kLn2;
}
// Where a block of a cluster keeps its part [rows_max][D]: behind its warps' outputs.
__host__ __device__ __forceinline__ int joint_at(int o_stride, int rows_max) { return kWarps * rows_max * o_stride; }

// Merges the warps' maxima, sums and outputs of the item's rows and writes them out. `o` holds the warps'
// unnormalised outputs [kWarps][rows_max][o_stride], ml their (maximum, sum) [kWarps][rows_max]. kN channels
// at a time.
template <class T, int kN>
__device__ __forceinline__ void leave(const DecodeArgs& a, const Item& it, int part, const float* o,
                                      int o_stride, const float2* ml, int rows_max,
                                      float2* joint_ml) {
  const int rows = it.tokens * it.heads, lane = threadIdx.x & 31;
  for (int row = threadIdx.x >> 5; row < rows; row += kWarps) {
    float m = -INFINITY, l = 0.f, f[kWarps];
#pragma unroll
    for (int w = 0; w < kWarps; ++w) m = fmaxf(m, ml[w * rows_max + row].x);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float2 p = ml[w * rows_max + row];
      f[w] = p.x == -INFINITY ? 0.f : exp2f(p.x - m);               // 0: the warp met no key of this row
      l += p.x == -INFINITY ? 0.f : f[w] * p.y;
    }
    for (int d = lane * kN; d < a.D; d += 32 * kN) {
      Elements<float, kN> x{};
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        if (ml[w * rows_max + row].x == -INFINITY) continue;        // (what lies there was not written)
        const Elements<float, kN> y = *reinterpret_cast<const Elements<float, kN>*>(o + (w * rows_max + row) * o_stride + d);
#pragma unroll
        for (int e = 0; e < kN; ++e) x.v[e] += f[w] * y.v[e];
      }
      if (part < 0) {
        write_row<T, kN>(a, it, row, d, m, l, x);
      } else if (part == 2) {
        *reinterpret_cast<Elements<float, kN>*>(const_cast<float*>(o) + joint_at(o_stride, rows_max) + row * a.D + d) = x;
        if (d == 0) joint_ml[row] = make_float2(m, l);
      } else {
        const int64_t slot = (int64_t)(2 * blockIdx.x + part) * rows_max + row;
        *reinterpret_cast<Elements<float, kN>*>(a.part_o + slot * a.D + d) = x;
        if (d == 0) a.part_ml[slot] = make_float2(m, l);
      }
    }
  }
}

__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The same address in another block of the cluster.
__device__ __forceinline__ uint32_t in_block(const void* p, uint32_t rank) {
  uint32_t y;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(y) : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(p))), "r"(rank));
  return y;
}
__device__ __forceinline__ float2 load_remote2(uint32_t at) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at));
  return v;
}
template <int kN> __device__ __forceinline__ Elements<float, kN> load_remote(uint32_t at) {
  Elements<float, kN> v;
  if constexpr (kN == 4)
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.v[0]), "=f"(v.v[1]), "=f"(v.v[2]), "=f"(v.v[3]) : "r"(at));
  else
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v.v[0]) : "r"(at));
  return v;
}
// The end of a cluster's item: every block has its part in shared memory; each joins a share of the channels.
template <class T, int kN>
__device__ __forceinline__ void join_cluster(const DecodeArgs& a, bool empty, const float* o, int o_stride,
                                             float2* joint_ml, int rows_max) {
  const uint32_t id = blockIdx.x >> a.cluster_log2, rank = blockIdx.x & (a.cluster - 1), b = id / a.items;
  const Item it = rows_of(a, b, id - b * a.items);
  const int rows = it.tokens * it.heads, lane = threadIdx.x & 31;
  if (empty)
    for (int i = threadIdx.x; i < rows; i += kThreads) joint_ml[i] = make_float2(-INFINITY, 0.f);
  cluster_barrier();
  const float* const joint_o = o + joint_at(o_stride, rows_max);
  for (int row = rank * kWarps + (threadIdx.x >> 5); row < rows; row += a.cluster * kWarps) {
    // lane z has block z's maximum and sum
    const float2 p = lane < a.cluster ? load_remote2(in_block(joint_ml + row, lane)) : make_float2(-INFINITY, 0.f);
    float m = p.x;
#pragma unroll
    for (int z = 4; z > 0; z >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, z));
    m = __shfl_sync(0xffffffffu, m, 0);
    const float w = p.x == -INFINITY ? 0.f : exp2f(p.x - m);
    float l = p.x == -INFINITY ? 0.f : w * p.y;
#pragma unroll
    for (int z = 4; z > 0; z >>= 1) l += __shfl_xor_sync(0xffffffffu, l, z);
    l = __shfl_sync(0xffffffffu, l, 0);
    const uint32_t there = __ballot_sync(0xffffffffu, p.x != -INFINITY);
    for (int d0 = 0; d0 < a.D; d0 += 32 * kN) {
      const int d = d0 + lane * kN;
      Elements<float, kN> x{};
#pragma unroll
      for (int z = 0; z < 8; ++z) {
        const float f = __shfl_sync(0xffffffffu, w, z);
        if (!(there >> z & 1) || d >= a.D) continue;                // (what lies there was not written)
        const Elements<float, kN> y = load_remote<kN>(in_block(joint_o + row * a.D + d, z));
#pragma unroll
        for (int e = 0; e < kN; ++e) x.v[e] += f * y.v[e];
      }
      if (d < a.D) write_row<T, kN>(a, it, row, d, m, l, x);
    }
  }
  cluster_barrier();                          // nobody leaves while others read
}

// ---- CUDA cores: rows that 16-byte copies cannot read -------------------------------------------------------
// A lane takes a key of a 32-key tile for the products with the queries, and every 32nd channel for the
// products with the values.
template <class T, class P, int kRows, int kD32>
__global__ void __launch_bounds__(kThreads) decode_simt_kernel(const __grid_constant__ DecodeArgs a) {
  constexpr bool kScaled = std::is_same<P, __nv_fp8_e4m3>::value;
  extern __shared__ float smem[];
  float* q = smem;                                      // [kRows][D]
  float* o = smem + kRows * a.D;                        // [kWarps][kRows][D]
  __shared__ float2 ml[kWarps * kRows], joint_ml[kRows];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Range r = my_range(a);
  allow_join(a);
  int b = r.b, length = r.length;
  uint32_t before = r.before;
  for (uint32_t at = r.begin; at < r.end;) {
    const uint32_t units = units_of(a, length), index = (at - before) / units;
    if (index >= a.items) {
      before += units * a.items;
      length = a.lengths[++b];
      continue;
    }
    const Item it = item_of(a, b, index, length);
    const uint32_t item_begin = before + index * units, item_end = item_begin + units;
    const uint32_t stop = min(item_end, r.end);
    const int rows = it.tokens * it.heads;
    __syncthreads();                                    // (the last segment's buffers are read)
    for (int i = threadIdx.x; i < kRows * a.D; i += kThreads) {
      const int row = i / a.D, d = i - row * a.D;
      float x = 0.f;
      if (row < rows) {
        const int tt = token_of(it, row), t = it.t0 + tt, h = it.head * a.group + it.h0 + row - tt * it.heads;
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
    const int begin = (at - item_begin) * a.unit;
    const int end = (int)min((int64_t)(stop - item_begin) * a.unit, (int64_t)it.n);
    for (int i0 = begin + warp * 32; i0 < end; i0 += kWarps * 32) {
      const int i = i0 + lane;
      int64_t page = -1;
      int slot = 0, j = 0;
      if (i < end) {
        int64_t pi;
        j = it.first + i * a.dilation;
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
#pragma unroll 8
        for (int d = 0; d < a.D; ++d) {
          const float kk = as_float(k[d]);
#pragma unroll
          for (int x = 0; x < kRows; ++x) s[x] += kk * q[x * a.D + d];
        }
      uint32_t seen[kRows];
#pragma unroll
      for (int x = 0; x < kRows; ++x) {
        const int p = it.p0 + token_of(it, x);
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
      // kAhead value rows are under way together
      constexpr int kAhead = kD32 > 4 ? 4 : 8;
      const int count = min(32, end - i0);
      for (int key0 = 0; key0 < count; key0 += kAhead) {
        P vv[kAhead][kD32];
#pragma unroll
        for (int z = 0; z < kAhead; ++z) {
          const int64_t off = __shfl_sync(0xffffffffu, v_at, key0 + z);     // (0, and no row's, behind the last)
          const P* v = static_cast<const P*>(a.value.base) + off;
          const bool has = key0 + z < count && __shfl_sync(0xffffffffu, (int)there, key0 + z);
#pragma unroll
          for (int e = 0; e < kD32; ++e) vv[z][e] = has && lane + 32 * e < a.D ? v[lane + 32 * e] : P(0.f);
        }
#pragma unroll
        for (int z = 0; z < kAhead; ++z)
#pragma unroll
          for (int x = 0; x < kRows; ++x) {
            const float p = __shfl_sync(0xffffffffu, s[x], key0 + z);
            // a NaN or an infinity stays with the rows that attend its token
            if (seen[x] >> (key0 + z) & 1)
#pragma unroll
              for (int e = 0; e < kD32; ++e) acc[x][e] += p * as_float(vv[z][e]);
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
    leave<T, 1>(a, it, part, o, a.D, ml, kRows, joint_ml);
    at = stop;
  }
  if (a.cluster > 1) join_cluster<T, 1>(a, r.begin == r.end, o, a.D, joint_ml, kRows);
}

// ---- tensor cores: fp16 / bf16 queries, 16-byte rows ---------------------------------------------------
// A warp works alone on tiles of kKeys keys with copies of its own (cp.async, kStages tiles in flight), so
// nothing waits for another warp before the item's end: 128 KB in flight per SM. The products are small next
// to the bytes (rows are padded to the instruction's 16: 2 x 16 flops a cached element), so mma.sync on
// fragments that ldmatrix takes out of the copied rows is enough (a 16-key bf16 tile: 32 of them, 256 of the
// 1365 cycles that its 8 KB take at the copy rate); tcgen05 would want 128-row tiles and the probabilities in
// shared memory or TMEM for the same bytes. Measured: 64 sequences of 4 x 128 channels behind 2048 tokens, 259 MB
// in 49 us (5.3 TB/s, 80 % of the copy rate); 16 whole 8-bit contexts, 312 MB in 71 us (67 %; 46 % of issue slots and
// 29 % of the tensor pipe in use: the two warps of a scheduler wait for their own chains of products, conversions,
// maxima and exponentials).
//
// Weights are rounded to the values' 16-bit type for the second product, like in the prefill kernels; maxima,
// sums and outputs are fp32. 8-bit rows are converted to fp16, which holds every e4m3 value, in registers. A key's scale multiplies its
// logits; a value's scale goes into its weight as 2^(s_j + log2 scale_j - m'), with a running maximum m' of
// its own, so that the largest of these weights is 1 whatever the scales are and fp16 loses only what is
// 2^-24 of it. Queries on 8-bit keys are multiplied by a power of two that brings the row's largest to [1, 2); channels
// below 2^-14 of it (bf16: 2^-17) are off by up to 2^-25 of it in fp16.
template <class T> struct Half2Of;
template <> struct Half2Of<__half> {
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    return bits_as<uint32_t>(__floats2half2_rn(x, y));
  }
};
template <> struct Half2Of<__nv_bfloat16> {
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    return bits_as<uint32_t>(__floats2bfloat162_rn(x, y));
  }
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float lg2(float x) {      // of a scale: 2^-126 at least, or 0 where there is no key
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(there ? 4 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending> __device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}
template <bool kTrans> __device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t at) {
  if (kTrans)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}
// Two 16 x 16 matrices of bytes, transposed: register z of matrix y (2 y + z) has column lane / 4 + 8 z of rows
// 4 (lane % 4) .. + 3.
__device__ __forceinline__ void ldmatrix_bytes(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}
template <class M> __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (std::is_same<M, __half>::value)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_e4m3(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Four e4m3 values -> two fp16 values each, the low ones and the high ones.
__device__ __forceinline__ void e4m3_to_f16(uint32_t x, uint32_t& low, uint32_t& high) {
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\tcvt.rn.f16x2.e4m3x2 %1, hi;\n\t}"
      : "=r"(low), "=r"(high) : "r"(x));
}

// Keys of a warp's tile: about 4 KB of them, for cached elements of `elem` bytes.
__host__ __device__ constexpr int tile_keys(int row_bytes, int elem) {
  return row_bytes >= 512 && elem == 4 ? 8 : row_bytes >= 256 ? 16 : 32;
}

// kElem: bytes of a cached element. k32: 32-bit queries (the CUDA-core kernel below).
template <int kDP, int kElem, int kRows, bool k32> struct Tile {
  static constexpr int kRowBytes = kDP * kElem;
  static constexpr int kChunks = kRowBytes / 16;                   // of a row
  static constexpr int kKeys = tile_keys(kRowBytes, kElem);
  // Two blocks of an SM with three tiles a warp under way. Two tiles: 64 sequences, window 2048 equal, 8-bit
  // contexts 72.6 instead of 73.7 us, 256 sequences, window 512 59.6 instead of 55.9; three blocks with two tiles
  // (registers capped at 168): equal, 73.8 and 56.1. The next tile's products with the keys ahead of this one's
  // weights, which leaves one tile under way: 49.6, 75.5 and 60.0 instead of 49.2, 73.7 and 55.9.
  static constexpr int kStages = 3;
  static constexpr int kMatrix = kKeys * kRowBytes;                // bytes of a tile of keys, or of values
  static constexpr int kStage = 2 * kMatrix;
  static constexpr int kExtra = 16 + (kElem == 1 ? 2 * kKeys * 4 : 0);     // which keys are there; scales
  static constexpr int kBlocks = kDP == 256 && kElem > 1 ? 1 : 2;        // of an SM
  static constexpr int kQueryPitch = k32 ? kDP * 4 : kDP * 2 + 16;   // bytes of a query row
  // tiles, then what goes with them, then the queries; at an item's end results lie where the tiles were
  static constexpr int kExtraAt = kWarps * kStages * kStage, kQueryAt = kExtraAt + kWarps * kStages * kExtra;
  static size_t bytes(int D) {
    const size_t merge = ((size_t)joint_at(D + 8, kRows) + (size_t)kRows * D) * sizeof(float);
    const size_t all = kQueryAt + (k32 ? kRows : 16) * kQueryPitch;
    return all > merge ? all : merge;
  }
  // Byte of a chunk in a tile. Chunks of a row are permuted so that eight neighbouring rows have any one
  // chunk in eight different groups of banks; at(row, c ^ x) == at(row, c) ^ (x << 4).
  static __device__ __forceinline__ uint32_t at(int row, int chunk) {
    // (32-bit queries: of two neighbouring rows, any four chunks c, c ^ 1, c ^ 2, c ^ 3)
    const int x = kChunks < 8 ? row >> 1 & 3 : k32 ? (row & 1) << 2 | (row >> 1 & 3) : row & 7;
    return row * kRowBytes + ((chunk ^ x) << 4);
  }
  // 8-bit keys for the tensor cores are read in rows 0, 1, 4, 5, 8, 9, 12, 13 and 2, 3, .. (see there).
  static constexpr bool kPairs = kElem == 1 && !k32;
  static constexpr uint32_t kOddGroup = kPairs ? (kChunks >= 8 ? 4 : 2) << 4 : 0;   // of the chunks of rows 8 .. 15
  static __device__ __forceinline__ uint32_t key_at(int row, int chunk) {
    if (!kPairs) return at(row, chunk);
    const int x = kChunks >= 8 ? (row & 1) | (row >> 1 & 6) : row >> 2 & 3;
    return row * kRowBytes + ((chunk ^ x) << 4);
  }
};

// What a warp does to get its tiles of an item's keys into shared memory.
template <class L, bool k8, int kElem> struct Feed {
  const DecodeArgs& a;
  const Item& it;
  const int* table;
  const uint8_t *k_base, *v_base;
  const float *ks_base, *vs_base;
  int begin, end, count;         // its first key, the end of the block's keys, its tiles
  uint8_t* extra;                // the warp's, stage 0
  uint32_t tiles_at, extra_at, key_off, value_off;   // (of the lane's copies)
  int chunks;                    // c, c + 4, .. of a row, that there are
  int page, slot;                // of this lane's key of the tile that is fetched next; page -1: there is none

  // Looked up a tile before its copies are issued.
  __device__ __forceinline__ void look_up(int s) {
    const int i = begin + s * a.step + (threadIdx.x & 31 & (L::kKeys - 1));
    page = -1;
    slot = 0;
    if (s < count && i < end) {
      const uint32_t j = it.first + i * a.dilation;
      uint32_t pi;
      if (a.table.shift >= 0) {
        pi = j >> a.table.shift;
        slot = j & (a.table.page_size - 1);
      } else {
        pi = j / (uint32_t)a.table.page_size;
        slot = j - pi * a.table.page_size;
      }
      if (pi < (uint32_t)a.table.max_pages) page = table[pi];
      if ((uint32_t)page >= (uint32_t)a.table.pages) page = -1;
    }
  }
  // Copies: four lanes to a key, 64 bytes of its row at a time.
  __device__ __forceinline__ void fetch(int s, int stage) {
    const int lane = threadIdx.x & 31, r0 = lane >> 2, c = lane & 3;
    if (s < count) {
      const bool there = page >= 0;
      const uint32_t mask = __ballot_sync(0xffffffffu, there);
      if (lane == 0) *reinterpret_cast<uint32_t*>(extra + stage * L::kExtra) = mask;
      int64_t k_at = -1, v_at = -1;
      if (there) {
        k_at = a.key.at(page, slot) * kElem;
        v_at = a.same_strides ? k_at : a.value.at(page, slot) * kElem;
      }
      const uint32_t key_to = tiles_at + stage * L::kStage + key_off, value_to = tiles_at + stage * L::kStage + value_off;
#pragma unroll
      for (int g = 0; g < L::kKeys / 8; ++g) {
        const int64_t ka = __shfl_sync(0xffffffffu, k_at, 8 * g + r0);
        const int64_t va = a.same_strides ? ka : __shfl_sync(0xffffffffu, v_at, 8 * g + r0);
        // zeros where there is nothing: copies of no bytes, whose addresses are not looked at
        const uint8_t* const k = k_base + (ka >= 0 ? ka + c * 16 : 0);
        const uint8_t* const v = v_base + (ka >= 0 ? va + c * 16 : 0);
        const int n = ka >= 0 ? chunks : 0;
#pragma unroll
        for (int i = 0; i < L::kChunks / 4; ++i) {
          const int bytes = 4 * i < n ? 16 : 0;
          copy16((key_to ^ (i << 6) ^ (g & 1 ? L::kOddGroup : 0)) + 8 * g * L::kRowBytes, k + i * 64, bytes);
          copy16((value_to ^ (i << 6)) + 8 * g * L::kRowBytes, v + i * 64, bytes);
        }
      }
      if (k8 && lane < L::kKeys) {
        const int64_t ks = there ? a.key.scale_at(page, slot) : 0;
        const int64_t vs = !there ? 0 : a.same_strides ? ks : a.value.scale_at(page, slot);
        const uint32_t to = extra_at + stage * L::kExtra + 16 + lane * 4;
        copy4(to, ks_base + ks, there);
        copy4(to + L::kKeys * 4, vs_base + vs, there);
      }
    }
    copy_commit();
  }
};

// The first n bits.
__device__ __forceinline__ uint32_t first_bits(int n) {
  return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1;
}
// Elements that are not finite (of a 32-bit word), as a mask over the word. 8 bits: e4m3 has a NaN only.
template <class T, bool k8> __device__ __forceinline__ uint32_t not_finite(uint32_t x) {
  if (k8) return __vcmpeq4(x & 0x7f7f7f7fu, 0x7f7f7f7fu);
  const uint32_t e = std::is_same<T, __half>::value ? 0x7c007c00u : 0x7f807f80u;
  return __vcmpeq2(x & e, e);
}

// kRows 8: items of at most eight rows, so that the lower halves of the instructions' results are not looked at.
template <class T, bool k8, int kDP, int kRows>
__global__ void __launch_bounds__(kThreads, Tile<kDP, k8 ? 1 : 2, kRows, false>::kBlocks)
decode_mma_kernel(const __grid_constant__ DecodeArgs a) {
  using M = typename std::conditional<k8, __half, T>::type;        // operands of the products
  using L = Tile<kDP, k8 ? 1 : 2, kRows, false>;
  constexpr int kKeys = L::kKeys, kStages = L::kStages, kGroups = kKeys / 16, kSteps = kDP / 16;
  constexpr int kX = kRows / 8, kE = 2 * kX;                       // rows and results of a fragment in use
  // bf16 queries, 8-bit keys, eight rows: the products with the keys in 8 bits, see below
  constexpr bool kSplit = k8 && kRows == 8 && std::is_same<T, __nv_bfloat16>::value;
  constexpr int kElem = k8 ? 1 : 2;
  extern __shared__ __align__(1024) uint8_t tiles[];
  __shared__ float2 ml[kWarps * kRows], joint_ml[kRows];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int r0 = lane >> 2, c = lane & 3;                          // rows r0, r0 + 8 and columns 2c, 2c + 1
  uint8_t* const my_tiles = tiles + warp * kStages * L::kStage;
  uint8_t* const my_extra = tiles + L::kExtraAt + warp * kStages * L::kExtra;
  uint8_t* const queries = tiles + L::kQueryAt;
  const uint32_t tiles_at = static_cast<uint32_t>(__cvta_generic_to_shared(my_tiles));
  const uint32_t extra_at = static_cast<uint32_t>(__cvta_generic_to_shared(my_extra));
  // Fragments of keys. 16 bits: keys 8 z + 0 .. 7 are the columns of product z of two. 8 bits: keys 4 i + 2 z
  // and + 1, so that a thread's columns of both products are four neighbouring keys, as the transposing load
  // of the values has them.
  const int key_z = kSplit || !k8 ? lane >> 4 : lane >> 3 & 1, key_chunk = kSplit || !k8 ? lane >> 3 & 1 : lane >> 4;
  const uint32_t key_off = L::key_at(k8 ? (lane & 6) * 2 + (lane & 1) + 2 * key_z : (lane & 7) + 8 * key_z, key_chunk);
  const auto column = [&](int i, int e) { return k8 ? 16 * (i >> 1) + 4 * c + 2 * (i & 1) + e : 8 * i + 2 * c + e; };
  const uint32_t value_off = L::kMatrix + L::at(lane & 15, lane >> 4);   // of values
  const int my_chunks = a.D * kElem / 16 - c;                      // chunks c, c + 4, .. that a row has

  const Range r = my_range(a);
  allow_join(a);
  int b = r.b, length = r.length;
  uint32_t before = r.before;
  for (uint32_t at = r.begin; at < r.end;) {
    const uint32_t units = units_of(a, length), index = (at - before) / units;
    if (index >= a.items) {
      before += units * a.items;
      length = a.lengths[++b];
      continue;
    }
    const Item it = item_of(a, b, index, length);
    const uint32_t item_begin = before + index * units, item_end = item_begin + units;
    const uint32_t stop = min(item_end, r.end);
    const int rows = it.tokens * it.heads;
    const int begin = (at - item_begin) * a.unit + warp * kKeys;
    const int end = (int)min((int64_t)(stop - item_begin) * a.unit, (int64_t)it.n);
    const int count = end > begin ? (end - begin + a.step - 1) / a.step : 0;          // this warp's tiles

    Feed<L, k8, kElem> feed{a, it, a.table.entry + b * a.table.stride,
                            static_cast<const uint8_t*>(a.key.base) + it.head * a.key.head * kElem,
                            static_cast<const uint8_t*>(a.value.base) + it.head * a.value.head * kElem,
                            a.key.scale + it.head * a.key.s_head, a.value.scale + it.head * a.value.s_head,
                            begin, end, count, my_extra, tiles_at, extra_at, L::key_at(r0, c),
                            L::kMatrix + L::at(r0, c), my_chunks, -1, 0};
    feed.look_up(0);
#pragma unroll 1
    for (int s = 0; s < kStages - 1; ++s) {
      feed.fetch(s, s);
      feed.look_up(s + 1);
    }

    // The queries into shared memory, and from there as A fragments: rows r0 and r0 + 8.
#pragma unroll 1
    for (int i = threadIdx.x; i < kRows * (kDP / 8); i += kThreads) {
      const int row = i / (kDP / 8), d = i % (kDP / 8) * 8;
      Raw<T, 8> piece{};
      if (row < rows && d < a.D) {
        const int tt = token_of(it, row), h = it.head * a.group + it.h0 + row - tt * it.heads;
        const T* const src = static_cast<const T*>(a.query) + b * a.q_batch + (it.t0 + tt) * a.q_token + h * a.q_head + d;
        if (a.q_wide) {
          piece = *reinterpret_cast<const Raw<T, 8>*>(src);
        } else {
          T x[8];
          for (int e = 0; e < 8; ++e) x[e] = src[e];
          memcpy(&piece, x, 16);
        }
      }
      *reinterpret_cast<Raw<T, 8>*>(queries + row * L::kQueryPitch + d * 2) = piece;
    }
    __syncthreads();
    uint32_t q[kSplit ? kSteps / 2 : kSteps][4];
    float row_scale[kX];
    int row_token[kX];
#pragma unroll
    for (int x = 0; x < kX; ++x) {
      row_token[x] = token_of(it, r0 + 8 * x);
      row_scale[x] = a.scale_log2;
    }
    if constexpr (!k8) {
      // channels 16 k + 2c, + 1 and 8 further
      const uint32_t from = static_cast<uint32_t>(__cvta_generic_to_shared(queries)) +
                            (kX == 2 ? lane & 15 : lane & 7) * L::kQueryPitch + (lane >> 4) * 16;
#pragma unroll
      for (int k = 0; k < kSteps; ++k) {
        ldmatrix4<false>(q[k], from + k * 32);
        if (kX == 1) q[k][1] = q[k][3] = 0;
      }
    } else {
      // channels 16 k + 4c .. + 3, the four that one 32-bit word of a key row holds
#pragma unroll
      for (int x = 0; x < kX; ++x) {
        float v[kSteps][4], most = 0.f;
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
          to_floats<T, 4>(*reinterpret_cast<const Raw<T, 4>*>(queries + (r0 + 8 * x) * L::kQueryPitch + (16 * k + 4 * c) * 2), v[k]);
#pragma unroll
          for (int e = 0; e < 4; ++e) most = fmaxf(most, fabsf(v[k][e]));
        }
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        // The row times the power of two that brings its largest magnitude to [1, 2) (kSplit: [128, 256)), where
        // that power and its inverse are normal numbers.
        constexpr int kUp = kSplit ? 7 : 0;
        const int e = min((__float_as_int(most) >> 23) - 127, kUp ? 127 : 126);
        float factor = 1.f;
        if (e > kUp - 126) {
          factor = __int_as_float((127 + kUp - e) << 23);
          // (never 0, which the -inf of a token that is not attended must not meet: logits of that size are 0)
          row_scale[x] = fmaxf(row_scale[x] * __int_as_float((127 - kUp + e) << 23), __int_as_float(1));
        }
        if constexpr (kSplit) {
          // e4m3 has no infinity: NaNs in its place, which only the tokens that the row attends bring to it
          if (!(most < INFINITY)) factor = __int_as_float(0x7fc00000);
          // A bf16 number is the sum of two e4m3 ones: the nearest one and what is left (four bits and sign,
          // times 16). Row r0 of the instruction is the first, row r0 + 8 the second. Nothing is lost of channels
          // within 2^13 of the row's largest; what is left of smaller ones ends at e4m3's smallest step, which is
          // 2^-21 of the largest channel at most (an 8-bit key is off by 2^-4 of itself).
#pragma unroll
          for (int k = 0; k < kSteps; ++k) {
            float left[4];
            uint32_t hi = 0;
#pragma unroll
            for (int z = 0; z < 4; z += 2) {
              const __nv_fp8x2_storage_t two = __nv_cvt_float2_to_fp8x2(make_float2(v[k][z] * factor, v[k][z + 1] * factor), __NV_SATFINITE, __NV_E4M3);
              const float2 back = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(two, __NV_E4M3)));
              left[z] = 16.f * (v[k][z] * factor - back.x);
              left[z + 1] = 16.f * (v[k][z + 1] * factor - back.y);
              hi |= (uint32_t)two << (8 * z);
            }
            q[k / 2][2 * (k & 1)] = hi;
            q[k / 2][2 * (k & 1) + 1] = from_floats<__nv_fp8_e4m3, 4>(left);
          }
        } else {
#pragma unroll
          for (int k = 0; k < kSteps; ++k)
#pragma unroll
            for (int z = 0; z < 2; ++z) {
              q[k][x + 2 * z] = Half2Of<M>::pack(v[k][2 * z] * factor, v[k][2 * z + 1] * factor);
              if (kX == 1) q[k][1 + 2 * z] = 0;
            }
        }
      }
    }
    // Tiles whose first key lies in [safe_from, safe_to] are attended whole, or not, by all rows alike.
    const bool alike = it.tokens == 1;
    const int64_t safe_from = (int64_t)it.p0 + it.tokens - a.window, safe_to = (int64_t)it.p0 - kKeys + 1;

    float acc[kDP / 8][4], m[kX], l[kX], mv[kX];
#pragma unroll
    for (int i = 0; i < kDP / 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][e] = 0.f;
#pragma unroll
    for (int x = 0; x < kX; ++x) {
      m[x] = mv[x] = -INFINITY;
      l[x] = 0.f;
    }

    int stage = 0;
#pragma unroll 1
    for (int s = 0; s < count; ++s) {
      copy_wait<kStages - 2>();
      __syncwarp();                        // the tile is there, and everyone is done with the one before it
      feed.fetch(s + kStages - 1, stage == 0 ? kStages - 1 : stage - 1);
      feed.look_up(s + kStages);
      const uint32_t base = tiles_at + stage * L::kStage;
      const uint8_t* extra = my_extra + stage * L::kExtra;
      uint8_t* const values = my_tiles + stage * L::kStage + L::kMatrix;
      stage = stage == kStages - 1 ? 0 : stage + 1;

      // p = queries x keys: column(i, 0) and column(i, 1) of rows r0 (0, 1) and r0 + 8 (2, 3). With 16 keys the sums
      // over the channels go in two, so that no chain of products is longer than four.
      constexpr int kChains = kGroups == 1 ? 2 : 1;
      float part[kChains][2 * kGroups][4];
#pragma unroll
      for (int z = 0; z < kChains; ++z)
#pragma unroll
        for (int i = 0; i < 2 * kGroups; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) part[z][i][e] = 0.f;
      const uint32_t keys = base + key_off;
      if constexpr (kSplit) {
        // 8-bit operands: the keys as they are, four times the rate of 16-bit ones (m16n8k32 4.5 cycles, the
        // 16-bit m16n8k16 8 cycles) and no conversions. The products of e4m3 numbers are exact.
#pragma unroll
        for (int k = 0; k < kSteps / 2; ++k)
#pragma unroll
          for (int g = 0; g < kGroups; ++g) {
            uint32_t f[4];
            ldmatrix4<false>(f, (keys ^ (k << 5)) + 16 * g * L::kRowBytes);
            mma_e4m3(part[k % kChains][2 * g], q[k], f[0], f[1]);
            mma_e4m3(part[k % kChains][2 * g + 1], q[k], f[2], f[3]);
          }
      } else if constexpr (!k8) {
#pragma unroll
        for (int k = 0; k < kSteps; ++k)
#pragma unroll
          for (int g = 0; g < kGroups; ++g) {
            uint32_t f[4];
            ldmatrix4<false>(f, (keys ^ (k << 5)) + 16 * g * L::kRowBytes);
            mma<M>(part[k % kChains][2 * g], q[k], f[0], f[1]);
            mma<M>(part[k % kChains][2 * g + 1], q[k], f[2], f[3]);
          }
      } else {
#pragma unroll
        for (int k = 0; k < kSteps; k += 2)
#pragma unroll
          for (int g = 0; g < kGroups; ++g) {
            uint32_t f[4];
            ldmatrix4<false>(f, (keys ^ (k << 4)) + 16 * g * L::kRowBytes);
#pragma unroll
            for (int z = 0; z < 2; ++z) {
              uint32_t low, high;
              e4m3_to_f16(f[2 * z], low, high);
              mma<M>(part[z % kChains][2 * g], q[k + z], low, high);
              e4m3_to_f16(f[2 * z + 1], low, high);
              mma<M>(part[z % kChains][2 * g + 1], q[k + z], low, high);
            }
          }
      }
      float p[2 * kGroups][kE], lv[2 * kGroups][2];
#pragma unroll
      for (int i = 0; i < 2 * kGroups; ++i) {
#pragma unroll
        for (int e = 0; e < kE; ++e) {
          p[i][e] = part[0][i][e];
          if (kChains == 2) p[i][e] += part[kChains - 1][i][e];
          if (kSplit) p[i][e] += 0.0625f * (kChains == 2 ? part[0][i][e + 2] + part[kChains - 1][i][e + 2] : part[0][i][e + 2]);
        }
        if constexpr (k8) {
          const float2 ks = *reinterpret_cast<const float2*>(extra + 16 + column(i, 0) * 4);
          const float2 vs = *reinterpret_cast<const float2*>(extra + 16 + (kKeys + column(i, 0)) * 4);
          lv[i][0] = lg2(vs.x);
          lv[i][1] = lg2(vs.y);
#pragma unroll
          for (int e = 0; e < kE; ++e) p[i][e] *= e & 1 ? ks.y : ks.x;
        }
      }

      // which keys each row attends
      const uint32_t there = *reinterpret_cast<const uint32_t*>(extra) & first_bits(kKeys);
      const int j0 = it.first + (begin + s * a.step) * a.dilation;
      const bool differ = !alike && !(j0 >= safe_from && j0 <= safe_to);
      if (there != first_bits(kKeys) || differ) {
        uint32_t on[2] = {there, there};
        if (differ) {
#pragma unroll
          for (int x = 0; x < kX; ++x) {
            const int upto = it.p0 + row_token[x] - j0 + 1;        // keys j <= p and j > p - window
            const int64_t from = upto - a.window;
            on[x] &= first_bits(upto) & ~first_bits(from > 0 ? (int)min(from, (int64_t)32) : 0);
          }
        }
#pragma unroll
        for (int i = 0; i < 2 * kGroups; ++i)
#pragma unroll
          for (int e = 0; e < kE; ++e)
            if (!(on[e >> 1] >> column(i, e & 1) & 1)) {
              p[i][e] = -INFINITY;
              if (k8 && kX == 1) lv[i][e & 1] = 0.f;               // left out, whatever its scale is
            }
      }

      // the running maximum of the logits (and of the logits with the values' scales)
      float base_m[kX], base_v[kX], keep[kX];
#pragma unroll
      for (int x = 0; x < kX; ++x) {
        float top = -INFINITY, topv = -INFINITY;
#pragma unroll
        for (int i = 0; i < 2 * kGroups; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            top = fmaxf(top, p[i][2 * x + e]);
            if (k8) topv = fmaxf(topv, fmaf(p[i][2 * x + e], row_scale[x], lv[i][e]));
          }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float next = fmaxf(m[x], top * row_scale[x]);
        // nothing attended yet: no difference of infinities. (A NaN logit is passed over by the maximum and
        // comes back in the exponential.)
        base_m[x] = next == -INFINITY ? 0.f : next;
        keep[x] = ex2(m[x] - base_m[x]);
        l[x] *= keep[x];
        m[x] = next;
        if (k8) {
          topv = fmaxf(topv, __shfl_xor_sync(0xffffffffu, topv, 1));
          topv = fmaxf(topv, __shfl_xor_sync(0xffffffffu, topv, 2));
          const float nextv = fmaxf(mv[x], topv);
          base_v[x] = nextv == -INFINITY ? 0.f : nextv;
          keep[x] = ex2(mv[x] - base_v[x]);
          mv[x] = nextv;
        }
      }
      if (__any_sync(0xffffffffu, !(keep[0] == 1.f && keep[kX - 1] == 1.f))) {
#pragma unroll
        for (int i = 0; i < kDP / 8; ++i)
#pragma unroll
          for (int e = 0; e < kE; ++e) acc[i][e] *= keep[e >> 1];
      }
      uint32_t w[kGroups][4];              // the weights as A fragments
#pragma unroll
      for (int i = 0; i < 2 * kGroups; ++i) {
        float y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int e = 0; e < kE; ++e) {
          const int x = e >> 1;
          const float ex = ex2(fmaf(p[i][e], row_scale[x], -base_m[x]));
          l[x] += ex;
          y[e] = k8 ? ex2(fmaf(p[i][e], row_scale[x], lv[i][e & 1]) - base_v[x]) : ex;
          if (k8 && kX == 2 && p[i][e] == -INFINITY) y[e] = 0.f;   // (two rows share the scale)
        }
        w[i >> 1][2 * (i & 1)] = Half2Of<M>::pack(y[0], y[1]);
        w[i >> 1][2 * (i & 1) + 1] = Half2Of<M>::pack(y[2], y[3]);
      }

      // Rows attend different keys of this tile: 0 x NaN of a value must not reach the rows that do not
      // attend it. Values that are not finite (hardly ever any) go straight to the sums of the rows that
      // do, whatever their weights, and become zeros in the tile.
      if (differ) {
        uint32_t bad = 0;
        for (int i = lane; i < L::kMatrix / 4; i += 32)
          if (not_finite<T, k8>(reinterpret_cast<const uint32_t*>(values)[i])) bad |= 1u << (i / (L::kRowBytes / 4));
        bad = __reduce_or_sync(0xffffffffu, bad) & there;
        for (; bad; bad &= bad - 1) {
          const int key = __ffs(bad) - 1, upto = it.p0 - j0 - key;          // p0 - j
#pragma unroll
          for (int i = 0; i < kDP / 8; ++i) {                               // channels 8 i + 2c, + 1
            using Two = typename RawOf<2 * kElem>::type;
            Two* const two_at = reinterpret_cast<Two*>(values + L::at(key, i * 8 * kElem >> 4) + (i * 8 * kElem & 15) + 2 * c * kElem);
            const uint32_t two = *two_at, odd = not_finite<T, k8>(two);
#pragma unroll
            for (int x = 0; x < kX; ++x) {
              const int back = upto + row_token[x];                         // p - j
              if (back < 0 || back >= a.window) continue;
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                if (!(odd >> (8 * kElem * e) & 1)) continue;
                float y = __int_as_float(0x7fc00000);
                if constexpr (!k8) y = as_float(bits_as<T>((uint16_t)(two >> (16 * e))));
                acc[i][2 * x + e] += y;
              }
            }
            __syncwarp();
            if (odd && r0 == 0) *two_at = (Two)(two & ~odd);
          }
        }
        __syncwarp();
      }

      // values: B fragments of 8-channel columns for 16 keys at a time
      const uint32_t vals = base + value_off;
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        if constexpr (!k8) {
#pragma unroll
          for (int n = 0; n < kSteps; ++n) {
            uint32_t f[4];
            ldmatrix4<true>(f, (vals ^ (n << 5)) + 16 * g * L::kRowBytes);
            mma<M>(acc[2 * n], w[g], f[0], f[1]);
            mma<M>(acc[2 * n + 1], w[g], f[2], f[3]);
          }
        } else {
#pragma unroll
          for (int n = 0; n < kSteps; n += 2) {
            uint32_t f[4];
            ldmatrix_bytes(f, (vals ^ (n << 4)) + 16 * g * L::kRowBytes);
#pragma unroll
            for (int z = 0; z < 4; ++z) {
              uint32_t low, high;
              e4m3_to_f16(f[z], low, high);
              mma<M>(acc[2 * n + z], w[g], low, high);
            }
          }
        }
      }
    }

    // the warps' results side by side in shared memory
    copy_wait<0>();
    __syncthreads();
    float* const o = reinterpret_cast<float*>(tiles);
    const int o_stride = a.D + 8;
#pragma unroll
    for (int x = 0; x < kX; ++x) {
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
      l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
      if (m[x] == -INFINITY && l[x] != l[x]) m[x] = 0.f;           // only NaN logits: they count
      const int row = r0 + 8 * x;
      if (row >= rows) continue;
      if (c == 0) ml[warp * kRows + row] = make_float2(m[x], l[x]);
      if (m[x] == -INFINITY) continue;                             // (not read)
      const float f = k8 ? ex2(mv[x] - m[x]) : 1.f;
      float* const dst = o + (warp * kRows + row) * o_stride;
#pragma unroll
      for (int i = 0; i < kDP / 8; ++i)
        if (8 * i + 2 * c < a.D)
          *reinterpret_cast<float2*>(dst + 8 * i + 2 * c) = make_float2(f * acc[i][2 * x], f * acc[i][2 * x + 1]);
    }
    __syncthreads();
    const int part = part_of(a, r, item_begin, item_end, (int64_t)b * a.items + index);
    leave<T, 4>(a, it, part, o, o_stride, ml, kRows, joint_ml);
    at = stop;
    if (at < r.end) __syncthreads();                               // before the next item's tiles come
  }
  if (a.cluster > 1)
    join_cluster<T, 4>(a, r.begin == r.end, reinterpret_cast<const float*>(tiles), a.D + 8, joint_ml, kRows);
}

// ---- CUDA cores: fp32 queries, 16-byte rows ----------------------------------------------------------------
// fp32 products and sums. The same tiles and copies as above; eight keys at a time: four lanes to a key for the
// products with the queries, every lane a share of the channels for the products with the values. A key costs
// kRows x D multiply-adds for each of both against D cached elements of 4 bytes: at 8 rows 1/2 of what the
// cores do while the memory delivers them.
template <bool k8, int kDP, int kRows>
__global__ void __launch_bounds__(kThreads, Tile<kDP, k8 ? 1 : 4, kRows, true>::kBlocks)
decode_fma_kernel(const __grid_constant__ DecodeArgs a) {
  using L = Tile<kDP, k8 ? 1 : 4, kRows, true>;
  using P = typename std::conditional<k8, __nv_fp8_e4m3, float>::type;
  constexpr int kElem = k8 ? 1 : 4, kKeys = L::kKeys, kStages = L::kStages;
  constexpr int kShare = L::kRowBytes / 32, kPiece = kShare < 16 ? kShare : 16;    // bytes of a value row for a lane
  constexpr int kPieces = kShare / kPiece, kChannels = kPiece / kElem;             // pieces of them, channels each
  constexpr int kOfChunk = 16 / kElem;                                             // channels of a chunk
  extern __shared__ __align__(1024) uint8_t tiles[];
  __shared__ float2 ml[kWarps * kRows], joint_ml[kRows];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int r0 = lane >> 2, c = lane & 3;
  uint8_t* const my_tiles = tiles + warp * kStages * L::kStage;
  uint8_t* const my_extra = tiles + L::kExtraAt + warp * kStages * L::kExtra;
  float* const queries = reinterpret_cast<float*>(tiles + L::kQueryAt);            // [kRows][kDP]
  const uint32_t tiles_at = static_cast<uint32_t>(__cvta_generic_to_shared(my_tiles));
  const uint32_t extra_at = static_cast<uint32_t>(__cvta_generic_to_shared(my_extra));
  const int my_chunks = a.D * kElem / 16 - c;

  const Range r = my_range(a);
  allow_join(a);
  int b = r.b, length = r.length;
  uint32_t before = r.before;
  for (uint32_t at = r.begin; at < r.end;) {
    const uint32_t units = units_of(a, length), index = (at - before) / units;
    if (index >= a.items) {
      before += units * a.items;
      length = a.lengths[++b];
      continue;
    }
    const Item it = item_of(a, b, index, length);
    const uint32_t item_begin = before + index * units, item_end = item_begin + units;
    const uint32_t stop = min(item_end, r.end);
    const int rows = it.tokens * it.heads;
    const int begin = (at - item_begin) * a.unit + warp * kKeys;
    const int end = (int)min((int64_t)(stop - item_begin) * a.unit, (int64_t)it.n);
    const int count = end > begin ? (end - begin + a.step - 1) / a.step : 0;          // this warp's tiles
    Feed<L, k8, kElem> feed{a, it, a.table.entry + b * a.table.stride,
                            static_cast<const uint8_t*>(a.key.base) + it.head * a.key.head * kElem,
                            static_cast<const uint8_t*>(a.value.base) + it.head * a.value.head * kElem,
                            a.key.scale + it.head * a.key.s_head, a.value.scale + it.head * a.value.s_head,
                            begin, end, count, my_extra, tiles_at, extra_at, L::key_at(r0, c),
                            L::kMatrix + L::at(r0, c), my_chunks, -1, 0};
    feed.look_up(0);
#pragma unroll 1
    for (int s = 0; s < kStages - 1; ++s) {
      feed.fetch(s, s);
      feed.look_up(s + 1);
    }
#pragma unroll 1
    for (int i = threadIdx.x; i < kRows * (kDP / 4); i += kThreads) {
      const int row = i / (kDP / 4), d = i % (kDP / 4) * 4;
      float4 piece = make_float4(0.f, 0.f, 0.f, 0.f);
      if (row < rows && d < a.D) {
        const int tt = token_of(it, row), h = it.head * a.group + it.h0 + row - tt * it.heads;
        const float* const src = static_cast<const float*>(a.query) + b * a.q_batch + (it.t0 + tt) * a.q_token + h * a.q_head + d;
        piece = a.q_wide ? *reinterpret_cast<const float4*>(src) : make_float4(src[0], src[1], src[2], src[3]);
      }
      *reinterpret_cast<float4*>(queries + row * kDP + d) = piece;
    }
    __syncthreads();
    int row_token[kRows];
    float acc[kRows][kPieces * kChannels], m[kRows], l[kRows];
#pragma unroll
    for (int x = 0; x < kRows; ++x) {
      row_token[x] = token_of(it, x);
      m[x] = -INFINITY;
      l[x] = 0.f;
#pragma unroll
      for (int e = 0; e < kPieces * kChannels; ++e) acc[x][e] = 0.f;
    }
    const int64_t safe_from = (int64_t)it.p0 + it.tokens - a.window, safe_to = (int64_t)it.p0 - kKeys + 1;

    int stage = 0;
#pragma unroll 1
    for (int s = 0; s < count; ++s) {
      copy_wait<kStages - 2>();
      __syncwarp();
      feed.fetch(s + kStages - 1, stage == 0 ? kStages - 1 : stage - 1);
      feed.look_up(s + kStages);
      const uint8_t* const keys = my_tiles + stage * L::kStage;
      const uint8_t* const values = keys + L::kMatrix;
      const uint8_t* const extra = my_extra + stage * L::kExtra;
      stage = stage == kStages - 1 ? 0 : stage + 1;
      const uint32_t there = *reinterpret_cast<const uint32_t*>(extra) & first_bits(kKeys);
      const int j0 = it.first + (begin + s * a.step) * a.dilation;
      const bool differ = it.tokens > 1 && !(j0 >= safe_from && j0 <= safe_to);
      const bool masked = there != first_bits(kKeys) || differ;
      const auto attends = [&](int x, int key) {      // row x the key of the tile
        const int back = it.p0 + row_token[x] - (j0 + key);
        return (there >> key & 1) && (!differ || (back >= 0 && back < a.window));
      };
#pragma unroll 1
      for (int key0 = 0; key0 < kKeys; key0 += 8) {
        const int key = key0 + r0;
        float p[kRows];
#pragma unroll
        for (int x = 0; x < kRows; ++x) p[x] = 0.f;
#pragma unroll kRows == 8 ? (k8 ? 1 : 2) : 4
        for (int i = 0; i < L::kChunks / 4; ++i) {
          const int chunk = c + 4 * i;
          float k[kOfChunk];
          to_floats<P, kOfChunk>(*reinterpret_cast<const Raw<P, kOfChunk>*>(keys + L::at(key, chunk)), k);
#pragma unroll
          for (int x = 0; x < kRows; ++x)
#pragma unroll
            for (int e = 0; e < kOfChunk; e += 4) {
              const float4 q = *reinterpret_cast<const float4*>(queries + x * kDP + chunk * kOfChunk + e);
              p[x] = fmaf(q.x, k[e], p[x]);
              p[x] = fmaf(q.y, k[e + 1], p[x]);
              p[x] = fmaf(q.z, k[e + 2], p[x]);
              p[x] = fmaf(q.w, k[e + 3], p[x]);
            }
        }
        float factor = a.scale_log2, v_scale = 1.f;
        if (k8) {
          factor *= *reinterpret_cast<const float*>(extra + 16 + key * 4);
          v_scale = *reinterpret_cast<const float*>(extra + 16 + (kKeys + key) * 4);
        }
        bool rescale = false;
        float keep[kRows];
#pragma unroll
        for (int x = 0; x < kRows; ++x) {
          p[x] += __shfl_xor_sync(0xffffffffu, p[x], 1);
          p[x] += __shfl_xor_sync(0xffffffffu, p[x], 2);
          const bool on = !masked || attends(x, key);
          p[x] = on ? p[x] * factor : -INFINITY;
          float top = p[x];
#pragma unroll
          for (int f = 4; f < 32; f <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, f));
          const float next = fmaxf(m[x], top);
          // nothing attended yet: no difference of infinities. (A NaN logit is passed over by the maximum and
          // comes back in the exponential.)
          const float base = next == -INFINITY ? 0.f : next;
          keep[x] = exp2f(m[x] - base);
          rescale = rescale || !(keep[x] == 1.f);
          p[x] = exp2f(p[x] - base);
          l[x] = l[x] * keep[x] + p[x];
          m[x] = next;
          if (k8) p[x] = on ? p[x] * v_scale : 0.f;
        }
        if (rescale) {                                 // (the same for every lane)
#pragma unroll
          for (int x = 0; x < kRows; ++x)
#pragma unroll
            for (int e = 0; e < kPieces * kChannels; ++e) acc[x][e] *= keep[x];
        }
#pragma unroll kRows == 8 ? 4 : 8
        for (int z = 0; z < 8; ++z) {
          float v[kPieces * kChannels];
#pragma unroll
          for (int y = 0; y < kPieces; ++y) {
            const int off = (lane + 32 * y) * kPiece;
            float part[kChannels];
            to_floats<P, kChannels>(*reinterpret_cast<const Raw<P, kChannels>*>(values + L::at(key0 + z, off >> 4) + (off & 15)), part);
#pragma unroll
            for (int e = 0; e < kChannels; ++e) v[y * kChannels + e] = part[e];
          }
#pragma unroll
          for (int x = 0; x < kRows; ++x) {
            const float w = __shfl_sync(0xffffffffu, p[x], 4 * z);
            // a NaN or an infinity stays with the rows that attend its token
            if (masked && !attends(x, key0 + z)) continue;
#pragma unroll
            for (int e = 0; e < kPieces * kChannels; ++e) acc[x][e] = fmaf(w, v[e], acc[x][e]);
          }
        }
      }
    }

    copy_wait<0>();
    __syncthreads();
    float* const o = reinterpret_cast<float*>(tiles);
    const int o_stride = a.D + 8;
#pragma unroll
    for (int x = 0; x < kRows; ++x) {
#pragma unroll
      for (int f = 4; f < 32; f <<= 1) l[x] += __shfl_xor_sync(0xffffffffu, l[x], f);
      if (m[x] == -INFINITY && l[x] != l[x]) m[x] = 0.f;           // only NaN logits: they count
      if (lane == 0) ml[warp * kRows + x] = make_float2(m[x], l[x]);
#pragma unroll
      for (int y = 0; y < kPieces; ++y)
#pragma unroll
        for (int e = 0; e < kChannels; ++e) {
          const int d = (lane + 32 * y) * kChannels + e;
          if (x < rows && d < a.D) o[(warp * kRows + x) * o_stride + d] = acc[x][y * kChannels + e];
        }
    }
    __syncthreads();
    const int part = part_of(a, r, item_begin, item_end, (int64_t)b * a.items + index);
    leave<float, 4>(a, it, part, o, o_stride, ml, kRows, joint_ml);
    at = stop;
    if (at < r.end) __syncthreads();                               // before the next item's tiles come
  }
  if (a.cluster > 1)
    join_cluster<float, 4>(a, r.begin == r.end, reinterpret_cast<const float*>(tiles), a.D + 8, joint_ml, kRows);
}

// ---- the join --------------------------------------------------------------------------------------------
// A warp per row of an item; items that one block had are done. A lane has a part's maximum and sum, then the
// lanes share the channels, kN each.
template <class T, int kN>
__global__ void __launch_bounds__(kThreads) decode_join_kernel(const __grid_constant__ DecodeArgs a,
                                                               int rows_max) {
  const int lane = threadIdx.x & 31;
  const uint32_t id_row = blockIdx.x * kWarps + (threadIdx.x >> 5), id = id_row / rows_max;
  const int row = (int)(id_row - id * rows_max);
  const bool mine = id < a.B * a.items;
  const int b = id / a.items;
  const Item it = rows_of(a, b, id - b * a.items);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (!mine || row >= it.tokens * it.heads) return;
  const int2 covered = a.covered[id];
  if (covered.y <= 1) return;
  // the first block's part is its second one (the item began there), the others' their first
  const auto slot = [&](int i) { return (2 * (covered.x + i) + (i == 0 ? 1 : 0)) * rows_max + row; };
  constexpr int kMostPieces = 256 / (32 * kN);       // of a lane
  float m = -INFINITY, l = 0.f, acc[kMostPieces][kN];
#pragma unroll
  for (int y = 0; y < kMostPieces; ++y)
#pragma unroll
    for (int e = 0; e < kN; ++e) acc[y][e] = 0.f;
  for (int i0 = 0; i0 < covered.y; i0 += 32) {
    const int count = min(32, covered.y - i0);
    const float2 p = lane < count ? a.part_ml[slot(i0 + lane)] : make_float2(-INFINITY, 0.f);
    float top = p.x;
#pragma unroll
    for (int f = 16; f > 0; f >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, f));
    const float next = fmaxf(m, top), base = next == -INFINITY ? 0.f : next;
    const float keep = exp2f(m - base);
    const float w = p.x == -INFINITY ? 0.f : exp2f(p.x - base);
    float sum = p.x == -INFINITY ? 0.f : w * p.y;
#pragma unroll
    for (int f = 16; f > 0; f >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, f);
    l = l * keep + sum;
    m = next;
    const uint32_t there = __ballot_sync(0xffffffffu, p.x != -INFINITY);      // others were not written
#pragma unroll
    for (int y = 0; y < kMostPieces; ++y)
#pragma unroll
      for (int e = 0; e < kN; ++e) acc[y][e] *= keep;
    // eight parts' loads under way together
    for (int i = 0; i < count; i += 8) {
#pragma unroll
      for (int y = 0; y < kMostPieces; ++y) {
        const int d = (lane + 32 * y) * kN;
        Elements<float, kN> o[8];
#pragma unroll
        for (int z = 0; z < 8; ++z) {
          o[z] = Elements<float, kN>{};
          if ((there >> (i + z) & 1) && d < a.D)
            o[z] = *reinterpret_cast<const Elements<float, kN>*>(a.part_o + (int64_t)slot(i0 + i + z) * a.D + d);
        }
#pragma unroll
        for (int z = 0; z < 8; ++z) {
          const float f = __shfl_sync(0xffffffffu, w, i + z);
#pragma unroll
          for (int e = 0; e < kN; ++e) acc[y][e] += f * o[z].v[e];
        }
      }
    }
  }
#pragma unroll
  for (int y = 0; y < kMostPieces; ++y) {
    const int d = (lane + 32 * y) * kN;
    if (d >= a.D) continue;
    Elements<float, kN> x;
#pragma unroll
    for (int e = 0; e < kN; ++e) x.v[e] = acc[y][e];
    write_row<T, kN>(a, it, row, d, m, l, x);
  }
}

// ---- host --------------------------------------------------------------------------------------------------

struct Plan {
  bool in_chunks;           // the kernels with tiles; otherwise rows that 16-byte copies cannot read
  int rows_max;             // rows of an item
  int step, unit;
  int item_tokens, item_heads, token_blocks, head_blocks, cluster, parts;
  int64_t items;
  int64_t covered_bytes, ml_bytes, o_bytes;
};

// Rows of whole 16-byte pieces on 16-byte boundaries.
int elem_bytes(int dtype) { return dtype == B200NA_E4M3 ? 1 : dtype == B200NA_F32 ? 4 : 2; }
bool reads_in_chunks(const b200na_kv_cache& c) {
  const int per = 16 / elem_bytes(c.dtype);
  const PagedPool k = paged_pool(c, false), v = paged_pool(c, true);
  return c.head_dim % per == 0 &&
         (reinterpret_cast<uintptr_t>(c.key) | reinterpret_cast<uintptr_t>(c.value)) % 16 == 0 &&
         (k.page | k.token | k.head | v.page | v.token | v.head) % per == 0;
}

int64_t round_up(int64_t n) { return (n + 255) / 256 * 256; }

int make_plan(Plan* p, int B, int T, int Hq, const b200na_kv_cache* cache, int max_pages, int kernel,
              int dilation, int dtype) {
  const int rc = check_cache(cache, reinterpret_cast<const int*>(16), 0, max_pages, dtype, B);
  if (rc != B200NA_OK) return rc;
  if (T < 0 || Hq < 1 || Hq % cache->heads || Hq > 65536 || kernel < 0 || dilation < 1)
    return B200NA_ERR_INVALID_ARGUMENT;
  const int group = Hq / cache->heads, D = cache->head_dim;
  p->in_chunks = reads_in_chunks(*cache);
  const int single = group == 1 && (T <= 1 || dilation > 1);        // one row an item
  p->rows_max = !p->in_chunks ? (single ? 1 : 8) : dtype == B200NA_F32 ? 8 : 16;
  p->item_heads = group < p->rows_max ? group : p->rows_max;
  p->head_blocks = (group + p->item_heads - 1) / p->item_heads;
  p->item_tokens = dilation > 1 ? 1 : p->rows_max / p->item_heads;
  if (p->item_tokens > T) p->item_tokens = T < 1 ? 1 : T;
  const int rows = p->item_tokens * p->item_heads;
  if (p->rows_max == 16 && rows <= 8) p->rows_max = 8;
  else if (p->in_chunks && dtype == B200NA_F32 && rows <= 4) p->rows_max = rows <= 2 ? 2 : 4;
  p->token_blocks = (int)(((int64_t)T + p->item_tokens - 1) / p->item_tokens);
  // a tile for each of a block's warps
  const int elem = elem_bytes(cache->dtype);
  p->step = kWarps * (p->in_chunks ? tile_keys((D <= 64 ? 64 : D <= 128 ? 128 : 256) * elem, elem) : 32);
  p->items = (int64_t)cache->heads * p->token_blocks * p->head_blocks;
  if (B > 0 && p->items * p->rows_max > (int64_t)0x7fffffff / B) return B200NA_ERR_INVALID_ARGUMENT;
  // units if every sequence were as long as the table allows: larger ones where 31 bits would not count them
  int64_t most = (int64_t)max_pages * cache->page_size;
  if (most > 0x7fffffff - 4096) return B200NA_ERR_UNSUPPORTED;
  if (kernel > 0 && most > (int64_t)kernel + p->item_tokens) most = (int64_t)kernel + p->item_tokens;
  p->unit = p->step;
  while (B * p->items * (most / p->unit + 1) > 0x7fffffff && p->unit <= most && p->unit < 1 << 30) p->unit *= 2;
  const int64_t units = B * p->items * (most / p->unit + 1);
  if (units > 0x7fffffff) return B200NA_ERR_INVALID_ARGUMENT;
  const int held = p->in_chunks && D > 128 && elem > 1 ? kMostParts / 2 : kMostParts;   // (Tile::kBlocks)
  p->parts = (int)(units < held ? (units < 1 ? 1 : units) : held);
  // Clusters of the largest size that leaves every block a place of its own (of one block where the items alone
  // have none), where a block's share is bounded. Against ranges and their join (us; bf16, 4 heads of 128 channels, units
  // of 64 keys):
  //  - equal lengths, a place for each block: 256 items of 33 units (window 2048) 47 / 53; 16 sequences, 10, 20 and 40
  //    units a block 23 / 27, 35 / 39, 60 / 64; 64 sequences, 20, 40 and 80 units 33 / 38, 58 / 63, 107 / 114
  //  - lengths from almost nothing to the table's: 64 sequences, 10, 20, 40 and 80 units a block 17 / 23, 27 / 34,
  //    46 / 46, 82 / 69; 16 sequences, 5, 10, 20 and 40 units 12.6 / 15.1, 19 / 19, 30 / 29, 50 / 42
  //  - more items than places, 33 units each: 300 items 77 / 61, 360 84 / 71, 440 86 / 85, 512 90 / 96, 592 103 / 106,
  //    680 129 / 124, 1024 176 / 178
  //  - few items, so that eight blocks each leave places unused: 4 sequences, 4, 10, 20 and 40 units a block 12.5 / 12.9,
  //    18.9 / 17.1, 29.5 / 27.2, 48 / 40, of lengths that differ 8 times 18 / 17 (10), 28 / 22 (20), 46 / 31 (40)
  // So 40 is where uneven lengths take what the join costs, with items that fill the GPU. A little above 296 items, and
  // with a few long sequences, ranges would take up to a third less.
  const int64_t item_units = most / p->unit + 1, item_count = B * p->items;
  p->cluster = 1;
  while (p->cluster < 8 && p->cluster < item_units && item_count * p->cluster * 2 <= held) p->cluster *= 2;
  if (item_units > kClusterUnits * p->cluster) p->cluster = 0;
  if (p->cluster) {
    p->covered_bytes = p->ml_bytes = p->o_bytes = 0;
    return B200NA_OK;
  }
  p->covered_bytes = round_up(B * p->items * (int64_t)sizeof(int2));
  p->ml_bytes = round_up((int64_t)2 * p->parts * p->rows_max * sizeof(float2));
  p->o_bytes = round_up((int64_t)2 * p->parts * p->rows_max * cache->head_dim * sizeof(float));
  return B200NA_OK;
}

template <class K>
int opt_in(K kernel, size_t bytes) {
  if (bytes > 32 * 1024)   // (48 KB with the static arrays)
    B200NA_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
  return B200NA_OK;
}

// The first launch: clusters that have an item each, or as many blocks as there are ranges.
int launch(void (*kernel)(DecodeArgs), const DecodeArgs& a, size_t smem, cudaStream_t s) {
  const int rc = opt_in(kernel, smem);
  if (rc != B200NA_OK) return rc;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(a.cluster ? (unsigned)a.B * a.items * a.cluster : (unsigned)a.parts);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = a.cluster;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = a.cluster > 1 ? 1 : 0;
  B200NA_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, a));
  return B200NA_OK;
}

template <class T, class P, int kRows, int kD32>
int launch_simt(const DecodeArgs& a, cudaStream_t s) {
  const size_t smem = (size_t)(2 + kWarps) * kRows * a.D * sizeof(float);
  return launch(decode_simt_kernel<T, P, kRows, kD32>, a, smem, s);
}
template <class T, class P>
int run_simt(const DecodeArgs& a, int rows_max, cudaStream_t s) {
  if (rows_max == 1) return a.D <= 128 ? launch_simt<T, P, 1, 4>(a, s) : launch_simt<T, P, 1, 8>(a, s);
  return a.D <= 128 ? launch_simt<T, P, 8, 4>(a, s) : launch_simt<T, P, 8, 8>(a, s);
}

template <bool k8, int kDP, int kRows> int launch_fma(const DecodeArgs& a, cudaStream_t s) {
  return launch(decode_fma_kernel<k8, kDP, kRows>, a, Tile<kDP, k8 ? 1 : 4, kRows, true>::bytes(a.D), s);
}
template <bool k8, int kRows> int run_fma(const DecodeArgs& a, cudaStream_t s) {
  return a.D <= 64 ? launch_fma<k8, 64, kRows>(a, s)
         : a.D <= 128 ? launch_fma<k8, 128, kRows>(a, s) : launch_fma<k8, 256, kRows>(a, s);
}

template <class T, bool k8, int kDP, int kRows>
int launch_mma(const DecodeArgs& a, cudaStream_t s) {
  return launch(decode_mma_kernel<T, k8, kDP, kRows>, a, Tile<kDP, k8 ? 1 : 2, kRows, false>::bytes(a.D), s);
}
template <class T, bool k8, int kRows> int run_mma_rows(const DecodeArgs& a, cudaStream_t s) {
  return a.D <= 64 ? launch_mma<T, k8, 64, kRows>(a, s)
         : a.D <= 128 ? launch_mma<T, k8, 128, kRows>(a, s) : launch_mma<T, k8, 256, kRows>(a, s);
}
// rows of whole 16-byte pieces
template <class T>
int run_tiles(const DecodeArgs& a, bool eight_bits, int rows_max, cudaStream_t s) {
  if constexpr (std::is_same<T, float>::value) {
    if (eight_bits)
      return rows_max == 2 ? run_fma<true, 2>(a, s) : rows_max == 4 ? run_fma<true, 4>(a, s) : run_fma<true, 8>(a, s);
    return rows_max == 2 ? run_fma<false, 2>(a, s) : rows_max == 4 ? run_fma<false, 4>(a, s) : run_fma<false, 8>(a, s);
  } else {
    if (eight_bits) return rows_max == 8 ? run_mma_rows<T, true, 8>(a, s) : run_mma_rows<T, true, 16>(a, s);
    return rows_max == 8 ? run_mma_rows<T, false, 8>(a, s) : run_mma_rows<T, false, 16>(a, s);
  }
}

template <class T>
int run(const DecodeArgs& a, bool in_chunks, int cache_dtype, int rows_max, cudaStream_t s) {
  int rc = in_chunks ? run_tiles<T>(a, cache_dtype == B200NA_E4M3, rows_max, s)
           : cache_dtype == B200NA_E4M3 ? run_simt<T, __nv_fp8_e4m3>(a, rows_max, s) : run_simt<T, T>(a, rows_max, s);
  if (rc != B200NA_OK || a.cluster) return rc;
  cudaLaunchConfig_t cfg{};
  const int64_t warps = (int64_t)a.B * a.items * rows_max;
  const int64_t blocks = (warps + kWarps - 1) / kWarps;
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  B200NA_CUDA_TRY(in_chunks ? cudaLaunchKernelEx(&cfg, decode_join_kernel<T, 4>, a, rows_max)
                            : cudaLaunchKernelEx(&cfg, decode_join_kernel<T, 1>, a, rows_max));
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
  if (!query || !out || !lengths || (!workspace && !p.cluster)) return B200NA_ERR_INVALID_ARGUMENT;
  if ((reinterpret_cast<uintptr_t>(workspace) | reinterpret_cast<uintptr_t>(out)) % 16) return B200NA_ERR_ALIGNMENT;
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
  a.capacity = cache->pages > 0 ? max_pages * cache->page_size : 0;
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
  a.items = (uint32_t)p.items;
  a.parts = p.parts;
  a.cluster = p.cluster;
  a.step = p.step;
  a.unit = p.unit;
  while (1 << a.unit_log2 < a.unit) ++a.unit_log2;
  while (1 << a.cluster_log2 < a.cluster) ++a.cluster_log2;
  a.q_wide = reinterpret_cast<uintptr_t>(query) % 16 == 0 && (a.q_batch | a.q_token | a.q_head) % (16 / elem_bytes(dtype)) == 0;
  a.same_strides = a.key.page == a.value.page && a.key.token == a.value.token &&
                   a.key.s_page == a.value.s_page && a.key.s_token == a.value.s_token;
  uint8_t* w = static_cast<uint8_t*>(workspace);
  a.covered = reinterpret_cast<int2*>(w);
  a.part_ml = reinterpret_cast<float2*>(w + p.covered_bytes);
  a.part_o = reinterpret_cast<float*>(w + p.covered_bytes + p.ml_bytes);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  switch (dtype) {
    case B200NA_F32: return run<float>(a, p.in_chunks, cache->dtype, p.rows_max, s);
    case B200NA_F16: return run<__half>(a, p.in_chunks, cache->dtype, p.rows_max, s);
    default: return run<__nv_bfloat16>(a, p.in_chunks, cache->dtype, p.rows_max, s);
  }
}
