// Attention of new tokens over a paged key/value cache: chunks of a prompt,
// single decode tokens and ragged mixtures of both.
//
// Sequence b has seq_lens[b] cached tokens (the new ones included), token j in
// row j % page_size of page page_table[b][j / page_size]; its new tokens are
// rows [cu_q[b], cu_q[b + 1]) of q and sit at the end of the sequence. With
// base = seq_lens[b] - (cu_q[b + 1] - cu_q[b]), query i attends to the keys
// j <= base + i:
//   o_i = sum_j p_ij v_j,  p_ij = softmax_j(scale q_i . k_j)
// and a query without any key (base + i < 0) returns zeros.
//
// Floor: every live K/V row is read from HBM once per KV head; 4 D operations
// per (query head, key) pair on the tensor cores and one exponential.
//
// Both kernels are persistent: the work items -- (sequence, KV heads, query
// rows) with their number of key tiles -- are listed, and the tiles of all
// items, in order, cut into equal contiguous shares, one per CTA: by every CTA
// for itself where a sequence is one item per head group (few query rows), by
// a small schedule kernel otherwise.
// A long context with few queries is thereby spread over the whole GPU and a
// ragged batch stays balanced without the host knowing any length. Items cut
// between CTAs leave FP32 partials (max, sum, output) in the workspace, which a
// third kernel joins in CTA order with the whole GPU. (Joined by the last CTA
// of an item, they took up to 24 us: 590 KB through one SM.)
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "tc.cuh"
#include "types16.cuh"

namespace mfb {
namespace paged {

constexpr int MAX_B = 8192;
constexpr int MAX_SMS = 160;  // bounds the workspace: shares are at most 2 (few rows) or 1 (chunks) per SM

__device__ int g_status;  // id of a bounded wait that gave up, or kBadPage / kBadLength
constexpr int kBadPage = 1001, kBadLength = 1002;

// A work item, and the record of a share: the item its first unit lies in.
struct __align__(16) Item {
  int b, hg;         // sequence, KV-head group
  int tok0, ntok;    // query tokens: q rows tok0 .. tok0 + ntok - 1
  int pos0;          // position of the first of them (negative: no keys yet)
  int keys;          // keys the last one sees (0 if none)
  int tiles;         // units: key tiles, at least 1 (0: no query tokens)
  int first;         // weight of the items before this one
  int shift, index;  // a unit weighs 1 << shift; position in the list
  int pad[2];
};

// The total weight is cut into `shares` ranges, the first `rest` of them one
// longer than `base`. A unit belongs to the share its weight starts in.
struct Header {
  int total, shares, base, rest;
  int cuts, pad[3];  // items of more than one share
};

struct Params {
  const uint16_t* q;
  uint16_t* o;
  float* lse;
  const int* cu_q;
  const int* seq_lens;
  const int* page_table;
  Header* head;
  Item* items;
  Item* starts;    // [grid] each share's first item
  Item* cuts;      // [grid] the items of more than one share, in any order
  float* part_o;   // [slots][part_rows] x D
  float2* part_ml; // [slots][part_rows]
  int N, B, H, Hk, G, max_q, max_pages, num_pages, page_shift;
  int tok_item;    // query tokens per item
  int hc;          // KV heads per item
  int unit;        // keys per unit
  int grid, max_items, part_rows;
  float scale_log2;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];\n" : "=r"(v) : "r"(a));
  return v;
}

// ---------------------------------------------------------------------------
// Schedule: one block. Items of sequence b: head groups x query blocks.
// ---------------------------------------------------------------------------
constexpr int SCHED_THREADS = 1024;

// Exclusive block scan of one value per thread; returns the prefix, total in *sum.
template <typename I>
__device__ __forceinline__ I block_scan(I v, I* warp_sums, I* sum) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  I incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const I y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  __syncthreads();  // the previous scan's readers are done with warp_sums
  if (lane == 31) warp_sums[warp] = incl;
  __syncthreads();
  if (warp == 0) {
    I w = warp_sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const I y = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += y;
    }
    warp_sums[lane] = w;
  }
  __syncthreads();
  *sum = warp_sums[31];
  return incl - v + (warp ? warp_sums[warp - 1] : 0);
}

// Weight a share holds at least, in either kernel: a cut costs its partials and
// their join, a long share leaves SMs idle. Rows, with 1, 2, 4, 8 and 16: one token
// over 200 keys 12.2, 12.5, 14.3, 18.3, 18.4 us; over 4000 14.5, 14.1, 14.5, 17.7,
// 22.6; 8 over up to 3000 16.6, 16.6, 16.8, 18.6, 24.6; 64 over up to 4096 58.5 in
// all. Tiles, with 2, 4, 8 and 16: 64 tokens over 300 keys 18.5, 20.6, 26.8, 43.4;
// 4 x 64 over 2000 21.7, 20.4, 22.7, 26.6; nine ragged chunks 38.9, 38.8, 38.9, 44.6.
constexpr int MIN_SHARE = 4;
__device__ __forceinline__ Header cut(const Params& p, int total) {
  Header h;
  h.total = total;
  h.shares = max(1, min(p.grid, total / MIN_SHARE));
  h.base = total / h.shares;
  h.rest = total - h.base * h.shares;
  h.cuts = h.pad[0] = h.pad[1] = h.pad[2] = 0;
  return h;
}
__device__ __forceinline__ int share_begin(const Header& h, int i) { return i * h.base + min(i, h.rest); }
__device__ __forceinline__ int share_of(const Header& h, int x) {
  const int split = h.rest * (h.base + 1);
  return x < split ? x / (h.base + 1) : h.rest + (x - split) / h.base;
}
// First unit of an item that belongs to the share beginning at weight x.
__device__ __forceinline__ int unit_at(const Item& w, int x) {
  return min(w.tiles, max(0, (x - w.first + (1 << w.shift) - 1) >> w.shift));
}
__device__ __forceinline__ int last_weight(const Item& w) { return w.first + ((w.tiles - 1) << w.shift); }

// Query rows of sequence b inside q: arguments that contradict each other
// (cu_q outside [0, N] or decreasing, more than max_q new tokens, lengths
// outside the page table) are clamped, so no access leaves the buffers, and
// recorded in the status word.
__device__ __forceinline__ void sequence(const Params& p, int b, int* q0, int* nq, int* base, int* len) {
  const int c0 = p.cu_q[b], c1 = p.cu_q[b + 1], s = p.seq_lens[b];
  const int lo = min(max(c0, 0), p.N), hi = min(max(c1, lo), p.N);
  const long long cap = (long long)p.max_pages << p.page_shift;
  *q0 = lo;
  *nq = min(hi - lo, p.max_q);
  *len = (int)min((long long)max(s, 0), cap);
  *base = *len - (hi - lo);
  if (c0 != lo || c1 != hi || *nq != hi - lo || *len != s) atomicCAS(&g_status, 0, kBadLength);
}

// Sequence b has cdiv(new tokens, tok_item) items per head.
__global__ void __launch_bounds__(SCHED_THREADS) schedule_kernel(Params p) {
  allow_dependents();
  extern __shared__ int item_base[];  // [B] items before each sequence
  __shared__ int warp_sums[32], s_cuts;
  __shared__ long long wide_sums[32];
  const int tid = threadIdx.x;
  if (tid == 0) s_cuts = 0;
  // Sequences whose cu_q contradict each other may claim the same rows, each all
  // of them: their items are counted in 64 bits and those past max_items dropped.
  long long listed = 0;
  for (int b0 = 0; b0 < p.B; b0 += SCHED_THREADS) {
    const int b = b0 + tid;
    int q0, nq = 0, base, len;
    long long sum;
    if (b < p.B) sequence(p, b, &q0, &nq, &base, &len);
    const long long pre = block_scan((long long)cdiv(nq, p.tok_item) * p.Hk, wide_sums, &sum);
    if (b < p.B) item_base[b] = (int)min(listed + pre, (long long)p.max_items);
    listed += sum;
  }
  const int items = (int)min(listed, (long long)p.max_items);
  __syncthreads();
  auto make = [&](int i) {
    Item it;
    int q0, nq, base, len, lo = 0, hi = p.B - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (item_base[mid] <= i) lo = mid;
      else hi = mid - 1;
    }
    it.b = lo;
    sequence(p, lo, &q0, &nq, &base, &len);
    const int blocks = cdiv(nq, p.tok_item), local = i - item_base[lo];
    it.hg = local / blocks;
    const int t0 = (local - it.hg * blocks) * p.tok_item;
    it.tok0 = q0 + t0;
    it.ntok = min(p.tok_item, nq - t0);
    it.pos0 = base + t0;
    it.keys = min(max(it.pos0 + it.ntok, 0), len);
    it.tiles = it.ntok > 0 ? max(1, cdiv(it.keys, p.unit)) : 0;
    // Two query tiles share a unit's keys but need twice the softmax.
    it.shift = it.ntok * p.G > 128 ? 1 : 0;
    it.index = i;
    it.first = it.pad[0] = it.pad[1] = 0;
    return it;
  };
  // A pass for the total weight, one for prefixes and shares; a single block
  // of items keeps the first pass's results.
  Item mine{};
  int total = 0, pre = 0, sum;
  for (int i0 = 0; i0 < items; i0 += SCHED_THREADS) {
    const int i = i0 + tid;
    if (i < items) mine = make(i);
    pre = block_scan(i < items ? mine.tiles << mine.shift : 0, warp_sums, &sum);
    total += sum;
  }
  Header h = cut(p, total);
  int carry = 0;
  for (int i0 = 0; i0 < items; i0 += SCHED_THREADS) {
    const int i = i0 + tid;
    if (items > SCHED_THREADS) {
      if (i < items) mine = make(i);
      pre = block_scan(i < items ? mine.tiles << mine.shift : 0, warp_sums, &sum);
    }
    if (i < items) {
      mine.first = carry + pre;
      p.items[i] = mine;
      // Shares that begin in this item.
      const int end = mine.first + (mine.tiles << mine.shift);
      if (mine.tiles) {
        int s = share_of(h, mine.first);
        if (s != share_of(h, last_weight(mine))) p.cuts[atomicAdd(&s_cuts, 1)] = mine;
        if (share_begin(h, s) < mine.first) ++s;
        for (; s < h.shares && share_begin(h, s) < end; ++s) p.starts[s] = mine;
      }
    }
    carry += sum;
  }
  __syncthreads();
  h.cuts = s_cuts;
  if (tid == 0) *p.head = h;
}

// ---------------------------------------------------------------------------
// Joining the partials of a cut item. Segment (share c, which) owns a slot:
// which = 0 where the share begins inside (or at) the item, 1 where the item
// begins later in the share. Of a share's segments only the first and the last
// can be cut, and of two of them only the first has which = 0.
// ---------------------------------------------------------------------------
__device__ __forceinline__ int slot_of(const Header& h, const Item& w, int c) {
  return 2 * c + (share_begin(h, c) < w.first ? 1 : 0);
}

// Layouts of a slot's [rows][D] floats, in float4. ROWS32 interleaves blocks of
// 32 rows, [row / 32][D / 4][row % 32]: a warp whose lanes own rows then writes
// and reads whole lines. Otherwise rows are contiguous.
template <int D, bool ROWS32>
__device__ __forceinline__ long long part_at(const Params& p, int slot, int row, int d4) {
  const long long r = (long long)slot * p.part_rows + row;
  return ROWS32 ? ((r >> 5) * (D / 4) + d4) * 32 + (r & 31) : r * (D / 4) + d4;
}

// No key: -inf. A NaN sum (a query that is not finite) stays NaN, like the output beside it.
__device__ __forceinline__ float lse_of(float m, float l) {
  return l == 0.f ? -INFINITY : (m + __log2f(l)) * 0.6931471805599453f;
}

// Joins the cut items. Each is split by rows over an equal part of the blocks;
// a block's threads are float4 columns x lanes, a lane taking every lanes-th
// part. U columns x K parts are in flight per thread: a join waits for the
// latency of its loads. The lanes meet in shared memory, in lane order.
constexpr int JOIN_THREADS = 256;

template <typename T, int D, bool ROWS32, int U, int K>
__device__ __forceinline__ void join_rows(const Params& p, const Header& h, const Item& w, int c0, int n, int r0,
                                          int r1, float4* s_o, float2* s_ml) {
  const int tid = threadIdx.x, cols = (r1 - r0) * (D / 4), nrow = r1 - r0;
  int lanes = 1;
  while (U == 1 && lanes * 2 * cols <= JOIN_THREADS && lanes * K < n) lanes *= 2;
  const int wide = JOIN_THREADS / lanes, lane = tid / wide;
  for (int x0 = tid % wide; x0 - tid % wide < cols; x0 += U * wide) {
    int row[U], d4[U];
    float m[U], l[U];
    float4 acc[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int x = min(x0 + u * wide, cols - 1);
      // Rows run fastest where they do in the slot.
      const int q = ROWS32 ? x / nrow : x / (D / 4);
      row[u] = r0 + (ROWS32 ? x - q * nrow : q);
      d4[u] = ROWS32 ? q : x - q * (D / 4);
      m[u] = -INFINITY;
      l[u] = 0.f;
      acc[u] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    for (int k0 = lane; k0 < n; k0 += K * lanes) {
      float2 ml[K][U];
      float4 ov[K][U];
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int part = k0 + k * lanes;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          ml[k][u] = make_float2(-INFINITY, 0.f);
          ov[k][u] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (part < n) {
            const int slot = slot_of(h, w, c0 + part);
            ml[k][u] = p.part_ml[(long long)slot * p.part_rows + row[u]];
            ov[k][u] = reinterpret_cast<const float4*>(p.part_o)[part_at<D, ROWS32>(p, slot, row[u], d4[u])];
          }
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float mn = m[u];
#pragma unroll
        for (int k = 0; k < K; ++k) mn = fmaxf(mn, ml[k][u].x);
        const float ref = mn == -INFINITY ? 0.f : mn, a = ex2(m[u] - ref);
        l[u] *= a, acc[u].x *= a, acc[u].y *= a, acc[u].z *= a, acc[u].w *= a;
#pragma unroll
        for (int k = 0; k < K; ++k) {
          const float g = ex2(ml[k][u].x - ref);
          l[u] = fmaf(ml[k][u].y, g, l[u]);
          acc[u].x = fmaf(ov[k][u].x, g, acc[u].x);
          acc[u].y = fmaf(ov[k][u].y, g, acc[u].y);
          acc[u].z = fmaf(ov[k][u].z, g, acc[u].z);
          acc[u].w = fmaf(ov[k][u].w, g, acc[u].w);
        }
        m[u] = mn;
      }
    }
    if (lanes > 1) {  // U == 1
      __syncthreads();
      s_o[tid] = acc[0];
      s_ml[tid] = make_float2(m[0], l[0]);
      __syncthreads();
      for (int k = 1; lane == 0 && k < lanes; ++k) {
        const float2 o = s_ml[tid + k * wide];
        const float4 v = s_o[tid + k * wide];
        const float mn = fmaxf(m[0], o.x), ref = mn == -INFINITY ? 0.f : mn, a = ex2(m[0] - ref), g = ex2(o.x - ref);
        l[0] = l[0] * a + o.y * g;
        acc[0] = make_float4(acc[0].x * a + v.x * g, acc[0].y * a + v.y * g, acc[0].z * a + v.z * g,
                             acc[0].w * a + v.w * g);
        m[0] = mn;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (lane > 0 || x0 + u * wide >= cols) continue;
      // Row of the slot: (token x group, KV head of the item).
      const int rt = row[u] / p.hc, hh = row[u] - rt * p.hc, t = rt / p.G;
      const long long at = (long long)(w.tok0 + t) * p.H + (w.hg * p.hc + hh) * p.G + (rt - t * p.G);
      const float inv = l[u] > 0.f ? 1.f / l[u] : 0.f;
      uint2 out;
      out.x = Num16<T>::pack2(acc[u].x * inv, acc[u].y * inv);
      out.y = Num16<T>::pack2(acc[u].z * inv, acc[u].w * inv);
      *reinterpret_cast<uint2*>(p.o + at * D + d4[u] * 4) = out;
      if (p.lse && d4[u] == 0) p.lse[at] = lse_of(m[u], l[u]);
    }
  }
}

template <typename T, int D, bool ROWS32>
__global__ void __launch_bounds__(JOIN_THREADS, 4) join_kernel(Params p) {
  __shared__ float4 s_o[JOIN_THREADS];
  __shared__ float2 s_ml[JOIN_THREADS];
  allow_dependents();
  wait_prerequisites();
  const Header h = *p.head;
  if (h.cuts == 0) return;
  const int chunks = max(1, (int)gridDim.x / h.cuts);  // blocks per item (cuts <= gridDim.x: fewer than shares)
  const int k = blockIdx.x / chunks, chunk = blockIdx.x - k * chunks;
  if (k >= h.cuts) return;
  const Item w = p.cuts[k];
  const int rows = w.ntok * p.G * p.hc, per = cdiv(rows, chunks), r0 = chunk * per, r1 = min(rows, r0 + per);
  if (r0 >= r1) return;
  const int c0 = share_of(h, w.first), n = share_of(h, last_weight(w)) - c0 + 1;
  // The last form for all: 159.5 instead of 155.2 us for two 2048-token chunks, 36.9
  // instead of 35.0 for 20 ragged ones; without the middle one 154.9 and 37.0.
  if (n <= 2) join_rows<T, D, ROWS32, 4, 2>(p, h, w, c0, n, r0, r1, s_o, s_ml);
  else if (n <= 4) join_rows<T, D, ROWS32, 2, 4>(p, h, w, c0, n, r0, r1, s_o, s_ml);
  else join_rows<T, D, ROWS32, 1, 8>(p, h, w, c0, n, r0, r1, s_o, s_ml);
}

// Key tile boxes of one unit: rows of a page, at most the unit's.
__device__ __forceinline__ int page_id(const Params& p, int b, int key) {
  const int id = p.page_table[(long long)b * p.max_pages + (key >> p.page_shift)];
  if ((unsigned)id < (unsigned)p.num_pages) return id;
  atomicCAS(&g_status, 0, kBadPage);
  return p.num_pages;  // outside the tensor: the load fills zeros
}

// Page ids of a stream of tiles, 32 boxes ahead: lane l holds the id of box
// 32 window + l (a box is `br` keys of one page, a tile `nb` boxes, a power of
// two up to 32). The next window's ids are read while this one is used, so
// the loads never wait for a table lookup.
struct PageIds {
  int b, br, nb, end;  // sequence, keys per box, boxes per tile, keys that are needed
  int window, cur, next;
  __device__ __forceinline__ int fetch(const Params& p, int w) const {
    // Unsigned: a window ahead of a sequence that ends just below 2^31 lies above it.
    const unsigned key = ((unsigned)w * 32u + (threadIdx.x & 31u)) * (unsigned)br;
    return key < (unsigned)end ? page_id(p, b, (int)key) : 0;
  }
  __device__ __forceinline__ PageIds(const Params& p, int seq, int rows, int boxes, int tile, int keys)
      : b(seq), br(rows), nb(boxes), end(keys), window(tile * boxes >> 5) {
    cur = fetch(p, window);
    next = fetch(p, window + 1);
  }
  // The id of box `lane % nb` (or any of the caller's choice) of a tile; tiles in order.
  __device__ __forceinline__ int get(const Params& p, int tile, int box) {
    if (tile * nb >> 5 != window) {
      ++window;
      cur = next;
      next = fetch(p, window + 1);
    }
    return __shfl_sync(0xffffffffu, cur, (tile * nb & 31) + box);
  }
};

// 4-D tiled load, no multicast.
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w,
                                            uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];\n" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
      : "memory");
}

// Steps to the next item of a share that ends at weight x1; false at its end.
__device__ __forceinline__ bool advance(const Params& p, Item& w, int x1) {
  if (w.first + (w.tiles << w.shift) >= x1) return false;
  w = p.items[w.index + 1];
  return true;
}

// ---------------------------------------------------------------------------
// Few query rows per KV head (new tokens x group <= 16): bandwidth-bound.
//
// A unit is 128 / hc keys of hc KV heads: 16 KB of K and of V per 64 head
// dims. A producer warp streams units through a ring (one TMA box per page
// touched); eight compute warps take 16 keys of one head each on the
// warp-level MMA (m16n8k16, the query rows as A: the kernel waits for memory,
// not for these products), with an FP32 online softmax. Probabilities are
// rounded to the cache's 16-bit type for the P.V product, as the fixed-capacity
// decode does; their sum is taken before the rounding.
// ---------------------------------------------------------------------------
constexpr int DW = 8;                    // compute warps
constexpr int D_THREADS = 32 * (DW + 1);

// Whether every warp of the 256 compute threads says yes.
__device__ __forceinline__ bool all_came(bool mine) {
  int all;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.s32 p, %1, 0;\n barrier.red.and.pred q, 1, 256, p;\n selp.s32 %0, 1, 0, q;\n}\n"
      : "=r"(all)
      : "r"((int)mine)
      : "memory");
  return all != 0;
}

// Item i (sequence i / groups, head group i % groups); its weight is its tiles.
__device__ __forceinline__ Item few_item(const Params& p, int i, int first) {
  Item w;
  int q0, nq, base, len;
  const int groups = p.Hk / p.hc;
  w.b = i / groups;
  w.hg = i - w.b * groups;
  sequence(p, w.b, &q0, &nq, &base, &len);
  w.tok0 = q0;
  w.ntok = nq;
  w.pos0 = base;
  w.keys = min(max(base + nq, 0), len);
  w.tiles = nq > 0 ? max(1, cdiv(w.keys, p.unit)) : 0;
  w.first = first;
  w.shift = 0;
  w.index = i;
  return w;
}
__device__ __forceinline__ bool few_advance(const Params& p, Item& w, int x1) {
  if (w.first + w.tiles >= x1) return false;
  w = few_item(p, w.index + 1, w.first + w.tiles);
  return true;
}

struct DLayout {
  uint32_t merge, q, bars, total;
};
__host__ __device__ inline DLayout dlayout(int D, int stages, int rows, int hc) {
  DLayout L;
  L.merge = (uint32_t)stages * 2u * 16384u * (uint32_t)(D / 64);
  const uint32_t m = hc < 8 ? 8u * (uint32_t)rows * (uint32_t)(D + 4) * 4u : 0u;  // [warp][row]{o[D], m, l}
  L.q = L.merge + m;  // an item's query rows, [token][head of the item][D]
  L.bars = L.q + (uint32_t)(rows * hc * D) * 2u;
  L.total = 1024 + L.bars + 16u * (uint32_t)stages + 16u;
  return L;
}

template <typename T, int D, bool R16>
__global__ void __launch_bounds__(D_THREADS, D == 64 ? 2 : 1)
    few_rows_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, Params p,
                    int stages, int rows_max) {
  constexpr int DH = D / 64;
  constexpr uint32_t kStage = 2u * 16384u * DH;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t sb = smem_u32(smem);
  const DLayout lay = dlayout(D, stages, rows_max, p.hc);
  float* merge = reinterpret_cast<float*>(smem + lay.merge);
  __shared__ int s_sums[DW + 1], s_cuts;
  __shared__ Item s_start, s_item;  // the share's first item, and the one whose queries lie in shared memory
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  auto full_bar = [&](int s) { return sb + lay.bars + 8u * s; };
  auto empty_bar = [&](int s) { return sb + lay.bars + 8u * (stages + s); };
  const uint32_t q_full = empty_bar(stages), q_empty = q_full + 8;
  if (tid == 0) {
    for (int s = 0; s < stages; ++s) {
      tc::mbar_init(full_bar(s), 1);
      tc::mbar_init(empty_bar(s), DW);
    }
    tc::mbar_init(q_full, 1);
    tc::mbar_init(q_empty, DW);
    tc::mbar_fence_init();
    tc::tma_prefetch_desc(&tk);
    tc::tma_prefetch_desc(&tv);
  }
  allow_dependents();
  // The schedule: each thread sums a run of items, and the one whose run holds
  // this share's first unit looks it up.
  const int items = p.B * (p.Hk / p.hc), per = cdiv(items, D_THREADS);
  const int i0 = min(items, tid * per), i1 = min(items, i0 + per);
  int local = 0;
  for (int i = i0; i < i1; ++i) local += few_item(p, i, 0).tiles;
  int incl = local;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  if (lane == 31) s_sums[warp] = incl;
  __syncthreads();
  int before = incl - local, total = 0;
#pragma unroll
  for (int w = 0; w <= DW; ++w) {
    if (w < warp) before += s_sums[w];
    total += s_sums[w];
  }
  const Header head = cut(p, total);
  const int share = blockIdx.x;
  if (share == 0) {
    // The first CTA lists the cut items for the join.
    if (tid == 0) s_cuts = 0;
    __syncthreads();
    for (int i = i0, first = before; total && i < i1; ++i) {
      const Item w = few_item(p, i, first);
      first += w.tiles;
      if (w.tiles && share_of(head, w.first) != share_of(head, last_weight(w))) p.cuts[atomicAdd(&s_cuts, 1)] = w;
    }
    __syncthreads();
    if (tid == 0) {
      Header h = head;
      h.cuts = s_cuts;
      *p.head = h;
    }
  }
  if (share >= head.shares || total == 0) return;
  const int x0 = share_begin(head, share), x1 = share_begin(head, share + 1);
  if (before <= x0 && x0 < before + local) {
    Item w = few_item(p, i0, before);
    while (w.first + w.tiles <= x0) w = few_item(p, w.index + 1, w.first + w.tiles);
    s_start = w;
  }
  __syncthreads();
  const int unit = p.unit, hc = p.hc;
  const int br = min(unit, 1 << p.page_shift), nb = unit / br;  // box rows, boxes per unit

  if (warp == DW) {
    // Producer: the boxes of K and V (and of both halves of 128-wide heads) are
    // issued by the lanes in parallel, all counted on the stage's barrier. An
    // item's record and queries go to shared memory while the item before it
    // still streams: a ring that stands still costs bandwidth that does not
    // come back.
    int it = 0, published = 0;
    bool ok = true;
    Item w = s_start;
    auto ids_of = [&](const Item& w) {
      return PageIds(p, w.b, br, nb, unit_at(w, x0), min(w.keys, unit_at(w, x1) * unit));
    };
    auto publish = [&](const Item& w) {
      ok = tc::mbar_wait_w(q_empty, (published & 1) ^ 1, &g_status, 4);
      if (!ok) return;
      ++published;
      const uint32_t bytes = (uint32_t)(hc * p.G * D) * 2u;  // of a token
      if (lane == 0) {
        s_item = w;
        tc::mbar_expect_tx(q_full, bytes * w.ntok);
      }
      __syncwarp();
      for (int t = lane; t < w.ntok; t += 32)
        tc::bulk_load(sb + lay.q + t * bytes, p.q + ((long long)(w.tok0 + t) * p.H + w.hg * hc * p.G) * D, bytes, q_full);
    };
    PageIds ids = ids_of(w);
    publish(w);
    while (ok) {
      const int u0 = unit_at(w, x0), u1 = unit_at(w, x1);
      Item next = w;
      PageIds next_ids = ids;
      const bool more = w.first + w.tiles < x1;
      for (int u = u0; u < u1; ++u, ++it) {
        const int st = it % stages;
        if (!(ok = tc::mbar_wait_w(empty_bar(st), ((it / stages) & 1) ^ 1, &g_status, 1))) break;
        const int live = min(nb, cdiv(max(w.keys - u * unit, 0), br));  // boxes that hold keys
        const uint32_t box = (uint32_t)br * hc * 128u;
        if (lane == 0) tc::mbar_expect_tx(full_bar(st), box * 2u * DH * live);
        __syncwarp();
        for (int j = lane; j - lane < live * 2 * DH; j += 32) {
          const int bx = j % max(live, 1), rest = j / max(live, 1);  // rest: half, then K or V
          const int pid = ids.get(p, u, bx);
          if (j < live * 2 * DH) {
            const int half = rest % DH, kv = rest / DH;
            const uint32_t dst = sb + st * kStage + kv * (kStage / 2) + half * 16384u + bx * box;
            tma_load_4d(dst, kv ? &tv : &tk, half * 64, (u * unit + bx * br) & ((1 << p.page_shift) - 1), w.hg * hc,
                        pid, full_bar(st));
          }
        }
        if (more && u == min(u0 + stages, u1) - 1) {  // the units before this item's are consumed
          do {  // sequences without new tokens have no units
            few_advance(p, next, x1);
          } while (next.tiles == 0);
          next_ids = ids_of(next);
          publish(next);
          if (!ok) break;
        }
      }
      if (!ok || !more) break;
      w = next;
      ids = next_ids;
    }
    if (!ok)  // a wait gave up: let the copies in flight land before the CTA ends
      for (int f = max(0, it - stages); f < it; ++f) tc::mbar_wait_w(full_bar(f % stages), (f / stages) & 1, &g_status, 3);
    return;
  }

  // Compute warps: head hl of the item's hc, keys [16 sl, 16 sl + 16) of each unit.
  const int hl = warp % hc, sl = warp / hc, slices = DW / hc;
  const int g4 = lane >> 2, c4 = lane & 3;
  // ldmatrix row offsets of this lane in a 64-dim half of a stage's K or V.
  auto row_off = [&](int i) {
    const int pos = sl * 16 + i;
    return (uint32_t)((pos / br) * (br * hc * 128) + hl * br * 128 + (pos % br) * 128);
  };
  const int ki = (lane & 7) + ((lane >> 4) << 3), vi = (lane & 7) + ((lane >> 3) & 1) * 8;
  const uint32_t koff = row_off(ki), voff = row_off(vi);
  const int G = p.G;
  int it = 0;
  bool ok = true;
  auto finish = [&](const Item& w, int rh, int d4, float mm, float ll, const float4& a) {
    const int row = rh / hc, h = rh - row * hc;
    const float inv = ll > 0.f ? 1.f / ll : 0.f;
    const long long at = (long long)(w.tok0 + row / G) * p.H + (w.hg * hc + h) * G + row % G;
    uint2 out;
    out.x = Num16<T>::pack2(a.x * inv, a.y * inv);
    out.y = Num16<T>::pack2(a.z * inv, a.w * inv);
    *reinterpret_cast<uint2*>(p.o + at * D + d4 * 4) = out;
    if (p.lse && d4 == 0) p.lse[at] = lse_of(mm, ll);
  };
  Item w = s_start;
  for (int taken = 0;; ++taken) {
    // The next item that has units. Where the warps meet inside the loop they
    // also agree on whether it came.
    bool came = tc::mbar_wait_w(q_full, taken & 1, &g_status, 5);
    if (slices > 1) came = all_came(came);
    if (!came) break;
    w = s_item;
    const int u0 = unit_at(w, x0), u1 = unit_at(w, x1);
    const int rows = w.ntok * G, hk = w.hg * hc + hl;
    uint32_t qa[D / 16][4];
    int lim[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = g4 + 8 * e, t = r / G;
      const bool live = r < rows && (R16 || e == 0);
      lim[e] = live ? min(w.pos0 + t + 1, w.keys) : 0;
      const uint32_t qrow = sb + lay.q + (uint32_t)((t * hc + hl) * G + r % G) * (2u * D) + 4u * c4;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        qa[kk][e] = live ? lds32(qrow + kk * 32) : 0u;
        qa[kk][2 + e] = live ? lds32(qrow + kk * 32 + 16) : 0u;
      }
    }
    __syncwarp();
    if (lane == 0) tc::mbar_arrive(q_empty);
    float o[D / 8][4];
#pragma unroll
    for (int n = 0; n < D / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    for (int u = u0; u < u1; ++u, ++it) {
      const int st = it % stages;
      // After a wait that gave up the warp goes on without waiting, so that
      // the named barriers below still meet.
      if (ok) ok = tc::mbar_wait_w(full_bar(st), (it / stages) & 1, &g_status, 2);
      if (ok) {
        const uint32_t kt = sb + st * kStage, vt = kt + kStage / 2;
        const int key0 = u * unit + sl * 16;
        if (key0 < w.keys) {
          float sc[2][4];
#pragma unroll
          for (int n = 0; n < 2; ++n) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            uint32_t f[4];
            const int chunk = ((kk & 3) * 2 + ((lane >> 3) & 1)) ^ (ki & 7);
            ldmatrix_x4(kt + (kk >> 2) * 16384 + koff + chunk * 16, f[0], f[1], f[2], f[3]);
            Num16<T>::mma(sc[0], qa[kk], f);
            Num16<T>::mma(sc[1], qa[kk], f + 2);
          }
          float v[2][4];  // [row half][key of this lane]
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
              for (int c = 0; c < 2; ++c)
                v[e][2 * n + c] = key0 + n * 8 + 2 * c4 + c < lim[e] ? sc[n][2 * e + c] * p.scale_log2 : -INFINITY;
          uint32_t pa[4] = {0u, 0u, 0u, 0u};
#pragma unroll
          for (int e = 0; e < (R16 ? 2 : 1); ++e) {
            float mx = fmaxf(fmaxf(v[e][0], v[e][1]), fmaxf(v[e][2], v[e][3]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const float mn = fmaxf(m[e], mx);
            const float ref = mn == -INFINITY ? 0.f : mn;
            const float a = ex2(m[e] - ref);
            m[e] = mn;
            float pr[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) pr[c] = ex2(v[e][c] - ref);
            l[e] = fmaf(l[e], a, (pr[0] + pr[1]) + (pr[2] + pr[3]));
#pragma unroll
            for (int n = 0; n < D / 8; ++n) o[n][2 * e] *= a, o[n][2 * e + 1] *= a;
            pa[e] = Num16<T>::pack2(pr[0], pr[1]);
            pa[2 + e] = Num16<T>::pack2(pr[2], pr[3]);
          }
          // Rows of V past the sequence hold whatever the page (or the ring)
          // held: zeros in their place, since 0 x NaN would not vanish.
          const bool tail = key0 + 16 > w.keys;
          uint32_t keep[2];
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const int k = key0 + n * 8 + 2 * c4;
            keep[n] = (k < w.keys ? 0xFFFFu : 0u) | (k + 1 < w.keys ? 0xFFFF0000u : 0u);
          }
#pragma unroll
          for (int nd = 0; nd < D / 16; ++nd) {
            uint32_t f[4];
            const int chunk = ((nd & 3) * 2 + (lane >> 4)) ^ (vi & 7);
            ldmatrix_x4_trans(vt + (nd >> 2) * 16384 + voff + chunk * 16, f[0], f[1], f[2], f[3]);
            if (tail) f[0] &= keep[0], f[1] &= keep[1], f[2] &= keep[0], f[3] &= keep[1];
            Num16<T>::mma(o[2 * nd], pa, f);
            Num16<T>::mma(o[2 * nd + 1], pa, f + 2);
          }
        }
      }
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(empty_bar(st));
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
    }
    const bool cut = u0 > 0 || u1 < w.tiles;
    const int slot = slot_of(head, w, share);
    if (slices == 1) {
#pragma unroll
      for (int e = 0; e < (R16 ? 2 : 1); ++e) {
        const int r = g4 + 8 * e;
        if (r >= rows) continue;
        if (!cut) {
          const float inv = l[e] > 0.f ? 1.f / l[e] : 0.f;
          const long long at = (long long)(w.tok0 + r / G) * p.H + hk * G + r % G;
          uint16_t* orow = p.o + at * D + 2 * c4;
#pragma unroll
          for (int n = 0; n < D / 8; ++n)
            *reinterpret_cast<uint32_t*>(orow + n * 8) = Num16<T>::pack2(o[n][2 * e] * inv, o[n][2 * e + 1] * inv);
          if (p.lse && c4 == 0) p.lse[at] = lse_of(m[e], l[e]);
        } else {
          const long long at = (long long)slot * p.part_rows + r * hc + hl;
#pragma unroll
          for (int n = 0; n < D / 8; ++n)
            *reinterpret_cast<float2*>(p.part_o + at * D + n * 8 + 2 * c4) = make_float2(o[n][2 * e], o[n][2 * e + 1]);
          if (c4 == 0) p.part_ml[at] = make_float2(m[e], l[e]);
        }
      }
    } else {
      // Join the warps that share a head through shared memory.
#pragma unroll
      for (int e = 0; e < (R16 ? 2 : 1); ++e) {
        const int r = g4 + 8 * e;
        if (r >= rows) continue;
        float* dst = merge + (warp * rows_max + r) * (D + 4);
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
          *reinterpret_cast<float2*>(dst + n * 8 + 2 * c4) = make_float2(o[n][2 * e], o[n][2 * e + 1]);
        if (c4 == 0) dst[D] = m[e], dst[D + 1] = l[e];
      }
      asm volatile("bar.sync 1, 256;\n" ::: "memory");
      for (int y = tid; y < rows * hc * (D / 4); y += 32 * DW) {
        const int d4 = y % (D / 4), rh = y / (D / 4), r = rh / hc, h = rh % hc;
        float mm = -INFINITY, ll = 0.f;
        for (int s = 0; s < slices; ++s) mm = fmaxf(mm, merge[((s * hc + h) * rows_max + r) * (D + 4) + D]);
        const float ref = mm == -INFINITY ? 0.f : mm;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int s = 0; s < slices; ++s) {
          const float* src = merge + ((s * hc + h) * rows_max + r) * (D + 4);
          const float wgt = ex2(src[D] - ref);
          const float4 v4 = *reinterpret_cast<const float4*>(src + d4 * 4);
          ll = fmaf(src[D + 1], wgt, ll);
          a.x = fmaf(v4.x, wgt, a.x), a.y = fmaf(v4.y, wgt, a.y);
          a.z = fmaf(v4.z, wgt, a.z), a.w = fmaf(v4.w, wgt, a.w);
        }
        if (!cut) {
          finish(w, rh, d4, mm, ll, a);
        } else {
          const long long at = (long long)slot * p.part_rows + r * hc + h;
          *reinterpret_cast<float4*>(p.part_o + at * D + d4 * 4) = a;
          if (d4 == 0) p.part_ml[at] = make_float2(mm, ll);
        }
      }
      if (!cut) asm volatile("bar.sync 1, 256;\n" ::: "memory");  // before the area is written again
    }
    if (w.first + w.tiles >= x1) break;
  }
}

// ---------------------------------------------------------------------------
// Many query rows: tcgen05.
//
// An item is one KV head and up to 2 x 128 query rows, row r of a tile being
// (token r / G, head r % G of the group): every query head of the group and
// every token share the K/V tiles. Units are 128 keys.
//   warps 0-7   softmax: two groups of four, one query row (TMEM lane) per thread
//   warp 8      producer: Q tiles per item, K and V tiles (one TMA box per
//               page touched) through one ring, in the order they are used
//   warp 9      TMEM owner and MMA issuer (whole warp, one elected lane)
//   warps 10-11 idle: they complete the third warpgroup, whose registers go to
//               the softmax (a row's 128 scores stay in registers)
// S = Q K^T (TMEM), P = 2^(scale S - M) rounded to the cache's 16-bit type in
// place of S, O += P V (TMEM); the sum of P is kept in FP32 before rounding.
// M moves only when a row's maximum has risen by more than 2^8, the row's O
// and sum then being rescaled.
// The scores rotate through NB TMEM buffers: three for 64-wide heads, so that a
// group's next scores are there before its softmax ends; two for 128-wide ones
// (the outputs take the rest of TMEM). Products of M = 128 with A in shared
// memory take about 70 cycles per K = 16 step for N = 64 and N = 128 alike, and
// 44 or 64 with A in TMEM, so whole 128-key tiles: halves of 64 keys, which
// would double-buffer within the same columns, measured 2076 tensor cycles per
// unit of two query tiles against 1244.
// What bounds it is the softmax's latency: two 2048-token chunks over 8192 keys
// (155 us, 777 TFLOP/s) keep the special-function unit 71 %, the issue slots 51 %
// and the tensor pipe 40 % of the cycles busy, with two softmax warps on a
// scheduler that each load scores, take the maximum, weigh and store in turn.
// Items of more than 128 rows give each group one of the two query tiles;
// smaller ones give both groups the same queries and alternate key tiles
// between them; the two accumulators are then joined in the epilogue. Either
// way an item is a sequence of jobs (scores, softmax, product with V), job j
// being group j & 1's: of a tile per job, or of a tile per pair of jobs.
// ---------------------------------------------------------------------------
constexpr int T_THREADS = 384;
// 384 threads x 168 registers at launch = 64512 >= 256 x 208 + 128 x 80 = 63488.
constexpr int SOFTMAX_REGS = 208, OTHER_REGS = 80;

template <int D>
struct TShape {
  static constexpr int DH = D / 64;
  static constexpr uint32_t SLOT = 16384u * DH;  // one K or V tile
  static constexpr int SLOTS = D == 64 ? 10 : 5;
  static constexpr uint32_t Q = 0, RING = 2 * SLOT, ML = RING + SLOTS * SLOT;  // ML: (max, sum) of group 1's rows
  static constexpr uint32_t BARS = ML + 1024;
  static constexpr int NB = D == 64 ? 3 : 2;       // score buffers of 128 TMEM columns
  static constexpr uint32_t O = NB * 128;          // first column of the outputs
  static constexpr int NBARS = 2 * SLOTS + 3 + 2 * NB + 2 + 2;
  static constexpr uint32_t TOTAL = 1024 + BARS + 8 * (NBARS + 1);
};

// Instruction descriptor of kind::f16 with FP32 accumulation; A and B bf16 or fp16.
__host__ __device__ constexpr uint32_t idesc16(bool bf, int N, int b_mn) {
  return (1u << 4) | ((bf ? 1u : 0u) << 7) | ((bf ? 1u : 0u) << 10) | ((uint32_t)b_mn << 16) |
         ((uint32_t)(N >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;\n" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// 2^x for two x < 128 on the FMA and integer pipes, for part of a tile: less for
// the special-function unit, the busiest pipe. x = n + f with n the
// nearest integer (read off the low bits of x + 1.5 * 2^23 + 127, so that the
// shifted bits are the FP32 exponent of 2^n) and |f| <= 1/2; 2^f by the degree-4
// polynomial of least relative error on that interval (Remez exchange on
// p(f) 2^-f - 1), off by at most 2.7e-6 in FP32. From -126.5 down the result is
// exactly 0, as it has to be for masked keys; NaN stays NaN.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;\n" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint64_t ex2_poly2(uint64_t x) {
  const float2 f = unpair(x);
  x = pair(max_nan(f.x, -127.f), max_nan(f.y, -127.f));
  const uint64_t t = add2(x, pair(12583039.f, 12583039.f));
  const uint64_t r = fma2(add2(t, pair(-12583039.f, -12583039.f)), pair(-1.f, -1.f), x);
  uint64_t q = fma2(pair(9.570101911150505e-3f, 9.570101911150505e-3f), r, pair(5.5917860319385004e-2f, 5.5917860319385004e-2f));
  q = fma2(q, r, pair(0.24024744827864145f, 0.24024744827864145f));
  q = fma2(q, r, pair(0.6931218147366899f, 0.6931218147366899f));
  q = fma2(q, r, pair(0.999999261445712f, 0.999999261445712f));
  const float2 n = unpair(t);
  return mul2(q, pair(__int_as_float(__float_as_int(n.x) << 23), __int_as_float(__float_as_int(n.y) << 23)));
}
// One pair of keys in POLY_OF goes through the polynomial. Measured on a
// 2 x 2048-token prefill over 8192 keys: none 168, 1/8 157, 1/4 157, 3/8 166,
// 1/2 185 us.
constexpr int POLY_OF = 8;

// Four K = 16 steps of one product, issued by one elected lane of a converged
// warp: A in shared memory (descriptor steps of 32 bytes) or in tensor memory
// (8 columns), B in shared memory (steps of 32 bytes K-major, 2048 MN-major).
// One election and no arithmetic between the instructions: the issuing warp is
// a serial stage of every tile.
__device__ __forceinline__ void mma4_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred e, p, t;\n elect.sync _|e, 0xffffffff;\n setp.ne.b32 p, %4, 0;\n setp.eq.b32 t, 0, 0;\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], %5, %8, %3, t;\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], %6, %9, %3, t;\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], %7, %10, %3, t;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "l"(a + 2), "l"(a + 4), "l"(a + 6), "l"(b + 2), "l"(b + 4), "l"(b + 6)
      : "memory");
}
__device__ __forceinline__ void mma4_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred e, p, t;\n elect.sync _|e, 0xffffffff;\n setp.ne.b32 p, %4, 0;\n setp.eq.b32 t, 0, 0;\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [%5], %8, %3, t;\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [%6], %9, %3, t;\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [%7], %10, %3, t;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(a + 8), "r"(a + 16), "r"(a + 24), "l"(b + 128), "l"(b + 256),
      "l"(b + 384)
      : "memory");
}

// A value every lane of the warp holds, in a form the compiler knows to be
// uniform: what is computed from it stays in the uniform datapath, where the
// tensor instructions take their operands from.
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }

// Whole-warp bounded wait that suspends in the barrier instead of polling: the
// producer and the issuer share their schedulers with two softmax warps each,
// and every issue slot they spin in is taken from those.
__device__ __forceinline__ bool wait_quiet(uint32_t bar, uint32_t parity, int* status, int code) {
  const long long t0 = clock64();
  for (;;) {
    uint32_t done;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 20000;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    if (__all_sync(0xffffffffu, done)) return true;
    if (__any_sync(0xffffffffu, clock64() - t0 > (1LL << 32))) {
      atomicCAS(status, 0, code);
      return false;
    }
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(T_THREADS, 1)
    chunk_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                 const __grid_constant__ CUtensorMap tv, Params p) {
  using S = TShape<D>;
  constexpr int DH = S::DH;
  constexpr bool BF = std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t sb = smem_u32(smem), bars = sb + S::BARS;
  auto full_bar = [&](int s) { return bars + 8u * s; };
  auto empty_bar = [&](int s) { return bars + 8u * (S::SLOTS + s); };
  const uint32_t q_full = bars + 8u * (2 * S::SLOTS), q_empty = q_full + 8, tail_bar = q_full + 16;
  auto s_full = [&](int b) { return q_full + 24 + 8u * b; };
  auto p_full = [&](int b) { return q_full + 24 + 8u * (S::NB + b); };
  auto pv_done = [&](int g) { return q_full + 24 + 8u * (2 * S::NB + g); };
  const uint32_t o_free = pv_done(2), done_bar = o_free + 8;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + S::BARS + 8 * S::NBARS);
  const int tid = threadIdx.x, warp = uniform(tid >> 5), lane = tid & 31;
  int* status = &g_status;

  if (tid == 0) {
    for (int s = 0; s < S::SLOTS; ++s) {
      tc::mbar_init(full_bar(s), 1);
      tc::mbar_init(empty_bar(s), 1);
    }
    tc::mbar_init(q_full, 1);
    tc::mbar_init(q_empty, 1);
    tc::mbar_init(tail_bar, 1);
    for (int i = 0; i < S::NB; ++i) {
      tc::mbar_init(s_full(i), 1);
      tc::mbar_init(p_full(i), 4);  // one arrival per warp
    }
    tc::mbar_init(pv_done(0), 1);
    tc::mbar_init(pv_done(1), 1);
    tc::mbar_init(o_free, 256);
    tc::mbar_init(done_bar, 1);
    tc::mbar_fence_init();
    tc::tma_prefetch_desc(&tq);
    tc::tma_prefetch_desc(&tk);
    tc::tma_prefetch_desc(&tv);
  }
  if (warp == 9) {
    tc::tmem_alloc(smem_u32(tmem_slot), 512);
    tc::tmem_relinquish();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = uniform(*tmem_slot);
  wait_prerequisites();
  allow_dependents();
  const Header head = *p.head;
  const Item start = p.starts[blockIdx.x];
  const int share = blockIdx.x;
  const bool idle = uniform(share >= head.shares || head.total == 0);
  const int x0 = idle ? 0 : share_begin(head, share), x1 = idle ? 0 : share_begin(head, share + 1);
  const int G = p.G, tpt = 128 / G;  // tokens per query tile
  const int page = 1 << p.page_shift, br = min(128, page), nb = 128 / br;

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(OTHER_REGS));
    if (!idle && warp == 8) {
      int slot = 0, slot_ph = 0, fills = 0, seg = 0, tails = 0;
      bool ok = true;
      for (Item w = start; ok;) {
        const int j0 = unit_at(w, x0), j1 = unit_at(w, x1), n = j1 - j0;
        if (n > 0) {
          const bool dual = w.ntok > tpt;
          if (!(ok = wait_quiet(q_empty, (seg & 1) ^ 1, status, 11))) break;
          ++seg;
          if (lane == 0) {
            const int tiles = dual ? 2 : 1;
            tc::mbar_expect_tx(q_full, (uint32_t)(tiles * DH * tpt * G * 128));
            for (int t = 0; t < tiles; ++t)
              for (int h = 0; h < DH; ++h)
                tc::tma_load_3d(sb + S::Q + t * S::SLOT + h * 16384u, &tq, h * 64, w.hg * G, w.tok0 + t * tpt, q_full);
          }
          __syncwarp();
          const int end = min(w.keys, j1 * 128);
          PageIds k_ids(p, w.b, br, nb, j0, end), v_ids = k_ids;
          int kj = j0, vj = j0;
          auto load = [&](const CUtensorMap* map, int j, PageIds& ids, bool is_v) {
            if (!(ok = wait_quiet(empty_bar(slot), slot_ph ^ 1, status, 12))) return;
            const int valid = min(128, w.keys - j * 128), live = cdiv(max(valid, 0), br);
            const bool tail = is_v && valid < 128;
            const uint32_t bar = tail ? tail_bar : full_bar(slot), dst = sb + S::RING + slot * S::SLOT;
            if (lane == 0) tc::mbar_expect_tx(bar, (uint32_t)(live * br * 128 * DH));
            __syncwarp();
            const int bx = lane % max(live, 1), half = lane / max(live, 1);
            const int pid = ids.get(p, j, bx);
            if (half < DH && lane < live * DH)
              tma_load_4d(dst + half * 16384u + bx * br * 128, map, half * 64, (j * 128 + bx * br) & (page - 1), w.hg,
                          pid, bar);
            if (tail) {
              // Rows past the sequence hold whatever the page (or the ring) held;
              // zeros in their place, since 0 x NaN would not vanish in P V.
              ok = wait_quiet(tail_bar, tails & 1, status, 13);
              ++tails;
              for (int i = max(valid, 0) * 8 + lane; i < 128 * 8; i += 32)
                for (int h = 0; h < DH; ++h)
                  *reinterpret_cast<uint4*>(smem + S::RING + slot * S::SLOT + h * 16384u + i * 16) = make_uint4(0, 0, 0, 0);
              tc::fence_proxy_async_smem();
              __syncwarp();
              if (lane == 0) tc::mbar_arrive(full_bar(slot));
            }
            ++fills;
            if (++slot == S::SLOTS) slot = 0, slot_ph ^= 1;
          };
          // Jobs' order of need: step s runs the product of job s - NB, then the
          // scores of job s.
          const int jobs = dual ? 2 * n : n;
          for (int st = 0; ok && st < jobs + S::NB; ++st) {
            const int pj = st - S::NB;
            if (pj >= 0 && (!dual || !(pj & 1))) {
              load(&tv, vj++, v_ids, true);
              if (!ok) break;
            }
            if (st < jobs && (!dual || !(st & 1))) {
              load(&tk, kj++, k_ids, false);
            }
          }
        }
        if (!advance(p, w, x1)) break;
      }
      if (!ok)  // a wait gave up: let the copies in flight land before the CTA ends
        for (int f = max(0, fills - S::SLOTS); f < fills; ++f)
          wait_quiet(full_bar(f % S::SLOTS), (f / S::SLOTS) & 1, status, 14);
    } else if (!idle && warp == 9) {
      const uint32_t idesc_s = idesc16(BF, 128, 0), idesc_o = idesc16(BF, D, 1);
      const uint64_t q_desc = tc::smem_desc_sw128(sb + S::Q, 16, 1024);
      const uint64_t k_desc = tc::smem_desc_sw128(sb + S::RING, 16, 1024);
      const uint64_t v_desc = tc::smem_desc_sw128(sb + S::RING, 16384, 1024);
      int slot = 0, slot_ph = 0, seg = 0;
      int sbuf = 0, pbuf = 0, pph = 0;  // buffer of the next scores, of the next product, and its phase
      bool ok = true;
      for (Item w = start; ok;) {
        const int n = uniform(unit_at(w, x1) - unit_at(w, x0));
        if (n > 0) {
          const bool dual = uniform(w.ntok) > tpt;
          const int jobs = dual ? 2 * n : n;
          int ks = 0, vs = 0;
          if (!(ok = wait_quiet(q_full, seg & 1, status, 21))) break;
          for (int st = 0; ok && st < jobs + S::NB; ++st) {
            const int pj = st - S::NB;
            if (pj >= 0) {
              if (!dual || !(pj & 1)) {
                vs = slot;
                if (!(ok = wait_quiet(full_bar(vs), slot_ph, status, 22))) break;
                if (++slot == S::SLOTS) slot = 0, slot_ph ^= 1;
              }
              // The output accumulators of the previous item are read out.
              if (pj == 0 && !(ok = wait_quiet(o_free, (seg & 1) ^ 1, status, 24))) break;
              if (!(ok = wait_quiet(p_full(pbuf), pph, status, 25))) break;
              tc::tc_fence_after();
              const uint32_t o_t = tmem + S::O + (pj & 1) * D, p_t = tmem + pbuf * 128;
              const uint64_t vd = v_desc + (uint64_t)(vs * (S::SLOT >> 4));
              mma4_ts(o_t, p_t, vd, idesc_o, pj > 1 ? 1u : 0u);
              mma4_ts(o_t, p_t + 32, vd + 512, idesc_o, 1u);
              tc::mma_commit_w(pv_done(pj & 1));
              if (!dual || (pj & 1)) tc::mma_commit_w(empty_bar(vs));
              if (++pbuf == S::NB) pbuf = 0, pph ^= 1;
            }
            if (st < jobs) {
              if (!dual || !(st & 1)) {
                ks = slot;
                if (!(ok = wait_quiet(full_bar(ks), slot_ph, status, 23))) break;
                if (++slot == S::SLOTS) slot = 0, slot_ph ^= 1;
              }
              tc::tc_fence_after();
              const uint32_t s_t = tmem + sbuf * 128;
              const uint64_t qd = q_desc + (uint64_t)(dual && (st & 1) ? S::SLOT >> 4 : 0);
              const uint64_t kd = k_desc + (uint64_t)(ks * (S::SLOT >> 4));
              mma4_ss(s_t, qd, kd, idesc_s, 0u);
              if (D == 128) mma4_ss(s_t, qd + 1024, kd + 1024, idesc_s, 1u);
              tc::mma_commit_w(s_full(sbuf));
              if (!dual || (st & 1)) tc::mma_commit_w(empty_bar(ks));
              if (st == jobs - 1) tc::mma_commit_w(q_empty);
              if (++sbuf == S::NB) sbuf = 0;
            }
          }
          ++seg;
        }
        if (!uniform(advance(p, w, x1))) break;
      }
      tc::mma_commit_w(done_bar);
      wait_quiet(done_bar, 0, status, 26);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(SOFTMAX_REGS));
    const int grp = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane;
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const uint32_t o_t = tmem + lane_off + S::O + grp * D;
    float2* ml_s = reinterpret_cast<float2*>(smem + S::ML);
    const float sl2 = p.scale_log2;
    int nj0 = 0, nj1 = 0;  // jobs each group has had
    int buf = 0, ph = 0;   // buffer and phase of the item's job 0
    bool ok = true;
    // The item's record is read again behind the jobs: its registers are needed there.
    for (int index = start.index; !idle; ++index) {
      int j0, n, limit;
      bool dual, live;
      const int row_tok = r / G;
      {
        const Item w = p.items[index];
        j0 = unit_at(w, x0);
        n = unit_at(w, x1) - j0;
        if (n <= 0) {
          if (w.first + (w.tiles << w.shift) >= x1) break;
          continue;
        }
        dual = w.ntok > tpt;
        const int t = (dual ? grp * tpt : 0) + row_tok;
        live = r < tpt * G && t < w.ntok;
        // Keys this row sees; rows that do not exist mask nothing and are never read.
        limit = live ? min(w.pos0 + t + 1, w.keys) : 0x7fffffff;
      }
      const bool warp_live = __any_sync(0xffffffffu, live);
      float M = -INFINITY;
      uint64_t l2 = pair(0.f, 0.f);
      const int jobs = dual ? 2 * n : n;
      int mine = grp ? nj1 : nj0;
      int bj = buf + grp, pj = ph;  // buffer and phase of this group's next job
      if (bj >= S::NB) bj -= S::NB, pj ^= 1;
      for (int j = grp; j < jobs; j += 2, ++mine) {
        if (ok) ok = tc::mbar_wait_w(s_full(bj), pj, status, 31);
        if (ok && warp_live) {
          const uint32_t s_t = tmem + lane_off + bj * 128;
          const int lim = limit - (j0 + (dual ? j >> 1 : j)) * 128;
          const bool masked = __any_sync(0xffffffffu, lim < 128);
          tc::tc_fence_after();
          uint32_t v[128];
#pragma unroll
          for (int c = 0; c < 4; ++c) tc::tmem_ld_32x32b_x32(s_t + c * 32, v + c * 32);
          tc::tmem_ld_wait();
          if (masked) {
#pragma unroll
            for (int i = 0; i < 128; ++i) v[i] = i < lim ? v[i] : 0xFF800000u;
          }
          float mx[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) mx[e] = fmaxf(__uint_as_float(v[e]), __uint_as_float(v[e + 4]));
#pragma unroll
          for (int i = 8; i < 128; i += 8)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              mx[e] = max3(mx[e], __uint_as_float(v[i + e]), __uint_as_float(v[i + e + 4]));
          const float top = max3(fmaxf(mx[0], mx[1]), mx[2], mx[3]) * sl2;
          const bool up = top > M + 8.f, move = up && M != -INFINITY;
          if (__any_sync(0xffffffffu, move)) {
            // This group's previous product may still be adding to O.
            ok = tc::mbar_wait_w(pv_done(grp), (mine - 1) & 1, status, 34);
            tc::tc_fence_after();
            const float a = move ? ex2(M - top) : 1.f;
            const float2 lv = unpair(l2);
            l2 = pair(lv.x * a, lv.y * a);
#pragma unroll
            for (int c = 0; c < D / 16; ++c) {
              uint32_t ov[16];
              tc::tmem_ld_32x32b_x16(o_t + c * 16, ov);
              tc::tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 16; ++e) ov[e] = __float_as_uint(__uint_as_float(ov[e]) * a);
              tc::tmem_st_32x32b_x16(o_t + c * 16, ov);
            }
          }
          if (up) M = top;
          const float neg = M == -INFINITY ? 0.f : -M;
          const uint64_t sl = pair(sl2, sl2), ng = pair(neg, neg);
          // P over the scores: 16-bit pairs in the first 64 columns. Blocks of
          // 32 keys, the sums and conversions of one behind the exponentials
          // of the next, so that the special-function unit is rarely waited for.
          uint64_t e[2][16], sum[4] = {l2, pair(0.f, 0.f), pair(0.f, 0.f), pair(0.f, 0.f)};
          auto weigh = [&](int c, uint64_t* out) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int k = c * 32 + 2 * i;
              const uint64_t x = fma2(pair(__uint_as_float(v[k]), __uint_as_float(v[k + 1])), sl, ng);
              if (i % POLY_OF == 0) {
                out[i] = ex2_poly2(x);
              } else {
                const float2 f = unpair(x);
                out[i] = pair(ex2(f.x), ex2(f.y));
              }
            }
          };
          auto store = [&](int c, const uint64_t* in) {
            uint32_t pk[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              sum[i & 3] = add2(sum[i & 3], in[i]);
              const float2 f = unpair(in[i]);
              pk[i] = Num16<T>::pack2(f.x, f.y);
            }
            tc::tmem_st_32x32b_x16(s_t + c * 16, pk);
          };
          weigh(0, e[0]);
#pragma unroll
          for (int c = 1; c < 4; ++c) {
            weigh(c, e[c & 1]);
            store(c - 1, e[(c - 1) & 1]);
          }
          store(3, e[1]);
          l2 = add2(add2(sum[0], sum[1]), add2(sum[2], sum[3]));
          tc::tmem_st_wait();
          tc::tc_fence_before();
        }
        // With three buffers a job's scores do not wait for the product of the
        // group's job before it, and the epilogue's wait tells this item's last
        // product only from the one before by the phase's parity: that one has
        // to be done before the last can start.
        if (S::NB > 2 && j + 2 >= jobs && mine > 0 && ok) ok = tc::mbar_wait_w(pv_done(grp), (mine - 1) & 1, status, 35);
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(p_full(bj));
        bj += 2;
        if (bj >= S::NB) bj -= S::NB, pj ^= 1;
      }
      // The next item's job 0: `jobs` buffers on.
      buf += jobs % S::NB;
      ph ^= (jobs / S::NB) & 1;
      if (buf >= S::NB) buf -= S::NB, ph ^= 1;
      const float2 lv = unpair(l2);
      float l = lv.x + lv.y;
      const Item w = p.items[index];
      const int t = (dual ? grp * tpt : 0) + row_tok;

      // Epilogue: this group's rows (dual), or both groups' accumulators of
      // the same rows joined by group 0.
      const bool has1 = dual || n > 1, cut = j0 > 0 || j0 + n < w.tiles;
      nj0 += (jobs + 1) / 2;
      nj1 += jobs / 2;
      float a0 = 1.f, a1 = 0.f;
      if (!dual) {
        if (grp == 1) ml_s[r] = make_float2(M, l);
        asm volatile("bar.sync 1, 256;\n" ::: "memory");
        const float2 o = ml_s[r];
        asm volatile("bar.sync 1, 256;\n" ::: "memory");  // before the next item's are written
        if (grp == 0 && has1) {
          const float top = fmaxf(M, o.x), ref = top == -INFINITY ? 0.f : top;
          a0 = ex2(M - ref);
          a1 = ex2(o.x - ref);
          l = l * a0 + o.y * a1;
          M = top;
        }
      }
      const bool store = live && (dual || grp == 0);
      if ((dual || grp == 0) && ok) {
        ok = tc::mbar_wait_w(pv_done(grp), ((grp ? nj1 : nj0) - 1) & 1, status, 32);
        if (ok && !dual && has1) ok = tc::mbar_wait_w(pv_done(1), (nj1 - 1) & 1, status, 33);
        if (ok && warp_live) {
          tc::tc_fence_after();
          const float inv = cut ? 1.f : (l > 0.f ? 1.f / l : 0.f);
          const float f0 = a0 * inv, f1 = a1 * inv;
          const long long at = (long long)(w.tok0 + t) * p.H + w.hg * G + r % G;
          const int slot = slot_of(head, w, share), pr = t * G + r % G;
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            uint32_t ov[32];
            tc::tmem_ld_32x32b_x32(o_t + c * 32, ov);
            tc::tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e) ov[e] = __float_as_uint(__uint_as_float(ov[e]) * f0);
            if (!dual && has1) {
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                uint32_t o1[16];
                tc::tmem_ld_32x32b_x16(o_t + D + c * 32 + h * 16, o1);
                tc::tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 16; ++e)
                  ov[h * 16 + e] = __float_as_uint(fmaf(__uint_as_float(o1[e]), f1, __uint_as_float(ov[h * 16 + e])));
              }
            }
            if (!store) continue;
            if (cut) {
              float4* dst = reinterpret_cast<float4*>(p.part_o);
#pragma unroll
              for (int e = 0; e < 8; ++e)
                dst[part_at<D, true>(p, slot, pr, c * 8 + e)] =
                    make_float4(__uint_as_float(ov[4 * e]), __uint_as_float(ov[4 * e + 1]),
                                __uint_as_float(ov[4 * e + 2]), __uint_as_float(ov[4 * e + 3]));
            } else {
              uint4* dst = reinterpret_cast<uint4*>(p.o + at * D + c * 32);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                float f[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(ov[8 * e + i]);
                dst[e] = pack16x8<T>(f);
              }
            }
          }
          if (store && cut) p.part_ml[(long long)slot * p.part_rows + pr] = make_float2(M, l);
          if (store && !cut && p.lse) p.lse[at] = lse_of(M, l);
          tc::tc_fence_before();
        }
      }
      tc::mbar_arrive(o_free);
      if (w.first + (w.tiles << w.shift) >= x1) break;
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, 512);
  }
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------
inline size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

constexpr size_t MAX_SMEM = 227 * 1024 - 256;  // dynamic part of a CTA's shared memory
// Query rows per KV head the warp-level kernel takes, of any sequence of the call.
// Rows beyond 8 fill its products' second half; against the tiles they took (16/8
// heads of 64, with tokens x group = 10 and 16): 16 x 5 tokens over 4096 keys 38.5
// and 45.3 us, 16 x 8 39.5 and 45.2, 64 x 8 over 256 to 4096 65.9 and 99.0, 8 over
// 30000 24.8 and 31.6.
constexpr int FEW_ROWS = 16;

struct Plan {
  bool few;
  int hc, unit, tok_item, grid_cap, part_rows, slots;
  long long max_items;  // listed items
  size_t bytes;
  // The items' total weight is counted in 32 bits: its bound for a table of `span` positions per sequence.
  double max_weight(int B, int Hk, long long span) const {
    const double units = (double)((span + unit - 1) / unit);
    return few ? (double)B * (Hk / hc) * units : 2.0 * max_items * units;
  }
};

Plan plan(int N, int B, int max_q, int H, int Hk, int D) {
  Plan pl{};
  const int G = H / Hk;
  pl.few = (long long)max_q * G <= FEW_ROWS;
  if (pl.few) {
    pl.hc = Hk % 8 == 0 ? 8 : Hk % 4 == 0 ? 4 : Hk % 2 == 0 ? 2 : 1;
    pl.unit = 128 / pl.hc;
    pl.tok_item = max_q;
    pl.grid_cap = 2 * MAX_SMS;
    pl.max_items = 0;  // not listed: every CTA finds its own
    pl.part_rows = max_q * G * pl.hc;
  } else {
    pl.hc = 1;
    pl.unit = 128;
    pl.tok_item = 2 * (128 / G);
    pl.grid_cap = MAX_SMS;
    pl.max_items = (long long)Hk * (N / pl.tok_item + B);
    pl.part_rows = 256;
  }
  pl.slots = 2 * pl.grid_cap;
  pl.bytes = 256 + align256(sizeof(Item) * (size_t)pl.max_items) + 2 * align256(sizeof(Item) * (size_t)pl.grid_cap) +
             align256(sizeof(float) * (size_t)pl.slots * pl.part_rows * D) +
             align256(sizeof(float2) * (size_t)pl.slots * pl.part_rows);
  return pl;
}

void carve(Params& p, const Plan& pl, void* base, int D) {
  char* c = static_cast<char*>(base);
  auto take = [&](size_t n) {
    char* r = c;
    c += align256(n);
    return r;
  };
  p.head = reinterpret_cast<Header*>(take(sizeof(Header)));
  p.items = reinterpret_cast<Item*>(take(sizeof(Item) * (size_t)pl.max_items));
  p.starts = reinterpret_cast<Item*>(take(sizeof(Item) * (size_t)pl.grid_cap));
  p.cuts = reinterpret_cast<Item*>(take(sizeof(Item) * (size_t)pl.grid_cap));
  p.part_o = reinterpret_cast<float*>(take(sizeof(float) * (size_t)pl.slots * pl.part_rows * D));
  p.part_ml = reinterpret_cast<float2*>(take(sizeof(float2) * (size_t)pl.slots * pl.part_rows));
}

// {dim, row of the page, KV head, page}; box {64, rows, heads, 1}.
int make_tmap_pages(CUtensorMap* map, const void* base, bool bf, int D, int page_size, int Hk, int num_pages,
                    bool head_major, int box_rows, int box_heads) {
  const uint64_t token = (uint64_t)(head_major ? D : Hk * D) * 2, head = (uint64_t)(head_major ? page_size * D : D) * 2;
  const uint64_t dims[4] = {(uint64_t)D, (uint64_t)page_size, (uint64_t)Hk, (uint64_t)num_pages};
  const uint64_t strides[3] = {token, head, (uint64_t)page_size * Hk * D * 2};
  const uint32_t box[4] = {64, (uint32_t)box_rows, (uint32_t)box_heads, 1};
  return tc::make_tmap_16(map, base, bf, 4, dims, strides, box);
}

// Launches a kernel whose prologue may overlap the kernel before it.
template <typename... Formal, typename... Actual>
int launch_dependent(void (*kernel)(Formal...), int grid, int threads, size_t smem, cudaStream_t s, Actual&&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  MFB_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, args...));
  return MFB_OK;
}

template <typename T, int D, bool ROWS32>
int run_join(const Params& p, int sms, cudaStream_t s) {
  return launch_dependent(join_kernel<T, D, ROWS32>, 4 * sms, JOIN_THREADS, 0, s, p);
}

template <typename T, int D, bool R16>
int run_few(Params& p, const Plan& pl, const CUtensorMap& tk, const CUtensorMap& tv, int sms, cudaStream_t s) {
  const int rows = p.max_q * p.G;
  // Two or three units in the ring: 64 single tokens over up to 4096 keys 56.0 and
  // 58.6 us, 64 x 8 63.3 and 65.9, 16 x 8 over 4096 39.1 and 39.5, but 8 tokens over
  // 30000 keys 27.1 and 24.8.
  int stages = 3;
  while (stages > 2 && dlayout(D, stages, rows, pl.hc).total > MAX_SMEM) --stages;
  const size_t smem = dlayout(D, stages, rows, pl.hc).total;
  MFB_CUDA_TRY(cudaFuncSetAttribute(few_rows_kernel<T, D, R16>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)MAX_SMEM));
  const int per_sm = 2 * smem + 4096 <= 228 * 1024 ? 2 : 1;
  p.grid = std::min(per_sm * sms, pl.grid_cap);
  few_rows_kernel<T, D, R16><<<p.grid, D_THREADS, smem, s>>>(tk, tv, p, stages, rows);
  MFB_LAUNCH_CHECK("paged attention (few rows)");
  return run_join<T, D, false>(p, sms, s);
}

template <typename T, int D>
int run(Params& p, const Plan& pl, const void* q, const void* kp, const void* vp, int page_size, bool head_major,
        cudaStream_t s) {
  constexpr bool bf = std::is_same<T, __nv_bfloat16>::value;
  int dev = 0, sms = 148, st;
  MFB_CUDA_TRY(cudaGetDevice(&dev));
  MFB_CUDA_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
  sms = std::min(sms, MAX_SMS);
  CUtensorMap tk, tv, tq;
  const int br = std::min(pl.unit, page_size);
  if ((st = make_tmap_pages(&tk, kp, bf, D, page_size, p.Hk, p.num_pages, head_major, br, pl.hc))) return st;
  if ((st = make_tmap_pages(&tv, vp, bf, D, page_size, p.Hk, p.num_pages, head_major, br, pl.hc))) return st;
  if (pl.few) {
    return p.max_q * p.G <= 8 ? run_few<T, D, false>(p, pl, tk, tv, sms, s) : run_few<T, D, true>(p, pl, tk, tv, sms, s);
  }
  const uint64_t dims[3] = {(uint64_t)D, (uint64_t)p.H, (uint64_t)p.N};
  const uint64_t strides[2] = {(uint64_t)D * 2, (uint64_t)p.H * D * 2};
  const uint32_t box[3] = {64, (uint32_t)p.G, (uint32_t)(128 / p.G)};
  if ((st = tc::make_tmap_16(&tq, q, bf, 3, dims, strides, box))) return st;
  constexpr size_t smem = TShape<D>::TOTAL;
  static_assert(smem <= MAX_SMEM, "chunk kernel shared memory");
  MFB_CUDA_TRY(cudaFuncSetAttribute(chunk_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  p.grid = sms;
  schedule_kernel<<<1, SCHED_THREADS, sizeof(int) * (size_t)(p.B + 1), s>>>(p);
  MFB_LAUNCH_CHECK("paged attention schedule");
  if ((st = launch_dependent(chunk_kernel<T, D>, p.grid, T_THREADS, smem, s, tq, tk, tv, p))) return st;
  return run_join<T, D, true>(p, sms, s);
}

}  // namespace paged
}  // namespace mfb

using namespace mfb;

extern "C" size_t mfb_paged_attn_workspace_size(int N, int B, int max_q, int H, int Hk, int D) {
  if (N <= 0 || B <= 0 || B > paged::MAX_B || max_q <= 0 || H <= 0 || Hk <= 0 || H % Hk || H / Hk > 128 || D <= 0)
    return 0;
  return paged::plan(N, B, max_q, H, Hk, D).bytes;
}

extern "C" int mfb_paged_attn_check(int N, int B, int max_q, int max_pages, int num_pages, int page_size, int H, int Hk,
                                    int D) {
  MFB_CHECK_ARG(N > 0 && B > 0 && max_q > 0 && max_pages > 0 && num_pages > 0,
                "paged attention needs tokens, sequences and pages (N=%d B=%d max_q=%d)", N, B, max_q);
  MFB_CHECK_ARG(B <= paged::MAX_B, "paged attention batch %d above the supported %d sequences", B, paged::MAX_B);
  MFB_CHECK_ARG(H > 0 && Hk > 0 && H % Hk == 0, "Query heads must be divisible by KV heads (H=%d Hk=%d)", H, Hk);
  MFB_CHECK_ARG(H / Hk <= 128 && Hk <= 1024, "paged attention supports up to 1024 KV heads of 128 query heads (H=%d Hk=%d)",
                H, Hk);
  MFB_CHECK_ARG(D == 64 || D == 128, "paged attention head_dim %d unsupported (64 or 128)", D);
  MFB_CHECK_ARG(page_size >= 8 && (page_size & (page_size - 1)) == 0,
                "page_size %d must be a power of two of at least 8", page_size);
  MFB_CHECK_ARG((long long)page_size * Hk * D <= 1 << 30, "page of %d tokens too large", page_size);
  const long long span = (long long)max_pages * page_size;
  MFB_CHECK_ARG(span < (1LL << 31) - 128, "page table spans %lld positions (below 2^31 supported)", span);
  MFB_CHECK_ARG(paged::plan(N, B, max_q, H, Hk, D).max_weight(B, Hk, span) < 2147483647.0,
                "paged attention of %d tokens over tables of %lld positions exceeds 2^31 key tiles", N, span);
  return MFB_OK;
}

extern "C" int mfb_paged_attn(const void* q, const void* k_pages, const void* v_pages, const int32_t* cu_q,
                              const int32_t* seq_lens, const int32_t* page_table, void* o, float* lse, int N, int B,
                              int max_q, int max_pages, int num_pages, int page_size, int H, int Hk, int D,
                              int head_major, int dtype, float scale, void* workspace, size_t workspace_bytes,
                              void* stream) {
  int st = mfb_paged_attn_check(N, B, max_q, max_pages, num_pages, page_size, H, Hk, D);
  if (st) return st;
  MFB_CHECK_ARG(dtype == MFB_DTYPE_BF16 || dtype == MFB_DTYPE_F16, "paged attention dtype must be bf16 or fp16");
  MFB_CHECK_ARG(q && k_pages && v_pages && cu_q && seq_lens && page_table && o, "NULL paged attention argument");
  MFB_CHECK_ARG((((uintptr_t)q | (uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)o) & 15) == 0,
                "q, the pages and o must be 16-byte aligned");
  MFB_CHECK_ARG(isfinite(scale) && scale > 0.f, "paged attention scale must be positive and finite");
  const paged::Plan pl = paged::plan(N, B, max_q, H, Hk, D);
  if (!workspace || workspace_bytes < pl.bytes)
    return set_error(MFB_ERR_WORKSPACE, "paged attention workspace needs %zu bytes", pl.bytes);
  MFB_CHECK_ARG(((uintptr_t)workspace & 15) == 0, "workspace must be 16-byte aligned");
  paged::Params p{};
  p.q = (const uint16_t*)q;
  p.o = (uint16_t*)o;
  p.lse = lse;
  p.cu_q = cu_q;
  p.seq_lens = seq_lens;
  p.page_table = page_table;
  p.N = N;
  p.B = B;
  p.H = H;
  p.Hk = Hk;
  p.G = H / Hk;
  p.max_q = max_q;
  p.max_pages = max_pages;
  p.num_pages = num_pages;
  while ((1 << p.page_shift) < page_size) ++p.page_shift;
  p.tok_item = pl.tok_item;
  p.hc = pl.hc;
  p.unit = pl.unit;
  p.max_items = (int)pl.max_items;
  p.part_rows = pl.part_rows;
  p.scale_log2 = scale * kLog2e;
  paged::carve(p, pl, workspace, D);
  cudaStream_t s = (cudaStream_t)stream;
  const bool hm = head_major != 0;
  if (dtype == MFB_DTYPE_BF16)
    return D == 64 ? paged::run<__nv_bfloat16, 64>(p, pl, q, k_pages, v_pages, page_size, hm, s)
                   : paged::run<__nv_bfloat16, 128>(p, pl, q, k_pages, v_pages, page_size, hm, s);
  return D == 64 ? paged::run<__half, 64>(p, pl, q, k_pages, v_pages, page_size, hm, s)
                 : paged::run<__half, 128>(p, pl, q, k_pages, v_pages, page_size, hm, s);
}

extern "C" int mfb_paged_attn_status(int* code) {
  MFB_CHECK_ARG(code != nullptr, "code is NULL");
  int zero = 0;
  MFB_CUDA_TRY(cudaMemcpyFromSymbol(code, paged::g_status, sizeof(int)));
  if (*code) MFB_CUDA_TRY(cudaMemcpyToSymbol(paged::g_status, &zero, sizeof(int)));
  return MFB_OK;
}
