// Shared by the attention kernels over the paged cache (16-bit and 4-bit rows).
#pragma once
#include "paged.cuh"
#include "tensor_map.cuh"

namespace ha {

constexpr int attn4_tile(int d) { return d == 128 ? 128 : 256; }      // keys of a tile of 4-bit rows
constexpr int ITEM_ROWS = 16;         // query rows of an item, at most
constexpr int MAX_LINES = 256;        // lines (packs of a sequence's tokens) of one launch: their tiles are summed up in shared memory
// A weight's reference follows the running maximum only when that is 2^SLACK above it: with 16 rows a warp, some row's maximum grows at most of the first
// dozens of tiles, and each time all the sums are scaled.  Weights, held in 16 bits for the products, have that much room above.
constexpr float SLACK = 6.f;
constexpr float LN2 = 0.693147180559945309f, LOG2E = 1.44269504088896341f;

struct AttnArgs {
  PagedView c;
  const uint8_t* q;
  int64_t q_sb, q_sn, q_sh;           // bytes
  void* o;
  float* lse;
  int32_t n, H, Hk, group, blocks;    // blocks: items of a (token, K/V head): group / 16, rounded up
  int32_t pack, packs;                // neighbouring tokens of a sequence that share an item (pack * group <= 16, or one), and how many packs a sequence has
  int32_t line0, lines;               // (sequence, pack) pairs of this launch
  int32_t cluster;                    // CTAs that share an item, a cluster of them; 0: the list of tiles
  int32_t run_log2;                   // rows that are fetched together: 2^run_log2, the largest power of two that pages and tiles are made of
  int32_t runs;                       // 4 bits, rows of a page and their scales one behind the other, on 16-byte boundaries: 2 where a page holds a warp's keys of a tile, 1: a copy's
  FastDiv by_packs, by_blocks, by_group;
  float scale_log2;                   // magnitude of the softmax scale, times log2 e
  uint32_t flip;                      // sign bits of a pair of queries, where the scale is negative
  float* part;                        // [CTAs][2][ITEM_ROWS][D], then ...
  float2* part_stat;                  // [CTAs][2][ITEM_ROWS]: reference (log2), denominator
  int4* head;                         // [CTAs]: last item's first and end tile, its line, its number
  int32_t* meta;                      // all tiles, tiles of a CTA
};

template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldmatrix4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
template <int N>
__device__ __forceinline__ void cp_async_small(uint32_t dst, const void* src, uint32_t src_bytes) {      // 4 or 8 bytes
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(N), "r"(src_bytes) : "memory");
}
__device__ __forceinline__ uint4 lds128(const uint8_t* p) { return *reinterpret_cast<const uint4*>(p); }
__device__ __forceinline__ uint2 lds64(const uint8_t* p) { return *reinterpret_cast<const uint2*>(p); }
__device__ __forceinline__ uint32_t lds32(const uint8_t* p) { return *reinterpret_cast<const uint32_t*>(p); }
// an arrival on `bar` once this thread's cp.async so far are done
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) { asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory"); }
// (a & mask) ^ flip in one instruction (of two constants the compiler would make two)
__device__ __forceinline__ uint32_t and_xor(uint32_t a, uint32_t mask, uint32_t flip) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(r) : "r"(a), "r"(mask), "r"(flip));
  return r;
}
__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}
// A place in the list of tiles.
struct Walk {
  int line, item, tile, tiles;
  __device__ __forceinline__ void settle(const int* first, int lines) {         // skips lines without keys
    while (line < lines && (tiles = first[line + 1] - first[line]) == 0) ++line;
  }
  __device__ __forceinline__ void step(const int* first, int lines, int items) {
    if (++tile < tiles) return;
    tile = 0;
    if (++item < items) return;
    item = 0;
    ++line;
    settle(first, lines);
  }
};

__device__ __forceinline__ int chunk_at(int row, int chunk) { return chunk ^ (row & 7); }      // 16-byte chunk of a query row in shared memory

// Keys that a line sees, those of its last token that is one of the sequence; `last`: that token's place in the pack.
__device__ __forceinline__ int keys_of(const AttnArgs& a, int line, int& last) {
  const int b = a.by_packs(line), i0 = (line - b * a.packs) * a.pack;
  const int count = a.c.counts ? min(a.c.counts[b], a.n) : a.n;
  int len = a.c.lengths[b];
  if (len > a.c.capacity) {
    report_status(a.c.status, a.c.status_host, HA_DEV_BAD_INDEX);
    len = a.c.capacity;
  }
  last = max(min(a.pack, count - i0) - 1, 0);
  return i0 < count ? max(max(len, 0) - (count - 1 - i0 - last), 0) : 0;
}
// Keys that row `row` of an item does not see of those that the line's last token does: one for each token between (rows of padding like the last).
template <bool PACKED>
__device__ __forceinline__ int keys_short(const AttnArgs& a, int row, int last) { return PACKED ? max(last - a.by_group(row), 0) : 0; }

// What row `row` of an item is.
struct RowAt {
  int64_t o, lse;                     // its outputs: a row of o, an element of lse
  bool there, empty;                  // one of the call's rows; one of padding, or without keys
};
// (keys, last: what keys_of says of the line; PACKED: items of several tokens)
template <bool PACKED>
__device__ __forceinline__ RowAt row_at(const AttnArgs& a, int line, int item, int row, int keys = 1, int last = 0) {
  const int b = a.by_packs(line), i0 = (line - b * a.packs) * a.pack, h = a.by_blocks(item), block = item - h * a.blocks;
  const int t = PACKED ? a.by_group(row) : 0, of_group = block * ITEM_ROWS + row - t * a.group, i = i0 + t, head = h * a.group + of_group;
  RowAt r;
  r.there = t < a.pack && i < a.n && of_group < a.group;
  r.empty = t > last || keys <= last - t;
  r.o = ((int64_t)b * a.n + i) * a.H + head;
  r.lse = ((int64_t)b * a.H + head) * a.n + i;
  return r;
}
// ... and its query, from the first row's on.
__device__ __forceinline__ const uint8_t* query_of(const AttnArgs& a, int line, int item) {
  const int b = a.by_packs(line), i0 = (line - b * a.packs) * a.pack, h = a.by_blocks(item), block = item - h * a.blocks;
  return a.q + b * a.q_sb + i0 * a.q_sn + (int64_t)(h * a.group + block * ITEM_ROWS) * a.q_sh;
}
template <bool PACKED>
__device__ __forceinline__ int64_t query_row(const AttnArgs& a, int row) {
  const int t = PACKED ? a.by_group(row) : 0;
  return t * a.q_sn + (int64_t)(row - t * a.group) * a.q_sh;
}

// Tiles before each line (of one item; first[lines]: all) and keys of each line, by the CTA's first 128 threads; every thread calls it.
__device__ __forceinline__ void scan_lines(const AttnArgs& a, int tile_keys, int* first, int* keys, uint8_t* lasts, int* warp_sum) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int PER = (MAX_LINES + 1 + 127) / 128;
  int before = 0, mine[PER];
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const int line = tid * PER + u;
    int m = 0;
    if (line < a.lines) {
      int last;
      keys[line] = m = keys_of(a, a.line0 + line, last);
      lasts[line] = (uint8_t)last;
    }
    mine[u] = before;
    before += (m + tile_keys - 1) / tile_keys;
  }
  int incl = before;
#pragma unroll
  for (int y = 1; y < 32; y *= 2) {
    const int v = __shfl_up_sync(0xffffffffu, incl, y);
    if (lane >= y) incl += v;
  }
  if (lane == 31 && warp < 4) warp_sum[warp] = incl;
  __syncthreads();
  int ahead = incl - before;
  for (int w = 0; w < min(warp, 4); ++w) ahead += warp_sum[w];
#pragma unroll
  for (int u = 0; u < PER; ++u)
    if (tid * PER + u <= a.lines) first[tid * PER + u] = ahead + mine[u];
  __syncthreads();
}

template <typename T, int D>
__device__ __forceinline__ void empty_line(const AttnArgs& a, int line) {
  const int b = a.by_packs(line), i0 = (line - b * a.packs) * a.pack, tokens = min(a.pack, a.n - i0);
  uint4* o = reinterpret_cast<uint4*>((T*)a.o + ((int64_t)b * a.n + i0) * a.H * D);
  for (int e = threadIdx.x; e < tokens * a.H * D / 8; e += blockDim.x) o[e] = make_uint4(0, 0, 0, 0);
  for (int e = threadIdx.x; e < tokens * a.H; e += blockDim.x) a.lse[((int64_t)b * a.H + e / tokens) * a.n + i0 + e % tokens] = -INFINITY;
}

// This CTA's part [begin, end) of the list of tiles, and the place of its first; lines without keys get their outputs here.  With clusters, its part of
// one item's tiles: line 0 of what it sees, which is line `line0` of the call.  `least`: tiles of a part, at least.  Every thread calls it.
template <typename T, int D, bool CLUSTER>
__device__ __forceinline__ Walk take_part(const AttnArgs& a, int tile_keys, int least, int* first, int* keys, uint8_t* lasts, int* warp_sum, int items, int& begin, int& end, int& line0) {
  const int tid = threadIdx.x;
  if constexpr (CLUSTER) {
    const int unit = blockIdx.x / a.cluster, rank = blockIdx.x % a.cluster, line = unit / items;
    line0 = line;
    int last;
    const int m = keys_of(a, line, last), tiles = (m + tile_keys - 1) / tile_keys, share = (tiles + a.cluster - 1) / a.cluster;
    if (tid == 0) {
      first[0] = 0;
      first[1] = tiles;
      keys[0] = m;
      lasts[0] = (uint8_t)last;
    }
    __syncthreads();
    begin = min(rank * share, tiles);
    end = min(begin + share, tiles);
    if (m == 0 && rank == 0 && unit % items == 0) empty_line<T, D>(a, line);
    return Walk{0, unit % items, begin, tiles};
  } else {
    line0 = a.line0;
    scan_lines(a, tile_keys, first, keys, lasts, warp_sum);
    const int total = first[a.lines] * items;
    const int per = max((total + (int)gridDim.x - 1) / (int)gridDim.x, least);
    begin = min((int)blockIdx.x * per, total);
    end = min(begin + per, total);
    if (blockIdx.x == 0 && tid == 0) {
      a.meta[0] = total;
      a.meta[1] = per;
    }
    for (int line = blockIdx.x; line < a.lines; line += gridDim.x) {
      if (keys[line] == 0) empty_line<T, D>(a, a.line0 + line);
    }
    Walk at = {a.lines, 0, 0, 1};
    if (begin >= end) return at;
    int lo = 0, hi = a.lines;                  // the last line whose tiles begin at or before `begin`
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (first[mid] * items <= begin) lo = mid;
      else hi = mid;
    }
    at.line = lo;
    at.settle(first, a.lines);
    const int off = begin - first[at.line] * items;
    at.item = off / at.tiles;
    at.tile = off - at.item * at.tiles;
    return at;
  }
}

// End of an item, or of this CTA's part of it: the sums of the four warps that compute are joined through `sums` (a stage that has been read), and go out as
// the result or as a part.  `join`: all four warps are here and see what each wrote to shared memory; false: one gave up.
template <typename T, int D, int APART, bool CLUSTER, bool PACKED, typename W, typename J>
__device__ __forceinline__ bool finish_item(const AttnArgs& a, W& w, float2* stat, float* sums, const Walk& at, const int* first, int items, int begin, int end,
                                            bool last, int line0, int keys, int last_token, float* cluster_sums, float2* cluster_stat, J join) {
  constexpr int ROWS = W::ROWS, ROUNDS = W::ROUNDS, WIDTH = D / ROUNDS, LANES = 128 / ROWS;     // threads of a row
  static_assert(APART >= ROWS * WIDTH, "floats from one warp's sums to the next's");
  static_assert(WIDTH % (4 * LANES) == 0, "whole columns");
  const int tid = threadIdx.x, warp = tid >> 5;
  w.statistics(stat + warp * ITEM_ROWS);
  const int item_begin = first[at.line] * items + at.item * at.tiles, item_end = item_begin + at.tiles;
  const bool whole = !CLUSTER && item_begin >= begin && item_end <= end;
  const int row = tid / LANES;
  const RowAt ra = row_at<PACKED>(a, line0 + at.line, at.item, row, keys, last_token);
  const int slot = 2 * blockIdx.x + (item_begin <= begin ? 0 : 1);
  float part[4], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int y = 0; y < ROUNDS; ++y) {
    if (!join()) return false;               // the stage has been read (the round before, too); the statistics are there
    w.put(sums + warp * APART, y);
    if (y == 0) {
#pragma unroll
      for (int x = 0; x < 4; ++x) m = fmaxf(m, stat[x * ITEM_ROWS + row].x);
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float2 st = stat[x * ITEM_ROWS + row];
        part[x] = st.x == -INFINITY ? 0.f : fast_exp2(st.x - m);       // (its sums are zeros, or NaN)
        l = fmaf(part[x], st.y, l);
      }
    }
    if (!join()) return false;
    const float inv = whole ? 1.f / l : 1.f;
    float4 vs[WIDTH / (4 * LANES)];
#pragma unroll
    for (int j = 0; j < WIDTH / (4 * LANES); ++j) {
      const int col = (tid % LANES) * 4 + 4 * LANES * j;
      float4& v = vs[j];
      v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float4 f = *reinterpret_cast<const float4*>(sums + x * APART + row * WIDTH + (col ^ W::turn(row)));
        v.x = fmaf(part[x], f.x, v.x);
        v.y = fmaf(part[x], f.y, v.y);
        v.z = fmaf(part[x], f.z, v.z);
        v.w = fmaf(part[x], f.w, v.w);
      }
    }
    // (a cluster's part may lie where the sums did)
    if (CLUSTER && !join()) return false;
    if (ra.there) {
#pragma unroll
      for (int j = 0; j < WIDTH / (4 * LANES); ++j) {
        const int col = (tid % LANES) * 4 + 4 * LANES * j;
        const float4 v = vs[j];
        if (whole)
          *reinterpret_cast<uint2*>((T*)a.o + ra.o * D + y * WIDTH + col) =
              ra.empty ? make_uint2(0, 0) : make_uint2(pack2<T>(v.x * inv, v.y * inv), pack2<T>(v.z * inv, v.w * inv));
        else if (CLUSTER)
          *reinterpret_cast<float4*>(cluster_sums + row * D + y * WIDTH + col) = v;
        else
          *reinterpret_cast<float4*>(a.part + ((int64_t)slot * ITEM_ROWS + row) * D + y * WIDTH + col) = v;
      }
    }
    if (y == 0 && ra.there && tid % LANES == 0) {
      if (whole) a.lse[ra.lse] = ra.empty ? -INFINITY : (m + log2f(l)) * LN2;
      else if (CLUSTER) cluster_stat[row] = make_float2(m, l);
      else a.part_stat[slot * ITEM_ROWS + row] = make_float2(m, l);
    }
  }
  if (last && !CLUSTER && tid == 0) a.head[blockIdx.x] = make_int4(item_begin, item_end, a.line0 + at.line, at.item);
  return true;
}

__device__ __forceinline__ void cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_at(const void* p, int rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}

// End of an item that a cluster shares: each CTA joins its share of the rows from all CTAs' parts, read over distributed shared memory.  The first four warps of every
// CTA call it, those of a CTA without keys, too (a negative denominator); no CTA leaves before the others have read its part.
template <typename T, int D, bool PACKED, int MOST>
__device__ __forceinline__ void cluster_join(const AttnArgs& a, const float* sums, const float2* stat, int line, int item, int keys, int last) {
  const int tid = threadIdx.x, rank = blockIdx.x % a.cluster;
  constexpr int LANES = D / 4;                 // threads of a row, four columns each
  for (int row = rank + a.cluster * (tid / LANES); row < min(a.pack * a.group, ITEM_ROWS); row += a.cluster * (128 / LANES)) {
    const RowAt ra = row_at<PACKED>(a, line, item, row, keys, last);
    if (!ra.there) continue;
    const int col = tid % LANES * 4;
    float m = -INFINITY, l = 0.f;
    float2 st[MOST];
    float4 f[MOST];
#pragma unroll
    for (int x = 0; x < MOST; ++x) {
      st[x] = make_float2(-INFINITY, -1.f);
      if (x >= a.cluster) continue;
      asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(st[x].x), "=f"(st[x].y) : "r"(cluster_at(stat + row, x)));
      asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(f[x].x), "=f"(f[x].y), "=f"(f[x].z), "=f"(f[x].w) : "r"(cluster_at(sums + row * D + col, x)));
    }
#pragma unroll
    for (int x = 0; x < MOST; ++x) m = fmaxf(m, st[x].x);
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int x = 0; x < MOST; ++x) {
      if (st[x].y < 0.f) continue;
      const float w = st[x].x == -INFINITY ? 0.f : fast_exp2(st[x].x - m);
      l = fmaf(w, st[x].y, l);
      v.x = fmaf(w, f[x].x, v.x);
      v.y = fmaf(w, f[x].y, v.y);
      v.z = fmaf(w, f[x].z, v.z);
      v.w = fmaf(w, f[x].w, v.w);
    }
    const float inv = 1.f / l;
    *reinterpret_cast<uint2*>((T*)a.o + ra.o * D + col) = ra.empty ? make_uint2(0, 0) : make_uint2(pack2<T>(v.x * inv, v.y * inv), pack2<T>(v.z * inv, v.w * inv));
    if (col == 0) a.lse[ra.lse] = ra.empty ? -INFINITY : (m + log2f(l)) * LN2;
  }
}
template <typename T, int D, bool PACKED>
__device__ __forceinline__ void cluster_finish(const AttnArgs& a, const float* sums, const float2* stat, int line, int item, int keys, int last) {
  cluster_sync();
  if (a.cluster > 8) cluster_join<T, D, PACKED, 16>(a, sums, stat, line, item, keys, last);
  else cluster_join<T, D, PACKED, 8>(a, sums, stat, line, item, keys, last);
  cluster_sync();
}

// Kernels of 4-bit rows: CTAs of an SM, keys of a tile, and the launch of one kernel.
int attn4_resident(int d, int rows);
int attn4_launch(AttnArgs a, int dtype, int d, int ctas, cudaStream_t st);

}  // namespace ha
