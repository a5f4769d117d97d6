// Attention of a sequence's last tokens over its pages: one pass over K and V, split over the whole GPU.
//
//   s_j = scale q . k_j,  o = sum_j exp(s_j) v_j / sum_j exp(s_j),  lse = log sum_j exp(s_j),  j < keys of the row
//
// An item is the query rows that share a K/V head, up to 16, the rows of mma.sync.m16n8k16: the heads of one token, or of a few neighbouring tokens
// where they are less than that.  The products are thin (16 query rows against all keys), and K and V are read once: bytes bound the kernel.
// Tokens of an item see the same keys but for the last few; a value there that is no number is kept from the rows that do not see it.
//
// All items' keys, in tiles of TK, form one list; CTA c takes the c-th equal part of it, whatever the lengths are.  An item that lies within one CTA is
// finished there; of one that crosses to the next, each CTA writes its part (unnormalised sums, reference, denominator) to the workspace,
// and paged_combine_kernel adds them up in the order of the keys.  A CTA's own parts of an item: at most the first and the last of its list.
//
// Here: 16-bit rows, the joining of parts, the entry points.  (4-bit rows: paged_attn4.cu.)  A CTA: four warps that compute, each a quarter of a tile's
// keys with its own running maximum and sums, which are joined at the item's end; and one that fetches tiles into a ring of NS stages, across
// items, by tensor copies (128-byte swizzle; boxes of as many rows as both a page and a tile are made of, so that any page size will do).
// 1 x 131072 tokens, 32 heads x 64: 166 to 172 us from machine to machine, 6.2 to 6.5 TB/s (95 to 99 % of a copy's rate).  Batch of 32 x up to 8192, two
// K/V heads x 128: 27.2 us, 3.5 TB/s: what remains is the latency of a kernel's start, of a part's end and of the joining.
#include <string.h>

#include <algorithm>
#include <atomic>
#include <numeric>
#include <type_traits>

#include "paged_attn.cuh"

namespace ha {

namespace {

constexpr int THREADS = 160;
constexpr int BOX_ROWS = 32;          // rows of a tensor copy, at most: what is fetched behind the last key is less than that (49 x up to 7 tokens, 64 heads, pages of 256: 22.2 us by 64, 20.6 by 32;
                                      // long rows alike; by 16, 1 x 131072 with 32 heads x 64 gains 2 %, 16 x 4096 by clusters loses 10 %)
constexpr int CLUSTER_TILES = 10;     // tiles of a CTA, at most, where clusters share items
constexpr int CLUSTER_TILES_16 = 6;   // ... in clusters of 16

template <int D>
struct Stage {
  static constexpr int KW = 16;                              // keys of a warp
  static constexpr int TK = 4 * KW;
  static constexpr int ROW = 2 * D;                          // bytes of a row
  static constexpr int V = TK * ROW, Q = 2 * TK * ROW, BYTES = Q + ITEM_ROWS * ROW;
  static constexpr int CTAS = D == 128 ? 2 : 3, NS = D == 128 ? 3 : 4;
  static constexpr int BARS = 2 * NS + 1;
  static constexpr int SMEM = NS * BYTES + 4 * ITEM_ROWS * 8 + BARS * 8 + (2 * MAX_LINES + 8) * 4 + 16 + MAX_LINES;
  static_assert(4 * ITEM_ROWS * D * 4 <= Q, "the warps' sums fit a stage");
  static_assert(ITEM_ROWS * (D * 4 + 8) <= BYTES, "... and a cluster's part");
  static_assert(BYTES % 1024 == 0, "stages begin on the swizzle's boundary");
  static_assert(CTAS * (SMEM + 1024) <= 228 * 1024, "CTAs of an SM");
};

// Rows in shared memory: 128-byte slabs of 64 elements, 16-byte chunk c of row r at chunk c ^ (r & 7): the eight rows that one ldmatrix
// phase touches lie in different banks.  Queries: whole rows, chunks turned alike.
template <int TK>
__device__ __forceinline__ uint32_t slab_at(int row, int chunk) { return (chunk >> 3) * (TK * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4); }

template <typename T, int D, bool CLUSTER, bool PACKED>
struct Worker {
  using S = Stage<D>;
  static constexpr int ROWS = 16, ROUNDS = 1;
  static constexpr int NT = S::KW / 8;        // score fragments (eight keys each) of a warp's part of a tile
  // fp16 weights reach up to 2^15 and stay normal down to 2^-23 of that of the reference
  static constexpr float BIAS = std::is_same<T, __half>::value ? 15.f - SLACK : 0.f;

  // Of rows lane / 4 and lane / 4 + 8.  Weights are exp2(scale * product - shift), shift = scale * ref - BIAS, ref the largest product q . k when it was last
  // looked for: when one came that is above limit, SLACK above it as an exponent.
  float ref[2], shift[2], limit[2];
  uint64_t sum[2];                            // (even columns, odd columns)
  float acc[D / 8][4];
  uint32_t qf[D / 16][4];

  __device__ __forceinline__ void begin(const uint8_t* stage, const AttnArgs& a) {
    const int lane = threadIdx.x & 31;
    ref[0] = ref[1] = limit[0] = limit[1] = -INFINITY;
    shift[0] = shift[1] = 0.f;
    sum[0] = sum[1] = 0;
#pragma unroll
    for (int j = 0; j < D / 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[j][e] = 0.f;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      const int row = lane & 15;
      ldmatrix4(qf[ks], smem_u32(stage) + S::Q + row * 2 * D + chunk_at(row, 2 * ks + (lane >> 4)) * 16);
#pragma unroll
      for (int e = 0; e < 4; ++e) qf[ks][e] ^= a.flip;
    }
  }

  // New reference of the rows; the sums so far follow.
  __device__ __forceinline__ void raise(const float (&top)[2], float scale_log2) {
    float by[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const bool empty = ref[r] == -INFINITY;
      ref[r] = fmaxf(ref[r], quad_max(top[r]));
      const float now = ref[r] == -INFINITY ? 0.f : fmaf(ref[r], scale_log2, -BIAS);
      by[r] = empty ? 0.f : fast_exp2(shift[r] - now);       // (sums of a row without a score so far are zeros, or NaN)
      shift[r] = now;
      limit[r] = ref[r] + SLACK / scale_log2;
      sum[r] = fmul2(sum[r], dup_f2(by[r]));
    }
#pragma unroll
    for (int j = 0; j < D / 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[j][e] *= by[e >> 1];
  }

  // Rows of V behind the last key hold anything: zeros instead.
  __device__ __forceinline__ void clear_tail(uint8_t* stage, int left) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int e = max(left, 0) * (D / 8) + lane; e < S::KW * (D / 8); e += 32)
      *reinterpret_cast<uint4*>(stage + S::V + slab_at<S::TK>(warp * S::KW + e / (D / 8), e % (D / 8))) = make_uint4(0, 0, 0, 0);
    __syncwarp();
  }

  // Is there an infinity or a NaN among the values of V that the products take?  The second number of a weight, zero or negative, would make a NaN of an infinity;
  // and where the tokens of a pack see different keys, weight 0 would not take one out.  (Zero times the values, added up: 0 or NaN.)
  static __device__ __forceinline__ bool infinite(const uint32_t (&b)[D / 16][4]) {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    const uint32_t zero = 0;
    const T2 none = *reinterpret_cast<const T2*>(&zero);
    T2 found[4] = {none, none, none, none};
#pragma unroll
    for (int j = 0; j < D / 16; ++j)
#pragma unroll
      for (int y = 0; y < 4; ++y) found[y] = __hfma2(*reinterpret_cast<const T2*>(&b[j][y]), none, found[y]);
    const T2 all = __hadd2(__hadd2(found[0], found[1]), __hadd2(found[2], found[3]));
    return __any_sync(0xffffffffu, (*reinterpret_cast<const uint32_t*>(&all) & 0x7fff7fffu) != 0);
  }
  // ... then each row takes the values of the keys that it sees, one by one, by weights in 32 bits.
  __device__ __forceinline__ void add_singly(const AttnArgs& a, const uint8_t* stage, int left, int last, const float (&p)[NT][4]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = lane & 3;
    const int sees[2] = {left - keys_short<PACKED>(a, lane >> 2, last), left - keys_short<PACKED>(a, (lane >> 2) + 8, last)};
#pragma unroll 1
    for (int key = 0; key < S::KW; ++key) {
      float w[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float even = key < 8 ? p[0][2 * r] : p[1][2 * r], odd = key < 8 ? p[0][2 * r + 1] : p[1][2 * r + 1];
        w[r] = __shfl_sync(0xffffffffu, key & 1 ? odd : even, (lane & ~3) | ((key & 7) >> 1));
      }
#pragma unroll
      for (int j = 0; j < D / 8; ++j) {
        const float2 v = unpack2<T>(lds32(stage + S::V + slab_at<S::TK>(warp * S::KW + key, j) + 4 * c));
#pragma unroll
        for (int r = 0; r < 2; ++r)
          if (key < sees[r]) {
            acc[j][2 * r] = fmaf(w[r], v.x, acc[j][2 * r]);
            acc[j][2 * r + 1] = fmaf(w[r], v.y, acc[j][2 * r + 1]);
          }
      }
    }
  }

  // One tile: this warp's keys, of which the line's last token, the `last`-th of its pack, sees the first `left`.
  __device__ __forceinline__ void tile(const AttnArgs& a, const uint8_t* stage, int left, int last) {
    const float scale_log2 = a.scale_log2;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = lane & 3;
    const uint32_t at = smem_u32(stage);
    float x[NT][4];
    const int row = warp * S::KW + (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) x[t][e] = 0.f;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      uint32_t b[4];
      ldmatrix4(b, at + slab_at<S::TK>(row, 2 * ks + ((lane >> 3) & 1)));
      mma16816<T>(x[0], qf[ks], b[0], b[1]);
      mma16816<T>(x[1], qf[ks], b[2], b[3]);
    }
    // V's fragments before the weights are known, so that their latency is hidden; kept to the products with clusters, loaded once more in the list's kernel, where their
    // registers cost spills (tokens of a batch of 32 x 8192, kept: 29.8 us, loaded again: 27.6; of 16 x 4096 by clusters, appended, too: 15.5 and 17.3).
    uint32_t v[D / 16][4];
    const int vrow = warp * S::KW + (lane & 15);
#pragma unroll
    for (int j = 0; j < D / 16; ++j) ldmatrix4t(v[j], at + S::V + slab_at<S::TK>(vrow, 2 * j + (lane >> 4)));
    const bool singly = infinite(v);
    if (left - last < S::KW) {
      const int sees[2] = {left - keys_short<PACKED>(a, lane >> 2, last), left - keys_short<PACKED>(a, (lane >> 2) + 8, last)};
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (t * 8 + 2 * c + (e & 1) >= sees[e >> 1]) x[t][e] = -INFINITY;
    }
    const float top[2] = {fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[1][0], x[1][1])), fmaxf(fmaxf(x[0][2], x[0][3]), fmaxf(x[1][2], x[1][3]))};
    if (__any_sync(0xffffffffu, top[0] > limit[0] || top[1] > limit[1])) raise(top, scale_log2);
    // Weights as the sum of two numbers of T: the second holds what the first rounds off, so that the output's own rounding is the one that
    // counts.  The products are far from the bound (a second one costs nothing that the loads do not hide).
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float p0, p1;
        unpack_f2(ffma2(pack_f2(x[t][2 * r], x[t][2 * r + 1]), dup_f2(scale_log2), dup_f2(-shift[r])), p0, p1);
        x[t][2 * r] = p0 = fast_exp2(p0);
        x[t][2 * r + 1] = p1 = fast_exp2(p1);
        sum[r] = fadd2(sum[r], pack_f2(p0, p1));
        const uint32_t w = pack2<T>(p0, p1);
        const float2 f = unpack2<T>(w);
        hi[2 * t + r] = w;
        lo[2 * t + r] = pack2<T>(p0 - f.x, p1 - f.y);
      }
    if (singly) {
      add_singly(a, stage, left, last, x);
      return;
    }
#pragma unroll
    for (int j = 0; j < D / 16; ++j) {
      if (!CLUSTER) ldmatrix4t(v[j], at + S::V + slab_at<S::TK>(vrow, 2 * j + (lane >> 4)));
      mma16816<T>(acc[2 * j], hi, v[j][0], v[j][1]);
      mma16816<T>(acc[2 * j + 1], hi, v[j][2], v[j][3]);
      mma16816<T>(acc[2 * j], lo, v[j][0], v[j][1]);
      mma16816<T>(acc[2 * j + 1], lo, v[j][2], v[j][3]);
    }
  }

  // (shift, denominator) of the rows; a warp without keys has no part, one whose scores are all NaN has
  __device__ __forceinline__ void statistics(float2* stat) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float u, v;
      unpack_f2(sum[r], u, v);
      const float l = quad_sum(u + v);
      if ((lane & 3) == 0) stat[lane / 4 + 8 * r] = make_float2(ref[r] == -INFINITY && l == 0.f ? -INFINITY : shift[r], l);
    }
  }
  // This warp's sums, rows of D floats; columns of 8 turned by the row.
  static __device__ __forceinline__ int turn(int row) { return (row & 3) << 3; }
  __device__ __forceinline__ void put(float* to, int) {
    const int lane = threadIdx.x & 31, c = lane & 3;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int row = lane / 4 + 8 * half;
#pragma unroll
      for (int j = 0; j < D / 8; ++j)
        *reinterpret_cast<float2*>(to + row * D + ((j * 8 + 2 * c) ^ turn(row))) = make_float2(acc[j][2 * half], acc[j][2 * half + 1]);
    }
  }
};

// The warp that fetches: tiles begin .. end - 1 into the ring.  full[s]: every lane arrives once its copies are there; empty[s]: the four warps that compute.
template <int D, bool CLUSTER, bool PACKED>
__device__ __forceinline__ void fetch_tiles(const AttnArgs& a, const CUtensorMap* km, const CUtensorMap* vm, const int* first, const int* keys, Walk at,
                                            int begin, int end, int items, int line0, uint32_t base, uint32_t bars, int* abort_flag) {
  using S = Stage<D>;
  constexpr int NS = S::NS, TK = S::TK;
  const int lane = threadIdx.x & 31, lines = CLUSTER ? 1 : a.lines;
  // page (not yet looked at) and slot of the run `r` of a tile; of one without keys: 0, and not to be used
  auto look_up = [&](const Walk& w, int r, int& slot) {
    slot = 0;
    const int key = w.tile * TK + (r << a.run_log2);
    if (w.line >= lines || (r << a.run_log2) >= TK || key >= keys[w.line]) return 0;
    return paged_entry(a.c, a.by_packs(line0 + w.line), key, slot);
  };
  int slot, page = look_up(at, lane, slot);
  int s = 0;
  uint32_t round = 0;
  for (int it = begin; it < end; ++it) {
    const uint32_t full = bars + 8 * s, empty = bars + 8 * (NS + s), dst = base + s * S::BYTES;
    if (round > 0 && !mbar_wait_or_abort(empty, (round - 1) & 1, abort_flag)) break;
    Walk next = at;
    next.step(first, lines, items);
    if (it + 1 == end) next.line = lines;
    int next_slot;
    const int next_page = look_up(next, lane, next_slot);              // (under way while this tile's copies are started)
    const int h = a.by_blocks(at.item), left = keys[at.line] - at.tile * TK;
    for (int r0 = 0; (r0 << a.run_log2) < min(TK, left); r0 += 32) {
      if (r0 > 0) page = look_up(at, r0 + lane, slot);                 // (runs of less than TK / 32 rows)
      const int row = (r0 + lane) << a.run_log2;
      if (row >= min(TK, left) || !paged_checked(a.c, page)) continue;
      mbar_add_tx(full, 2 * S::ROW << a.run_log2);
#pragma unroll
      for (int x = 0; x < D / 64; ++x) {
        tma_tile(dst + x * TK * 128 + row * 128, km, 64 * x, slot, h, page, full);
        tma_tile(dst + S::V + x * TK * 128 + row * 128, vm, 64 * x, slot, h, page, full);
      }
    }
    if (it == begin || at.tile == 0) {
      const uint8_t* q = query_of(a, line0 + at.line, at.item);
      constexpr int C = 2 * D / 16;
#pragma unroll
      for (int e = lane; e < ITEM_ROWS * C; e += 32) {
        const int r = e / C, chunk = e % C;
        const bool there = row_at<PACKED>(a, line0 + at.line, at.item, r).there;
        cp_async16(dst + S::Q + r * 2 * D + chunk_at(r, chunk) * 16, q + (there ? query_row<PACKED>(a, r) : 0) + chunk * 16, there ? 16 : 0);
      }
    }
    cp_async_arrive(full);
    at = next;
    page = next_page;
    slot = next_slot;
    if (++s == NS) s = 0, ++round;
  }
  // nothing leaves while copies into its memory are under way
  cp_async_wait<0>();
  if (*reinterpret_cast<volatile int*>(abort_flag)) {
    // (the last NS tiles that were started: stages s .. NS - 1 of the round before, 0 .. s - 1 of this one)
    for (int y = 0; y < NS; ++y) {
      const uint32_t r = y < s ? round : round - 1;
      if (y < s || round > 0) mbar_wait(bars + 8 * y, r & 1);
    }
  }
}

template <typename T, int D, bool CLUSTER, bool PACKED>
__global__ void __launch_bounds__(THREADS, Stage<D>::CTAS)
    paged_attn_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ CUtensorMap km, const __grid_constant__ CUtensorMap vm) {
  using S = Stage<D>;
  constexpr int NS = S::NS, TK = S::TK;
  extern __shared__ __align__(1024) uint8_t smem[];
  float2* stat = reinterpret_cast<float2*>(smem + NS * S::BYTES);            // [4][ITEM_ROWS]
  int* first = reinterpret_cast<int*>(stat + 4 * ITEM_ROWS);                 // [lines + 1]
  int* abort_flag = first + MAX_LINES + 3;
  int* keys = first + MAX_LINES + 4;                                         // [lines]
  const uint32_t base = smem_u32(smem), bars = smem_u32(keys + MAX_LINES);   // full[NS], empty[NS], join
  int* warp_sum = keys + MAX_LINES + 2 * S::BARS;                            // [4]
  uint8_t* lasts = reinterpret_cast<uint8_t*>(warp_sum + 4);                 // [lines]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int items = a.Hk * a.blocks;
  if (tid == 0) {
    for (int y = 0; y < NS; ++y) {
      mbar_init(bars + 8 * y, 32);
      mbar_init(bars + 8 * (NS + y), 4);
    }
    mbar_init(bars + 8 * 2 * NS, 4);
    mbar_fence_init();
    *abort_flag = 0;
    if (a.c.pages > 0) {                       // (a pool without pages has no maps)
      asm volatile("prefetch.tensormap [%0];" ::"l"(&km) : "memory");
      asm volatile("prefetch.tensormap [%0];" ::"l"(&vm) : "memory");
    }
  }
  // The kernel behind is let in at the end: its CTAs would take the places that come free one by one, several on some SMs and none on others
  // (1 x 131072 tokens, 32 heads x 64, passes back to back: 242 us with an early release, 165 without).
  if (CLUSTER) chain_release();              // (short kernels, fewer CTAs than there is room for: the next one may be placed at once)
  chain_wait();
  // (parts of one tile would be as many to join as tiles: 1 x 8000 tokens, two K/V heads: 15.5 us, 12.5 with parts of two)
  int begin, end, line0;
  Walk at = take_part<T, D, CLUSTER>(a, TK, 2, first, keys, lasts, warp_sum, items, begin, end, line0);
  const int lines = CLUSTER ? 1 : a.lines, item = at.item;
  if (begin >= end && (!CLUSTER || keys[0] == 0)) return;
  if (warp == 4) {
    if (begin < end) fetch_tiles<D, CLUSTER, PACKED>(a, &km, &vm, first, keys, at, begin, end, items, line0, base, bars, abort_flag);
    if (CLUSTER) {                             // (these threads count in the cluster's barriers)
      __syncwarp();
      cluster_sync();
      cluster_sync();
    }
    return;
  }

  Worker<T, D, CLUSTER, PACKED> w;
  const uint32_t join_bar = bars + 8 * 2 * NS;
  uint32_t joined = 0;
  auto join = [&]() {
    __syncwarp();
    if (lane == 0) mbar_arrive(join_bar);
    return mbar_wait_or_abort(join_bar, joined++ & 1, abort_flag);
  };
  // with clusters: this CTA's part, in the same place of every CTA (no stage is used any more when it is written)
  float* cluster_sums = reinterpret_cast<float*>(smem);
  float2* cluster_stat = reinterpret_cast<float2*>(cluster_sums + ITEM_ROWS * D);
  int s = 0;
  uint32_t round = 0;
  bool ok = true;
#pragma unroll 1
  for (int it = begin; it < end; ++it) {
    uint8_t* stage = smem + s * S::BYTES;
    ok = mbar_wait_or_abort(bars + 8 * s, round & 1, abort_flag);
    if (!ok) break;
    if (it == begin || at.tile == 0) w.begin(stage, a);
    const int left = keys[at.line] - at.tile * TK - warp * S::KW;
    if (left < S::KW) w.clear_tail(stage, left);
    const int last = PACKED ? lasts[at.line] : 0;
    w.tile(a, stage, left, last);
    const bool ends = at.tile == at.tiles - 1 || it == end - 1;
    if (ends) {
      ok = finish_item<T, D, 16 * D, CLUSTER, PACKED>(a, w, stat, reinterpret_cast<float*>(stage), at, first, items, begin, end, it == end - 1, line0, keys[at.line], last, cluster_sums, cluster_stat,
                                              join);
      if (!ok) break;
    }
    // the stage is free (what was written to it by stores before what copies write to it next)
    if (ends || left < S::KW) fence_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(bars + 8 * (NS + s));
    at.step(first, lines, items);
    if (++s == NS) s = 0, ++round;
  }
  if constexpr (CLUSTER) {
    if (begin >= end || !ok) {
      if (tid < ITEM_ROWS) cluster_stat[tid] = make_float2(-INFINITY, -1.f);
    }
    __syncwarp();
    cluster_finish<T, D, PACKED>(a, cluster_sums, cluster_stat, line0, item, keys[0], lasts[0]);
  }
  if (!ok && !CLUSTER && tid == 0) a.head[blockIdx.x] = make_int4(0, 0, 0, 0);       // nothing to join from here
  if (!ok && lane == 0) report_timeout(a.c.status, a.c.status_host);
  chain_release();
}

// Joins the parts of the items that cross from one CTA's list to the next.  Block (c, y): rows ROWS y .. of the item that begins in CTA c's list and ends behind it;
// WARPS warps a row, each every WARPS-th part.  Latency alone, 3 to 5 us: a chain of four loads, and one more for every eight parts of a warp.
template <typename T, int D, int ROWS, int WARPS>
__global__ void __launch_bounds__(32 * WARPS * ROWS) paged_combine_kernel(const __grid_constant__ AttnArgs a) {
  constexpr int LANES = 32 * WARPS;
  __shared__ float red[ROWS][WARPS][D];
  __shared__ float red_m[ROWS][WARPS], red_l[ROWS][WARPS];
  chain_wait();
  const int c = blockIdx.x, sub = threadIdx.x / LANES, row = blockIdx.y * ROWS + sub, tid = threadIdx.x % LANES, warp = tid >> 5, lane = tid & 31;
  const int total = a.meta[0], per = a.meta[1];
  if ((int64_t)(c + 1) * per >= total) return;
  const int4 hd = a.head[c];
  if (hd.y <= (c + 1) * per || hd.x < c * per) return;                 // ends here, or began before
  int token;
  const int keys = keys_of(a, hd.z, token);
  const RowAt ra = row_at<true>(a, hd.z, hd.w, row, keys, token);
  const int last = (hd.y - 1) / per, pieces = ra.there ? last - c + 1 : 0;
  auto slot = [&](int p) { return 2 * (c + p) + (p == 0 && hd.x > c * per ? 1 : 0); };
  float m = -INFINITY;
  for (int p = tid; p < pieces; p += LANES) m = fmaxf(m, a.part_stat[slot(p) * ITEM_ROWS + row].x);
#pragma unroll
  for (int s = 1; s < 32; s *= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, s));
  if (lane == 0) red_m[sub][warp] = m;
  __syncthreads();
#pragma unroll
  for (int x = 0; x < WARPS; ++x) m = fmaxf(m, red_m[sub][x]);
  // pieces p = warp, warp + WARPS, ...: a lane D / 32 columns
  constexpr int E = D / 32;
  float v[E], l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) v[e] = 0.f;
#pragma unroll 8
  for (int p = warp; p < pieces; p += WARPS) {
    const float2 st = a.part_stat[slot(p) * ITEM_ROWS + row];
    const float* src = a.part + ((int64_t)slot(p) * ITEM_ROWS + row) * D + lane * E;
    float y[E];
    if constexpr (E == 4) {
      const float4 f = *reinterpret_cast<const float4*>(src);
      y[0] = f.x, y[1] = f.y, y[2] = f.z, y[3] = f.w;
    } else {
      const float2 f = *reinterpret_cast<const float2*>(src);
      y[0] = f.x, y[1] = f.y;
    }
    const float w = st.x == -INFINITY ? 0.f : fast_exp2(st.x - m);
    l = fmaf(w, st.y, l);
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = fmaf(w, y[e], v[e]);
  }
#pragma unroll
  for (int e = 0; e < E; ++e) red[sub][warp][lane * E + e] = v[e];
  if (lane == 0) red_l[sub][warp] = l;
  __syncthreads();
  if (!ra.there) return;
  l = red_l[sub][0];
#pragma unroll
  for (int x = 1; x < WARPS; ++x) l += red_l[sub][x];
  if (tid < D) {
    float y = red[sub][0][tid];
#pragma unroll
    for (int x = 1; x < WARPS; ++x) y += red[sub][x][tid];
    ((T*)a.o)[ra.o * D + tid] = from_f32<T>(ra.empty ? 0.f : y / l);
  }
  if (tid == 0) a.lse[ra.lse] = ra.empty ? -INFINITY : (m + log2f(l)) * LN2;
}

int attn_tile(const ha_paged_params& p) { return p.bits == 16 ? Stage<64>::TK : attn4_tile(p.d); }
// Tokens of a sequence that share an item's rows, and items of a (pack, K/V head).
int attn_pack(const ha_paged_params& p) {
  const int group = p.H / p.Hk, most = group < ITEM_ROWS ? ITEM_ROWS / group : 1;
  return p.n < most ? (p.n > 0 ? p.n : 1) : most;
}
int64_t attn_packs(const ha_paged_params& p) { return ((int64_t)p.n + attn_pack(p) - 1) / attn_pack(p); }
int attn_rows(const ha_paged_params& p) { return p.H / p.Hk * attn_pack(p); }
int attn_items(const ha_paged_params& p) { return p.Hk * ((p.H / p.Hk + ITEM_ROWS - 1) / ITEM_ROWS); }
int attn_resident(const ha_paged_params& p) {
  if (p.bits == 16) return p.d == 128 ? Stage<128>::CTAS : Stage<64>::CTAS;
  return attn4_resident(p.d, attn_rows(p));
}

// CTAs of a launch over `lines` lines: as many as are resident at once, and no more than there can be tiles.
int attn_ctas(const ha_paged_params& p, int lines) {
  const int tk = attn_tile(p), items = attn_items(p);
  const int64_t most = ((int64_t)p.columns * p.page_size + tk - 1) / tk * items * lines;
  const int resident = sm_count() * attn_resident(p);
  return (int)(most < 1 ? 1 : most < resident ? most : resident);
}

// Does the device hold a cluster of 16, which a part of a GPU need not?  Asked once a device, of the kernel with the most shared memory.
bool clusters_of_16() {
  static std::atomic<int> cache[64];       // 0: not asked, 1: yes, 2: no
  int dev = 0, known = 0;
  if (cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < 64) known = cache[dev].load(std::memory_order_relaxed);
  if (known != 0) return known == 1;
  auto kernel = paged_attn_kernel<__nv_bfloat16, 128, true, false>;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = 16;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = 16;
  cfg.blockDim = THREADS;
  cfg.dynamicSmemBytes = Stage<128>::SMEM;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  int held = 0;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Stage<128>::SMEM) != cudaSuccess ||
      cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&held, kernel, &cfg) != cudaSuccess) {
    held = 0;
    cudaGetLastError();                    // (an answer, not a failure of the call)
  }
  if (dev >= 0 && dev < 64) cache[dev].store(held > 0 ? 1 : 2, std::memory_order_relaxed);
  return held > 0;
}

// CTAs that share an item as a cluster, or 0.  Short contexts and few items: a cluster joins its parts over distributed shared memory, without a workspace and a
// second launch (1 x 515 tokens, two K/V heads: 8.2 -> 6.9 us on the device, 7.1 -> 2.7 us for the call).  Every item gets the same CTAs, however long it is, so that
// the list of tiles, which deals them out evenly, is for what takes longer than the joining: with CLUSTER_TILES 7 a batch of 16 x 4096 goes by the list, 17.4 us for 15.3 (1 x 5000 gains:
// 12.1 for 13.6); with 20, 1 x 8000 by clusters of 8, 19.5 us for 12.5; with 40 a batch of 32 x 8192, 37 us for 28.
// Clusters of 16 (more than every GPU promises) where the device holds them and they take no more than half of the room, since they need theirs within a part of the GPU: 1 x 515
// 7.05 -> 6.5 us, 1 x 5000 13.8 -> 10.0, 1 x 2051 in 4 bits 10.2 -> 9.2, 1 x 8000 in 4 bits 16.7 -> 12.2 (with all of the room 8 x 1000 took 13.7 us, by clusters of 8 7.7).  At
// eight tiles a CTA the list is faster again: 1 x 8000 12.5 and 12.1 us, 1 x 16000 in 4 bits 17.2 and 15.6.
int attn_cluster(const ha_paged_params& p) {
  const int64_t units = p.B * attn_packs(p) * attn_items(p);
  const int64_t tiles = ((int64_t)p.columns * p.page_size + attn_tile(p) - 1) / attn_tile(p), resident = (int64_t)sm_count() * attn_resident(p);
  if (units > resident || tiles == 0) return 0;
  int c = 1;
  while (c < 8 && c < tiles && units * 2 * c <= resident) c *= 2;
  if (c == 8 && tiles > 8 && units * 32 <= resident && clusters_of_16()) c = 16;
  return (tiles + c - 1) / c <= (c == 16 ? CLUSTER_TILES_16 : CLUSTER_TILES) ? c : 0;
}

// Lines of one launch: no more than shared memory counts, their tiles within 31 bits.
int64_t attn_lines(const ha_paged_params& p) {
  const int tk = attn_tile(p), items = attn_items(p);
  const int64_t tiles = ((int64_t)p.columns * p.page_size + tk - 1) / tk * items, all = p.B * attn_packs(p);
  int64_t lines = all < MAX_LINES ? all : MAX_LINES;
  if (tiles > 0 && lines > (0x7fffffffLL - 65536) / tiles) lines = (0x7fffffffLL - 65536) / tiles;
  return lines;
}

// Tensor maps of K and V pages: boxes of as many rows as both a page and a tile are made of.
bool attn_maps(const ha_paged_params& p, CUtensorMap* maps) {
  if (p.pages == 0) return true;
  const int run = std::gcd(p.page_size, BOX_ROWS);
  const int64_t row = p.page_size == 1 ? p.d : p.page_st;
  return encode_tile_map(&maps[0], p.dtype, p.k_pages, p.d, p.page_size, p.Hk, p.pages, row, p.page_sh, p.page_sp, run) &&
         encode_tile_map(&maps[1], p.dtype, p.v_pages, p.d, p.page_size, p.Hk, p.pages, row, p.page_sh, p.page_sp, run);
}

int64_t attn_workspace(const ha_paged_params& p, int ctas) { return 256 + (int64_t)ctas * (16 + 2 * ITEM_ROWS * (p.d * 4 + 8)); }

template <typename T, int D>
int launch_attn(const AttnArgs& a, const ha_paged_params& p, int ctas, cudaStream_t st) {
  using S = Stage<D>;
  CUtensorMap maps[2] = {};
  if (p.maps) memcpy(maps, p.maps, sizeof(maps));
  else if (!attn_maps(p, maps)) return HA_ERR_INVALID;
  auto launch = [&](auto kernel) {
    if (a.cluster > 0) launch_chained_clusters(kernel, ctas, THREADS, S::SMEM, a.cluster, st, a, maps[0], maps[1]);
    else launch_chained(kernel, ctas, THREADS, S::SMEM, st, a, maps[0], maps[1]);
  };
#define HA_PAGED_VARIANT(cluster, packed)                                                          \
  do {                                                                                             \
    HA_SMEM_ATTR_ONCE((paged_attn_kernel<T, D, cluster, packed>), S::SMEM, "ha_paged_attn");       \
    if (cluster) HA_ATTR_ONCE((paged_attn_kernel<T, D, cluster, packed>), cudaFuncAttributeNonPortableClusterSizeAllowed, 1, "ha_paged_attn"); \
    launch(paged_attn_kernel<T, D, cluster, packed>);                                              \
  } while (0)
  if (a.cluster > 0 && a.pack > 1) HA_PAGED_VARIANT(true, true);
  else if (a.cluster > 0) HA_PAGED_VARIANT(true, false);
  else if (a.pack > 1) HA_PAGED_VARIANT(false, true);
  else HA_PAGED_VARIANT(false, false);
#undef HA_PAGED_VARIANT
  HA_LAUNCHED("ha_paged_attn");
  return HA_OK;
}

template <int ROWS, int WARPS>
int launch_combine(const AttnArgs& a, const ha_paged_params& p, int ctas, cudaStream_t st) {
  const dim3 grid(ctas - 1, (std::min(attn_rows(p), ITEM_ROWS) + ROWS - 1) / ROWS);
  auto launch = [&](auto kernel) { launch_chained(kernel, grid, 32 * WARPS * ROWS, 0, st, a); };
  if (p.d == 64) {
    if (p.dtype == HA_BF16) launch(paged_combine_kernel<__nv_bfloat16, 64, ROWS, WARPS>);
    else launch(paged_combine_kernel<__half, 64, ROWS, WARPS>);
  } else {
    if (p.dtype == HA_BF16) launch(paged_combine_kernel<__nv_bfloat16, 128, ROWS, WARPS>);
    else launch(paged_combine_kernel<__half, 128, ROWS, WARPS>);
  }
  HA_LAUNCHED("ha_paged_attn");
  return HA_OK;
}

int attn_check(const ha_paged_params& p) {
  const int rc = paged_check(p);
  if (rc != HA_OK) return rc;
  // (by a scale below that the room above a reference, SLACK / scale, would be infinite)
  if (p.H < 1 || !(fabsf(p.scale) >= 0x1p-100f) || isinf(p.scale)) return HA_ERR_INVALID;
  if ((int64_t)p.B * p.n > 0x7fffffffLL - 65536 || (int64_t)p.H * p.d > 1 << 24) return HA_ERR_TOO_LARGE;
  if (p.B > 0 && p.n > 0 && attn_lines(p) < 1) return HA_ERR_TOO_LARGE;
  return HA_OK;
}

}  // namespace
}  // namespace ha

using namespace ha;

extern "C" {

int ha_paged_maps(const ha_paged_params* pp, void* maps) {
  if (!pp || !maps) return HA_ERR_INVALID;
  const ha_paged_params& p = *pp;
  ha_paged_params q = p;
  q.B = 0;
  const int rc = paged_check(q);
  if (rc != HA_OK) return rc;
  CUtensorMap m[2] = {};
  if (p.bits == 16 && !attn_maps(p, m)) return HA_ERR_INVALID;
  memcpy(maps, m, sizeof(m));
  return HA_OK;
}

int64_t ha_paged_attn_workspace_bytes(const ha_paged_params* pp) {
  if (!pp) return HA_ERR_INVALID;
  // (sizes alone: the pointers may be missing)
  const ha_paged_params& p = *pp;
  if ((p.bits != 16 && p.bits != 4) || (p.d != 64 && p.d != 128) || p.B < 0 || p.n < 0 || p.Hk < 1 || p.H < 1 || p.H % p.Hk != 0 || p.columns < 0 || p.page_size < 1)
    return HA_ERR_INVALID;
  if ((int64_t)p.columns * p.page_size > PAGED_MOST) return HA_ERR_TOO_LARGE;
  const int64_t all = p.B * attn_packs(p), lines = attn_lines(p);
  if (all == 0 || attn_cluster(p) > 0) return 0;
  return lines < 1 ? (int64_t)HA_ERR_TOO_LARGE : attn_workspace(p, attn_ctas(p, (int)lines));
}

int ha_paged_attn(const ha_paged_params* pp, void* stream) {
  if (!pp) return HA_ERR_INVALID;
  const ha_paged_params& p = *pp;
  const int rc = attn_check(p);
  if (rc != HA_OK) return rc;
  if (p.B == 0 || p.n == 0) return HA_OK;
  if (!p.q || !p.o || !p.lse || ((uintptr_t)p.q | (uintptr_t)p.o) % 16 != 0 || (p.q_sb | p.q_sn | p.q_sh) % 8 != 0) return HA_ERR_INVALID;
  const int ctas = attn_ctas(p, (int)attn_lines(p));
  const int cluster = attn_cluster(p);
  if (cluster == 0 && (!p.workspace || (uintptr_t)p.workspace % 16 != 0 || p.workspace_bytes < attn_workspace(p, ctas))) return HA_ERR_WORKSPACE;
  AttnArgs a = {};
  a.c = paged_view(p);
  a.q = (const uint8_t*)p.q;
  a.q_sb = p.q_sb * 2; a.q_sn = p.q_sn * 2; a.q_sh = p.q_sh * 2;
  a.o = p.o; a.lse = p.lse;
  a.n = p.n; a.H = p.H; a.Hk = p.Hk; a.group = p.H / p.Hk; a.blocks = (a.group + ITEM_ROWS - 1) / ITEM_ROWS;
  a.pack = attn_pack(p); a.packs = (int)attn_packs(p);
  a.by_packs = FastDiv((uint32_t)a.packs); a.by_blocks = FastDiv((uint32_t)a.blocks); a.by_group = FastDiv((uint32_t)a.group);
  a.scale_log2 = fabsf(p.scale) * LOG2E;
  a.flip = p.scale < 0.f ? 0x80008000u : 0u;
  a.cluster = cluster;
  uint8_t* ws = (uint8_t*)p.workspace;
  a.meta = (int32_t*)ws;
  a.head = (int4*)(ws + 256);
  a.part_stat = (float2*)(ws + 256 + (int64_t)ctas * 16);
  a.part = (float*)(ws + 256 + (int64_t)ctas * (16 + 2 * ITEM_ROWS * 8));
  if (p.bits == 16) {
    while ((1 << a.run_log2) < std::gcd(p.page_size, BOX_ROWS)) ++a.run_log2;
  } else {
    const int part = attn_tile(p) / 4, run = 1024 / p.d, sc = p.d / PAGED_GROUP * 4;
    const bool together = a.c.st == p.d / 2 && a.c.sst == sc &&
                   ((uintptr_t)p.k_scales | (uintptr_t)p.v_scales | (uintptr_t)a.c.ssp | (uintptr_t)a.c.ssh) % 16 == 0;
    a.runs = !together ? 0 : p.page_size % part == 0 ? 2 : p.page_size % run == 0 ? 1 : 0;
  }
  const cudaStream_t st = (cudaStream_t)stream;
  const bool bf = p.dtype == HA_BF16;
  const int64_t all = p.B * attn_packs(p), most = cluster > 0 ? all : attn_lines(p);
  for (int64_t line0 = 0; line0 < all; line0 += most) {
    a.line0 = (int)line0;
    a.lines = (int)(all - line0 < most ? all - line0 : most);
    const int now = cluster > 0 ? a.lines * p.Hk * a.blocks * cluster : attn_ctas(p, a.lines);
    int rc;
    if (p.bits == 4) rc = attn4_launch(a, p.dtype, p.d, now, st);
    else if (p.d == 64) rc = bf ? launch_attn<__nv_bfloat16, 64>(a, p, now, st) : launch_attn<__half, 64>(a, p, now, st);
    else rc = bf ? launch_attn<__nv_bfloat16, 128>(a, p, now, st) : launch_attn<__half, 128>(a, p, now, st);
    if (rc != HA_OK) return rc;
    if (now == 1 || cluster > 0) continue;
    // many parts of an item: more warps to a row (1 x 32768 tokens, two K/V heads, 148 parts each: 16.8 us, 18.1 by four warps; 4 x 30000, 37 parts: 21.8 and 22.3); few: fewer
    // blocks (8 x 30000, 18 parts: 28.7 us by two rows of four warps, 29.8 by eight warps a row; 32 x 8192: 27.1 and 29.2)
    if (now >= 32 * all * attn_items(p)) rc = launch_combine<1, 8>(a, p, now, st);
    else rc = launch_combine<2, 4>(a, p, now, st);
    if (rc != HA_OK) return rc;
  }
  return HA_OK;
}

}  // extern "C"
