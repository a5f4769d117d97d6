// Attention of a sequence's last tokens over its pages: one pass over K and V, split over the whole GPU.
//
//   s_j = scale q . k_j,  o = sum_j exp(s_j) v_j / sum_j exp(s_j),  lse = log sum_j exp(s_j),  j < keys of the row
//
// An item is the (up to 16) query heads of one token that share a K/V head: the 16 rows of mma.sync.m16n8k16, which is what one pass over the
// keys can serve.  The products are thin (16 query rows against all keys), and K and V are read once: bytes bound the kernel,
// and the operands go from shared memory to registers, where a 4-bit row has to pass anyway to become one.  A query row sees all or
// none of an item's keys, so that no masked value meets a product with weight 0.
//
// All items' keys, in tiles of TK, form one list; CTA c takes the c-th equal part of it, whatever the lengths are.  An item that lies within one CTA is
// finished there; of one that crosses to the next, each CTA writes its part (unnormalised sums, reference, denominator) to the workspace,
// and paged_combine_kernel adds them up in the order of the keys.  A CTA's own parts of an item: at most the first and the last of its list.
//
// A CTA: four warps that compute, each a quarter of a tile's keys with its own running maximum and sums, which are joined at the item's end; and one that
// fetches tiles into a ring of NS stages, across items: 16-bit rows by tensor copies (128-byte swizzle; boxes of as many rows as both a page and a
// tile are made of, so that any page size will do), 4-bit rows by plain bulk copies, queries and scales by cp.async.
#include <string.h>

#include <numeric>
#include <type_traits>

#include "paged.cuh"
#include "tensor_map.cuh"

namespace ha {

namespace {

constexpr int ITEM_ROWS = 16;
constexpr int MAX_LINES = 256;        // (sequence, token) pairs of one launch: their tiles are summed up in shared memory
constexpr int THREADS = 160;
constexpr float LN2 = 0.693147180559945309f, LOG2E = 1.44269504088896341f;

struct AttnArgs {
  PagedView c;
  const uint8_t* q;
  int64_t q_sb, q_sn, q_sh;           // bytes
  void* o;
  float* lse;
  int32_t n, H, Hk, group, blocks;    // blocks: items of a (token, K/V head): group / 16, rounded up
  int32_t line0, lines;               // (sequence, token) pairs of this launch
  int32_t run_log2;                   // rows that are fetched together: 2^run_log2, the largest power of two that pages and tiles are made of
  FastDiv by_n, by_blocks;
  float scale_log2;                   // magnitude of the softmax scale, times log2 e
  uint32_t flip;                      // sign bits of a pair of queries, where the scale is negative
  float* part;                        // [CTAs][2][ITEM_ROWS][D], then ...
  float2* part_stat;                  // [CTAs][2][ITEM_ROWS]: reference (log2), denominator
  int4* head;                         // [CTAs]: last item's first and end tile, its line, its number
  int32_t* meta;                      // all tiles, tiles of a CTA
};

template <int D, int BITS>
struct Stage {
  static constexpr int KW = BITS == 16 ? 16 : 32;            // keys of a warp
  static constexpr int TK = 4 * KW;
  static constexpr int ROW = BITS == 16 ? 2 * D : D / 2;     // bytes of a row
  static constexpr int G = D / PAGED_GROUP;
  static constexpr int SC = BITS == 16 ? 4 : 4 * G;          // bytes of a row's scales (16 bits: none)
  static constexpr int V = TK * ROW, KS = 2 * TK * ROW, VS = KS + (BITS == 16 ? 0 : TK * SC), Q = VS + (BITS == 16 ? 0 : TK * SC);
  static constexpr int BYTES = Q + ITEM_ROWS * 2 * D;
  static constexpr int CTAS = BITS == 16 ? (D == 128 ? 2 : 3) : 2;
  static constexpr int NS = BITS == 16 ? (D == 128 ? 3 : 4) : (D == 128 ? 4 : 8);
  static constexpr int ROUNDS = BITS == 16 ? 1 : 2;          // in which the warps' sums are joined: column ranges that fit a stage
  static constexpr int BARS = 2 * NS + 1;
  static constexpr int SMEM = NS * BYTES + 4 * ITEM_ROWS * 8 + BARS * 8 + (2 * MAX_LINES + 8) * 4 + 16;
  static_assert(4 * ITEM_ROWS * D / ROUNDS * 4 <= Q, "the warps' sums fit a stage");
  static_assert(BYTES % (BITS == 16 ? 1024 : 128) == 0, "stages begin on the swizzle's boundary");
  static_assert(CTAS * (SMEM + 1024) <= 228 * 1024, "CTAs of an SM");
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
// contiguous bytes (16-byte aligned, a multiple of 16) to shared memory, counted on `bar`
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
// an arrival on `bar` once this thread's cp.async so far are done
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) { asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ uint64_t dup_f2(float v) { return pack_f2(v, v); }
__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}
// 16-bit rows in shared memory: 128-byte slabs of 64 elements, 16-byte chunk c of row r at chunk c ^ (r & 7): the eight rows that one ldmatrix
// phase (or one quarter of a 128-bit load) touches lie in different banks.  Queries: whole rows, chunks turned alike.
template <int TK>
__device__ __forceinline__ uint32_t slab_at(int row, int chunk) { return (chunk >> 3) * (TK * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4); }
__device__ __forceinline__ int chunk_at(int row, int chunk) { return chunk ^ (row & 7); }
// 4-bit rows lie in key order.  Column 2c + e of a score fragment is key c + 4e of its eight: the four keys that one load of V takes then are
// neighbours, two to a bank instead of four.  Scales lie in column order: a lane's two keys side by side.
__device__ __forceinline__ int column_of(int key) { return (key & ~7) | ((key & 3) << 1) | ((key >> 2) & 1); }
__device__ __forceinline__ int key_of(int column) { return (column >> 1) | ((column & 1) << 2); }

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

template <typename T, int D, int BITS>
struct Worker {
  using S = Stage<D, BITS>;
  static constexpr int NT = S::KW / 8;        // score fragments (eight keys each) of a warp's part of a tile
  // (fp16 weights) weights reach up to 2^15 and stay normal down to 2^-29 of the largest
  static constexpr float BIAS = BITS == 4 || std::is_same<T, __half>::value ? 15.f : 0.f;

  // of rows lane / 4 and lane / 4 + 8.  Weights are exp2(score - shift); 16 bits: ref is the largest product q . k so far, shift = ref * scale - BIAS;
  // 4 bits: ref is the largest score so far, shift = ref + v_exp - BIAS, so that weight * step stays within fp16, too
  float ref[2], shift[2];
  uint64_t sum[2];                            // (even columns, odd columns)
  float acc[D / 8][4];
  uint32_t qf[D / 16][4];
  // 4-bit rows
  float q_unit[2], q_sum[S::G][2];            // score of a code sum; sum of the row's elements of a group, times the softmax scale
  float weight[S::G][4];                      // sums of the rounded weights of even columns, less those of odd ones (every column alike)
  uint64_t offset[S::G][2];                   // sums of weights times what a row's middle code stands for
  float v_exp;                                // power of two that no V step so far exceeds

  __device__ __forceinline__ void begin(const uint8_t* stage, const AttnArgs& a) {
    const int lane = threadIdx.x & 31;
    ref[0] = ref[1] = -INFINITY;
    shift[0] = shift[1] = 0.f;
    sum[0] = sum[1] = 0;
#pragma unroll
    for (int j = 0; j < D / 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[j][e] = 0.f;
    const uint8_t* q = stage + S::Q;
    if constexpr (BITS == 16) {
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        const int row = lane & 15;
        ldmatrix4(qf[ks], smem_u32(q) + row * 2 * D + chunk_at(row, 2 * ks + (lane >> 4)) * 16);
#pragma unroll
        for (int e = 0; e < 4; ++e) qf[ks][e] ^= a.flip;
      }
    } else {
      // Queries as fp16 operands: every row times the power of two that brings its largest element to 2^13 .. 2^14.  Lane c of a row's four
      // holds elements 16 c .. 16 c + 15 of each group, paired as the codes come out of their words: (0, 4), (1, 5) / 16, (2, 6), (3, 7) / 16.
      const int c = lane & 3;
      v_exp = -24.f;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int row = lane / 4 + 8 * half;
        float x[S::G][16], top = 0.f;
#pragma unroll
        for (int g = 0; g < S::G; ++g) {
          float s = 0.f;
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const uint4 w = lds128(q + row * 2 * D + chunk_at(row, 8 * g + 2 * c + u) * 16);
            const uint32_t ws[4] = {w.x ^ a.flip, w.y ^ a.flip, w.z ^ a.flip, w.w ^ a.flip};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float2 f = unpack2<T>(ws[j]);
              x[g][8 * u + 2 * j] = f.x;
              x[g][8 * u + 2 * j + 1] = f.y;
              s += f.x + f.y;
              top = max_nan(top, max_nan(fabsf(f.x), fabsf(f.y)));
            }
          }
          q_sum[g][half] = quad_sum(s) * a.scale_log2;
          weight[g][2 * half] = weight[g][2 * half + 1] = 0.f;
          offset[g][half] = 0;
        }
        top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // exponent of the largest element; a row of zeros stays one, one with a NaN or an infinity keeps it through the products
        const int e = max((int)(__float_as_uint(top) >> 23) & 255, 27);
        const float up = __uint_as_float((uint32_t)(127 + 13 + 127 - e) << 23), down = __uint_as_float((uint32_t)(e - 13) << 23);
        // codes are the subnormal fp16 numbers code * 2^-24 (or * 2^-20, against a sixteenth of the query's element)
        q_unit[half] = down * 16777216.f * a.scale_log2;
#pragma unroll
        for (int g = 0; g < S::G; ++g)
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float* e8 = &x[g][8 * u + 2 * h];
              qf[(g * 2 + u) * 2 + h][half] = pack2<__half>(e8[0] * up, e8[4] * up);
              qf[(g * 2 + u) * 2 + h][2 + half] = pack2<__half>(e8[1] * up * 0.0625f, e8[5] * up * 0.0625f);
            }
      }
    }
  }

  // New reference of the rows whose maximum grew (and of all, where a V step did); the sums so far follow.
  __device__ __forceinline__ void raise(const float (&top)[2], float v_top, float scale_log2) {
    float by[2];
    if constexpr (BITS == 4) {
#pragma unroll
      for (int s = 1; s < 32; s *= 2) v_top = fmaxf(v_top, __shfl_xor_sync(0xffffffffu, v_top, s));
      v_exp = fmaxf(v_exp, (float)((int)(__float_as_uint(v_top) >> 23) - 126));
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const bool empty = ref[r] == -INFINITY;
      ref[r] = fmaxf(ref[r], quad_max(top[r]));
      const float now = ref[r] == -INFINITY ? 0.f : BITS == 4 ? ref[r] + (v_exp - BIAS) : fmaf(ref[r], scale_log2, -BIAS);
      by[r] = empty ? 0.f : fast_exp2(shift[r] - now);
      // (sums of a row without a score so far are zeros, or NaN)
      shift[r] = now;
      sum[r] = fmul2(sum[r], dup_f2(by[r]));
    }
#pragma unroll
    for (int j = 0; j < D / 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[j][e] *= by[e >> 1];
    if constexpr (BITS == 4) {
#pragma unroll
      for (int g = 0; g < S::G; ++g) {
#pragma unroll
        for (int e = 0; e < 4; ++e) weight[g][e] *= by[e >> 1];
        offset[g][0] = fmul2(offset[g][0], dup_f2(by[0]));
        offset[g][1] = fmul2(offset[g][1], dup_f2(by[1]));
      }
    }
  }

  // Rows of V (4 bits: their scales) behind the last key hold anything: zeros instead.
  __device__ __forceinline__ void clear_tail(uint8_t* stage, int left) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    left = max(left, 0);
    if constexpr (BITS == 16) {
      for (int e = left * (D / 8) + lane; e < S::KW * (D / 8); e += 32) *reinterpret_cast<uint4*>(stage + S::V + slab_at<S::TK>(warp * S::KW + e / (D / 8), e % (D / 8))) = make_uint4(0, 0, 0, 0);
    } else {
      for (int e = left * S::G + lane; e < S::KW * S::G; e += 32) *reinterpret_cast<uint32_t*>(stage + S::VS + column_of(warp * S::KW + e / S::G) * S::SC + e % S::G * 4) = 0;
    }
    __syncwarp();
  }

  // One tile: this warp's keys, of which the first `left` exist.
  __device__ __forceinline__ void tile(const uint8_t* stage, int left, float scale_log2) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = lane & 3;
    if constexpr (BITS == 16) {
      float x[NT][4];
      const int row = warp * S::KW + (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[t][e] = 0.f;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        uint32_t b[4];
        ldmatrix4(b, smem_u32(stage) + slab_at<S::TK>(row, 2 * ks + ((lane >> 3) & 1)));
        mma16816<T>(x[0], qf[ks], b[0], b[1]);
        mma16816<T>(x[1], qf[ks], b[2], b[3]);
      }
      if (left < S::KW) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (t * 8 + 2 * c + (e & 1) >= left) x[t][e] = -INFINITY;
      }
      const float top[2] = {fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[1][0], x[1][1])), fmaxf(fmaxf(x[0][2], x[0][3]), fmaxf(x[1][2], x[1][3]))};
      if (__any_sync(0xffffffffu, top[0] > ref[0] || top[1] > ref[1])) raise(top, 0.f, scale_log2);
      // Weights as the sum of two numbers of T: the second holds what the first rounds off, so that the output's own rounding is the one that
      // counts.  The products are far from the bound (a second one costs nothing that the loads do not hide).
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float p0, p1;
          unpack_f2(ffma2(pack_f2(x[t][2 * r], x[t][2 * r + 1]), dup_f2(scale_log2), dup_f2(-shift[r])), p0, p1);
          p0 = fast_exp2(p0);
          p1 = fast_exp2(p1);
          sum[r] = fadd2(sum[r], pack_f2(p0, p1));
          const uint32_t w = pack2<T>(p0, p1);
          const float2 f = unpack2<T>(w);
          hi[2 * t + r] = w;
          lo[2 * t + r] = pack2<T>(p0 - f.x, p1 - f.y);
        }
      const int vrow = warp * S::KW + (lane & 15);
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        uint32_t b[4];
        ldmatrix4t(b, smem_u32(stage) + S::V + slab_at<S::TK>(vrow, 2 * j + (lane >> 4)));
        mma16816<T>(acc[2 * j], hi, b[0], b[1]);
        mma16816<T>(acc[2 * j + 1], hi, b[2], b[3]);
        mma16816<T>(acc[2 * j], lo, b[0], b[1]);
        mma16816<T>(acc[2 * j + 1], lo, b[2], b[3]);
      }
    } else {
      uint64_t x[NT][2];                       // scores less shift, of two keys, of a row
      const uint64_t below[2] = {dup_f2(-shift[0]), dup_f2(-shift[1])};
#pragma unroll
      for (int t2 = 0; t2 < NT; t2 += 2) {
        uint32_t w[2][2 * S::G], sc[2][2][S::G];                         // words of the groups in turn; of this lane's two keys: step, value of code 0
        float d[2][S::G][4];
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          const int at = warp * S::KW + (t2 + v) * 8;
          if constexpr (D == 128) {
            const uint4 f = lds128(stage + (at + key_of(lane / 4)) * S::ROW + c * 16), f2 = lds128(stage + S::KS + (at + 2 * c) * S::SC);
            w[v][0] = f.x, w[v][1] = f.y, w[v][2] = f.z, w[v][3] = f.w;
            sc[v][0][0] = f2.x, sc[v][0][1] = f2.y, sc[v][1][0] = f2.z, sc[v][1][1] = f2.w;
          } else {
            const uint2 f = lds64(stage + (at + key_of(lane / 4)) * S::ROW + c * 8), f2 = lds64(stage + S::KS + (at + 2 * c) * S::SC);
            w[v][0] = f.x, w[v][1] = f.y;
            sc[v][0][0] = f2.x, sc[v][1][0] = f2.y;
          }
#pragma unroll
          for (int g = 0; g < S::G; ++g)
#pragma unroll
            for (int e = 0; e < 4; ++e) d[v][g][e] = 0.f;
        }
        // (the products of one sum a few others apart)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int x8 = 0; x8 < 2; ++x8)
#pragma unroll
            for (int v = 0; v < 2; ++v)
#pragma unroll
              for (int g = 0; g < S::G; ++g) {
                const uint32_t a = w[v][u * S::G + g] >> (8 * x8);
                mma16816<__half>(d[v][g], qf[(g * 2 + u) * 2 + x8], a & 0x000f000fu, a & 0x00f000f0u);
              }
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          uint64_t y[2], z[2] = {below[0], below[1]};
#pragma unroll
          for (int g = 0; g < S::G; ++g) {
            const float2 f0 = unpack2<__half>(sc[v][0][g]), f1 = unpack2<__half>(sc[v][1][g]);
            const uint64_t step = pack_f2(f0.x, f1.x), zero = pack_f2(f0.y, f1.y);
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const uint64_t dd = pack_f2(d[v][g][2 * r], d[v][g][2 * r + 1]);
              y[r] = g == 0 ? fmul2(step, dd) : ffma2(step, dd, y[r]);
              z[r] = ffma2(zero, dup_f2(q_sum[g][r]), z[r]);
            }
          }
#pragma unroll
          for (int r = 0; r < 2; ++r) x[t2 + v][r] = ffma2(y[r], dup_f2(q_unit[r]), z[r]);
        }
      }
      if (left < S::KW) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float x0, x1;
            unpack_f2(x[t][r], x0, x1);
            x[t][r] = pack_f2(t * 8 + c < left ? x0 : -INFINITY, t * 8 + c + 4 < left ? x1 : -INFINITY);
          }
      }
      float top[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float x0, x1;
        unpack_f2(x[0][r], x0, x1);
        top[r] = fmaxf(x0, x1);
#pragma unroll
        for (int t = 1; t < NT; ++t) {
          unpack_f2(x[t][r], x0, x1);
          top[r] = fmax3(top[r], x0, x1);
        }
      }
      uint32_t vsc[NT][2][S::G];
      __half2 most = __half2half2(__ushort_as_half(0));
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int at = warp * S::KW + t * 8 + 2 * c;
        if constexpr (D == 128) {
          const uint4 v = lds128(stage + S::VS + at * S::SC);
          vsc[t][0][0] = v.x, vsc[t][0][1] = v.y, vsc[t][1][0] = v.z, vsc[t][1][1] = v.w;
        } else {
          const uint2 v = lds64(stage + S::VS + at * S::SC);
          vsc[t][0][0] = v.x, vsc[t][1][0] = v.y;
        }
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int g = 0; g < S::G; ++g) most = __hmax2(most, *reinterpret_cast<const __half2*>(&vsc[t][e][g]));
      }
      const float v_top = __low2float(most);
      // (score > ref, as scores less shift; a row without scores has ref -inf and shift 0)
      const bool grew = top[0] + shift[0] > ref[0] || top[1] + shift[1] > ref[1] || v_top >= __uint_as_float((uint32_t)((int)v_exp + 127) << 23);
      if (__any_sync(0xffffffffu, grew)) {
        const float old[2] = {shift[0], shift[1]};
        top[0] += old[0];
        top[1] += old[1];
        raise(top, v_top, scale_log2);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int r = 0; r < 2; ++r) x[t][r] = fadd2(x[t][r], dup_f2(old[r] - shift[r]));
      }
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float p0, p1;
          unpack_f2(x[t][r], p0, p1);
          x[t][r] = pack_f2(fast_exp2(p0), fast_exp2(p1));
          sum[r] = fadd2(sum[r], x[t][r]);
        }
#pragma unroll
      for (int u = 0; u < NT / 2; ++u) {
        // Weight times step, rounded to fp16.  What the middle code stands for is added in 32 bits, and the rounded weights are summed up by the
        // same products, so that a rounding meets (code - 7.5) and not the code.  Keys of odd columns enter as 15 - code with the weight's sign
        // turned: the sums stay near the middle, where tensor cores, which cut sums off instead of rounding them, lose nothing that counts
        // (262144 keys, fp16 output: error 1.3e-3 with plain codes).
        uint32_t p[S::G][4];
#pragma unroll
        for (int g = 0; g < S::G; ++g)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int t = 2 * u + h;
            const float2 f0 = unpack2<__half>(vsc[t][0][g]), f1 = unpack2<__half>(vsc[t][1][g]);
            const uint64_t step = pack_f2(f0.x, -f1.x), mid = ffma2(step, pack_f2(7.5f, -7.5f), pack_f2(f0.y, f1.y));
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              float a, b;
              unpack_f2(fmul2(x[t][r], step), a, b);
              p[g][2 * h + r] = pack2<__half>(a, b);
              offset[g][r] = ffma2(x[t][r], mid, offset[g][r]);
            }
          }
        uint32_t w[4][S::G];                                             // keys c, c + 4 of the first eight, of the second
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const int key = warp * S::KW + u * 16 + (y >> 1) * 8 + c + 4 * (y & 1);
          if constexpr (D == 128) {
            const uint2 v = lds64(stage + S::V + key * S::ROW + (lane >> 2) * 8);
            w[y][0] = v.x, w[y][1] = v.y;
          } else {
            w[y][0] = lds32(stage + S::V + key * S::ROW + (lane >> 2) * 4);
          }
        }
#pragma unroll
        for (int g = 0; g < S::G; ++g) {
          mma16816<__half>(weight[g], p[g], 0x3c003c00u, 0x3c003c00u);
#pragma unroll
          for (int h = 0; h < 2; ++h) {                                  // elements 0 - 3, 4 - 7 of the words
            const uint32_t sel = h ? 0x7632u : 0x5410u;
            const uint32_t a = __byte_perm(w[0][g], w[1][g], sel), b = __byte_perm(w[2][g], w[3][g], sel), a8 = a >> 8, b8 = b >> 8;
            constexpr uint32_t M0 = 0x000f000fu, M1 = 0x00f000f0u, X0 = 0x000f0000u, X1 = 0x00f00000u;
            float(*o)[4] = acc + g * 8 + h * 4;
            mma16816<__half>(o[0], p[g], (a & M0) ^ X0, (b & M0) ^ X0);
            mma16816<__half>(o[1], p[g], (a & M1) ^ X1, (b & M1) ^ X1);
            mma16816<__half>(o[2], p[g], (a8 & M0) ^ X0, (b8 & M0) ^ X0);
            mma16816<__half>(o[3], p[g], (a8 & M1) ^ X1, (b8 & M1) ^ X1);
          }
        }
      }
    }
  }

  // The lane's partial sums become the row's.
  __device__ __forceinline__ float finish(int r) {
    float a, b;
    unpack_f2(sum[r], a, b);
    if constexpr (BITS == 4) {
#pragma unroll
      for (int g = 0; g < S::G; ++g) {
        float u, v;
        unpack_f2(offset[g][r], u, v);
        offset[g][r] = pack_f2(quad_sum(u + v), 0.f);
      }
    }
    return quad_sum(a + b);
  }

  // This warp's sums of columns [round * D / ROUNDS ..) in the stage, rows of D / ROUNDS floats; columns of 8 turned by the row.
  __device__ __forceinline__ void put(float* to, int round) {
    const int lane = threadIdx.x & 31, c = lane & 3;
    constexpr int W = D / S::ROUNDS;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int row = lane / 4 + 8 * half, turn = (row & 3) << 3;
      float* line = to + row * W;
      if constexpr (BITS == 16) {
#pragma unroll
        for (int j = 0; j < D / 8; ++j) *reinterpret_cast<float2*>(line + ((j * 8 + 2 * c) ^ turn)) = make_float2(acc[j][2 * half], acc[j][2 * half + 1]);
      } else {
        // column 2c of fragment j is element 16 c + j of the group, column 2c + 1 element 16 c + 8 + j
#pragma unroll
        for (int g = 0; g < S::G; ++g) {
          if (S::G == S::ROUNDS && g != round) continue;
          float mid, none;
          unpack_f2(offset[g][half], mid, none);
          mid = fmaf(-7.5f, weight[g][2 * half], mid);
#pragma unroll
          for (int j = 0; j < 8; j += 2)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int col = 16 * c + 8 * e + j;
              if (S::G != S::ROUNDS && col / W != round) continue;
              *reinterpret_cast<float2*>(line + ((col % W) ^ turn)) =
                  make_float2(fmaf(acc[g * 8 + j][2 * half + e], 16777216.f, mid), fmaf(acc[g * 8 + j + 1][2 * half + e], 1048576.f, mid));
            }
        }
      }
    }
  }
};

// The warp that fetches: tiles begin .. end - 1 into the ring.  full[s]: every lane arrives once its copies are there; empty[s]: the four warps that compute.
template <int D, int BITS>
__device__ __forceinline__ void fetch_tiles(const AttnArgs& a, const CUtensorMap* km, const CUtensorMap* vm, const int* first, const int* keys, Walk at,
                                            int begin, int end, int items, uint32_t base, uint32_t bars, int* abort_flag) {
  using S = Stage<D, BITS>;
  constexpr int NS = S::NS, TK = S::TK;
  const int lane = threadIdx.x & 31, run = 1 << a.run_log2;
  // page and slot of the run `r` of a tile; page -1: no key there, or no page
  auto look_up = [&](const Walk& w, int r, int& slot) {
    slot = 0;
    const int key = w.tile * TK + (r << a.run_log2);
    if (w.line >= a.lines || (r << a.run_log2) >= TK || key >= keys[w.line]) return -1;
    return paged_slot(a.c, a.by_n(a.line0 + w.line), key, slot);
  };
  int slot, page = look_up(at, lane, slot);
  int s = 0;
  uint32_t round = 0;
  for (int it = begin; it < end; ++it) {
    const uint32_t full = bars + 8 * s, empty = bars + 8 * (NS + s), dst = base + s * S::BYTES;
    if (round > 0 && !mbar_wait_or_abort(empty, (round - 1) & 1, abort_flag)) break;
    Walk next = at;
    next.step(first, a.lines, items);
    if (it + 1 == end) next.line = a.lines;
    int next_slot;
    const int next_page = look_up(next, lane, next_slot);              // (under way while this tile's copies are started)
    const int b = a.by_n(a.line0 + at.line), i = a.line0 + at.line - b * a.n;
    const int h = a.by_blocks(at.item), left = keys[at.line] - at.tile * TK;
    for (int r0 = 0; (r0 << a.run_log2) < min(TK, left); r0 += 32) {
      if (r0 > 0) page = look_up(at, r0 + lane, slot);                 // (runs of less than TK / 32 rows)
      const int row = (r0 + lane) << a.run_log2;
      if (page >= 0) {
        if constexpr (BITS == 16) {
          mbar_add_tx(full, 2 * S::ROW << a.run_log2);
#pragma unroll
          for (int x = 0; x < D / 64; ++x) {
            tma_tile(dst + x * TK * 128 + row * 128, km, 64 * x, slot, h, page, full);
            tma_tile(dst + S::V + x * TK * 128 + row * 128, vm, 64 * x, slot, h, page, full);
          }
        } else {
          const int64_t off = page * a.c.sp + h * a.c.sh + slot * a.c.st;
          const int rows = min(run, left - row);
          mbar_add_tx(full, 2 * S::ROW * rows);
          if (a.c.st == S::ROW) {
            bulk_copy(dst + row * S::ROW, a.c.k + off, rows * S::ROW, full);
            bulk_copy(dst + S::V + row * S::ROW, a.c.v + off, rows * S::ROW, full);
          } else {
            for (int y = 0; y < rows; ++y) {
              bulk_copy(dst + (row + y) * S::ROW, a.c.k + off + y * a.c.st, S::ROW, full);
              bulk_copy(dst + S::V + (row + y) * S::ROW, a.c.v + off + y * a.c.st, S::ROW, full);
            }
          }
        }
      }
      if constexpr (BITS == 4) {
        // scales of the rows of these 32 runs, a lane a row
        const int rows = min(32 << a.run_log2, TK);
        for (int y = lane; y < rows; y += 32) {
          const int q = y >> a.run_log2;
          const int pg = __shfl_sync(0xffffffffu, page, q), sl = __shfl_sync(0xffffffffu, slot, q) + (y & (run - 1));
          const int to = column_of((r0 << a.run_log2) + y);
          const int64_t off = pg >= 0 ? pg * a.c.ssp + h * a.c.ssh + sl * a.c.sst : 0;
          const uint32_t bytes = pg >= 0 ? S::SC : 0;
          cp_async_small<S::SC>(dst + S::KS + to * S::SC, a.c.ks + off, bytes);
          cp_async_small<S::SC>(dst + S::VS + to * S::SC, a.c.vs + off, bytes);
        }
      }
    }
    if (it == begin || at.tile == 0) {
      const int block = at.item - h * a.blocks, rows = min(a.group - block * ITEM_ROWS, ITEM_ROWS);
      const uint8_t* q = a.q + b * a.q_sb + i * a.q_sn + (int64_t)(h * a.group + block * ITEM_ROWS) * a.q_sh;
      constexpr int C = 2 * D / 16;
#pragma unroll
      for (int e = lane; e < ITEM_ROWS * C; e += 32) {
        const int r = e / C, chunk = e % C;
        cp_async16(dst + S::Q + r * 2 * D + chunk_at(r, chunk) * 16, q + (r < rows ? r : 0) * a.q_sh + chunk * 16, r < rows ? 16 : 0);
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

template <typename T, int D, int BITS>
__global__ void __launch_bounds__(THREADS, (Stage<D, BITS>::CTAS))
    paged_attn_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ CUtensorMap km, const __grid_constant__ CUtensorMap vm) {
  using S = Stage<D, BITS>;
  constexpr int NS = S::NS, TK = S::TK;
  extern __shared__ __align__(1024) uint8_t smem[];
  float2* stat = reinterpret_cast<float2*>(smem + NS * S::BYTES);            // [4][ITEM_ROWS]
  int* first = reinterpret_cast<int*>(stat + 4 * ITEM_ROWS);                 // [lines + 1] tiles before a line (of one item)
  int* keys = first + MAX_LINES + 4;                                         // [lines]
  const uint32_t base = smem_u32(smem), bars = smem_u32(keys + MAX_LINES);   // full[NS], empty[NS], join
  int* warp_sum = keys + MAX_LINES + 2 * S::BARS;                            // [4], abort flag in the last of ...
  int* abort_flag = first + MAX_LINES + 3;
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
  }
  chain_wait();

  // keys and tiles of every line: consecutive lines a thread
  {
    constexpr int PER = (MAX_LINES + 1 + 127) / 128;
    int before = 0, mine[PER];
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int line = tid * PER + u;
      int m = 0;
      if (line < a.lines) {
        const int b = a.by_n(a.line0 + line), i = a.line0 + line - b * a.n;
        const int count = a.c.counts ? min(a.c.counts[b], a.n) : a.n;
        int len = a.c.lengths[b];
        if (len > a.c.capacity) {
          report_status(a.c.status, a.c.status_host, HA_DEV_BAD_INDEX);
          len = a.c.capacity;
        }
        if (i < count) m = max(max(len, 0) - (count - 1 - i), 0);
        keys[line] = m;
      }
      mine[u] = before;
      before += (m + TK - 1) / TK;
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
  const int total = first[a.lines] * items;
  const int per = max((total + (int)gridDim.x - 1) / (int)gridDim.x, 1);
  const int begin = min((int)blockIdx.x * per, total), end = min(begin + per, total);
  if (blockIdx.x == 0 && tid == 0) {
    a.meta[0] = total;
    a.meta[1] = per;
  }
  // rows without keys
  for (int line = blockIdx.x; line < a.lines; line += gridDim.x) {
    if (keys[line] > 0) continue;
    const int b = a.by_n(a.line0 + line), i = a.line0 + line - b * a.n;
    uint4* o = reinterpret_cast<uint4*>((T*)a.o + (int64_t)(a.line0 + line) * a.H * D);
    for (int e = tid; e < a.H * D / 8; e += THREADS) o[e] = make_uint4(0, 0, 0, 0);
    for (int h = tid; h < a.H; h += THREADS) a.lse[((int64_t)b * a.H + h) * a.n + i] = -INFINITY;
  }
  if (begin >= end) return;

  Walk at;
  {
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
  }
  if (warp == 4) {
    fetch_tiles<D, BITS>(a, &km, &vm, first, keys, at, begin, end, items, base, bars, abort_flag);
    return;
  }

  Worker<T, D, BITS> w;
  const uint32_t join_bar = bars + 8 * 2 * NS;
  uint32_t joined = 0;
  // all four warps are here, and what they wrote to shared memory is visible
  auto join = [&]() {
    __syncwarp();
    if (lane == 0) mbar_arrive(join_bar);
    return mbar_wait_or_abort(join_bar, joined++ & 1, abort_flag);
  };
  int s = 0;
  uint32_t round = 0;
  bool ok = true;
#pragma unroll 1
  for (int it = begin; it < end && ok; ++it) {
    uint8_t* stage = smem + s * S::BYTES;
    ok = mbar_wait_or_abort(bars + 8 * s, round & 1, abort_flag);
    if (!ok) break;
    if (it == begin || at.tile == 0) w.begin(stage, a);
    const int left = keys[at.line] - at.tile * TK - warp * S::KW;
    if (left < S::KW) w.clear_tail(stage, left);
    w.tile(stage, left, a.scale_log2);
    const bool ends = at.tile == at.tiles - 1 || it == end - 1;
    if (ends) {
      // The item ends, or this CTA's part of it: the warps' sums are joined.
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float l = w.finish(r);
        // a warp without keys has no part; one whose scores are all NaN has
        if ((lane & 3) == 0) stat[warp * ITEM_ROWS + lane / 4 + 8 * r] = make_float2(w.ref[r] == -INFINITY && l == 0.f ? -INFINITY : w.shift[r], l);
      }
      const int b = a.by_n(a.line0 + at.line), i = a.line0 + at.line - b * a.n;
      const int h = a.by_blocks(at.item), block = at.item - h * a.blocks, rows = min(a.group - block * ITEM_ROWS, ITEM_ROWS);
      const int item_begin = first[at.line] * items + at.item * at.tiles, item_end = item_begin + at.tiles;
      const bool whole = item_begin >= begin && item_end <= end;
      const int row = tid >> 3;
      constexpr int W = D / S::ROUNDS;
      float* sums = reinterpret_cast<float*>(stage);
      float part[4], m = -INFINITY, l = 0.f;
#pragma unroll
      for (int y = 0; y < S::ROUNDS && ok; ++y) {
        ok = join();                           // the stage has been read (the round before, too); the statistics are there
        if (!ok) break;
        w.put(sums + warp * ITEM_ROWS * W, y);
        if (y == 0) {
#pragma unroll
          for (int x = 0; x < 4; ++x) m = fmaxf(m, stat[x * ITEM_ROWS + row].x);
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const float2 st = stat[x * ITEM_ROWS + row];
            part[x] = st.x == -INFINITY ? -1.f : fast_exp2(st.x - m);
            if (!(part[x] < 0.f)) l = fmaf(part[x], st.y, l);
          }
        }
        ok = join();
        if (!ok) break;
        const float inv = whole ? 1.f / l : 1.f;
        const int64_t out = ((int64_t)(a.line0 + at.line) * a.H + h * a.group + block * ITEM_ROWS + row) * D;
        const int slot = 2 * blockIdx.x + (item_begin <= begin ? 0 : 1);
#pragma unroll
        for (int j = 0; j < W / 32; ++j) {
          const int col = (tid & 7) * 4 + 32 * j;
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const float4 f = *reinterpret_cast<const float4*>(sums + (x * ITEM_ROWS + row) * W + (col ^ ((row & 3) << 3)));
            if (!(part[x] < 0.f)) {
              v.x = fmaf(part[x], f.x, v.x);
              v.y = fmaf(part[x], f.y, v.y);
              v.z = fmaf(part[x], f.z, v.z);
              v.w = fmaf(part[x], f.w, v.w);
            }
          }
          if (row < rows) {
            if (whole)
              *reinterpret_cast<uint2*>((T*)a.o + out + y * W + col) = make_uint2(pack2<T>(v.x * inv, v.y * inv), pack2<T>(v.z * inv, v.w * inv));
            else
              *reinterpret_cast<float4*>(a.part + ((int64_t)slot * ITEM_ROWS + row) * D + y * W + col) = v;
          }
        }
        if (y == 0 && row < rows && (tid & 7) == 0) {
          if (whole) a.lse[((int64_t)b * a.H + h * a.group + block * ITEM_ROWS + row) * a.n + i] = (m + log2f(l)) * LN2;
          else a.part_stat[slot * ITEM_ROWS + row] = make_float2(m, l);
        }
      }
      if (it == end - 1 && tid == 0) a.head[blockIdx.x] = make_int4(item_begin, item_end, a.line0 + at.line, at.item);
    }
    // the stage is free (what was written to it by stores before what copies write to it next)
    if (ends || left < S::KW) fence_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(bars + 8 * (NS + s));
    at.step(first, a.lines, items);
    if (++s == NS) s = 0, ++round;
  }
  if (!ok && lane == 0) report_timeout(a.c.status, a.c.status_host);
  chain_release();
}

// Joins the parts of the items that cross from one CTA's list to the next.  Block (c, row): the item that begins in CTA c's list and ends behind it.
template <typename T, int D>
__global__ void __launch_bounds__(128) paged_combine_kernel(const AttnArgs a) {
  __shared__ float red[4][D];
  __shared__ float red_m[4], red_l[4];
  chain_wait();
  const int c = blockIdx.x, row = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int total = a.meta[0], per = a.meta[1];
  if ((int64_t)(c + 1) * per >= total) return;
  const int4 hd = a.head[c];
  if (hd.y <= (c + 1) * per || hd.x < c * per) return;                 // ends here, or began before
  const int h = a.by_blocks(hd.w), block = hd.w - h * a.blocks, rows = min(a.group - block * ITEM_ROWS, ITEM_ROWS);
  if (row >= rows) return;
  const int last = (hd.y - 1) / per, pieces = last - c + 1;
  auto slot = [&](int p) { return 2 * (c + p) + (p == 0 && hd.x > c * per ? 1 : 0); };
  float m = -INFINITY;
  for (int p = tid; p < pieces; p += 128) m = fmaxf(m, a.part_stat[slot(p) * ITEM_ROWS + row].x);
#pragma unroll
  for (int s = 1; s < 32; s *= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, s));
  if (lane == 0) red_m[warp] = m;
  __syncthreads();
  m = fmaxf(fmaxf(red_m[0], red_m[1]), fmaxf(red_m[2], red_m[3]));
  // pieces p = warp, warp + 4, ...: a lane D / 32 columns
  constexpr int E = D / 32;
  float v[E], l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) v[e] = 0.f;
#pragma unroll 8
  for (int p = warp; p < pieces; p += 4) {
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
    if (st.x != -INFINITY) {
      const float w = fast_exp2(st.x - m);
      l = fmaf(w, st.y, l);
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = fmaf(w, y[e], v[e]);
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e) red[warp][lane * E + e] = v[e];
  if (lane == 0) red_l[warp] = l;
  __syncthreads();
  l = (red_l[0] + red_l[1]) + (red_l[2] + red_l[3]);
  const int head = h * a.group + block * ITEM_ROWS + row;
  const int b = a.by_n(hd.z), i = hd.z - b * a.n;
  if (tid < D) ((T*)a.o)[((int64_t)hd.z * a.H + head) * D + tid] = from_f32<T>(((red[0][tid] + red[1][tid]) + (red[2][tid] + red[3][tid])) / l);
  if (tid == 0) a.lse[((int64_t)b * a.H + head) * a.n + i] = (m + log2f(l)) * LN2;
}

int attn_tile(const ha_paged_params& p) { return p.bits == 16 ? 64 : 128; }
int attn_resident(const ha_paged_params& p) {
  if (p.bits == 16) return p.d == 128 ? Stage<128, 16>::CTAS : Stage<64, 16>::CTAS;
  return p.d == 128 ? Stage<128, 4>::CTAS : Stage<64, 4>::CTAS;
}

// CTAs of a launch over `lines` lines: as many as are resident at once, and no more than there can be tiles.
int attn_ctas(const ha_paged_params& p, int lines) {
  const int tk = attn_tile(p), items = p.Hk * ((p.H / p.Hk + ITEM_ROWS - 1) / ITEM_ROWS);
  const int64_t most = ((int64_t)p.columns * p.page_size + tk - 1) / tk * items * lines;
  const int resident = sm_count() * attn_resident(p);
  return (int)(most < 1 ? 1 : most < resident ? most : resident);
}

// Lines of one launch: no more than shared memory counts, their tiles within 31 bits.
int64_t attn_lines(const ha_paged_params& p) {
  const int tk = attn_tile(p), items = p.Hk * ((p.H / p.Hk + ITEM_ROWS - 1) / ITEM_ROWS);
  const int64_t tiles = ((int64_t)p.columns * p.page_size + tk - 1) / tk * items, all = (int64_t)p.B * p.n;
  int64_t lines = all < MAX_LINES ? all : MAX_LINES;
  if (tiles > 0 && lines > (0x7fffffffLL - 65536) / tiles) lines = (0x7fffffffLL - 65536) / tiles;
  return lines;
}

// Tensor maps of K and V pages: boxes of as many rows as both a page and a tile are made of.
bool attn_maps(const ha_paged_params& p, CUtensorMap* maps) {
  if (p.pages == 0) return true;
  const int run = std::gcd(p.page_size, 64);
  const int64_t row = p.page_size == 1 ? p.d : p.page_st;
  return encode_tile_map(&maps[0], p.dtype, p.k_pages, p.d, p.page_size, p.Hk, p.pages, row, p.page_sh, p.page_sp, run) &&
         encode_tile_map(&maps[1], p.dtype, p.v_pages, p.d, p.page_size, p.Hk, p.pages, row, p.page_sh, p.page_sp, run);
}

int64_t attn_workspace(const ha_paged_params& p, int ctas) { return 256 + (int64_t)ctas * (16 + 2 * ITEM_ROWS * (p.d * 4 + 8)); }

template <typename T, int D, int BITS>
int launch_attn(AttnArgs a, const ha_paged_params& p, cudaStream_t st) {
  using S = Stage<D, BITS>;
  while ((1 << a.run_log2) < std::gcd(p.page_size, S::TK)) ++a.run_log2;
  CUtensorMap maps[2] = {};
  if (BITS == 16) {
    if (p.maps) memcpy(maps, p.maps, sizeof(maps));
    else if (!attn_maps(p, maps)) return HA_ERR_INVALID;
  }
  HA_SMEM_ATTR_ONCE((paged_attn_kernel<T, D, BITS>), S::SMEM, "ha_paged_attn");
  const int64_t all = (int64_t)p.B * p.n, most = attn_lines(p);
  for (int64_t line0 = 0; line0 < all; line0 += most) {
    a.line0 = (int)line0;
    a.lines = (int)(all - line0 < most ? all - line0 : most);
    const int ctas = attn_ctas(p, a.lines);
    launch_chained(paged_attn_kernel<T, D, BITS>, ctas, THREADS, S::SMEM, st, a, maps[0], maps[1]);
    HA_LAUNCHED("ha_paged_attn");
    if (ctas > 1) {
      launch_chained(paged_combine_kernel<T, D>, dim3(ctas - 1, a.group < ITEM_ROWS ? a.group : ITEM_ROWS), 128, 0, st, a);
      HA_LAUNCHED("ha_paged_attn");
    }
  }
  return HA_OK;
}

int attn_check(const ha_paged_params& p) {
  const int rc = paged_check(p);
  if (rc != HA_OK) return rc;
  if (p.H < 1 || p.scale == 0.f) return HA_ERR_INVALID;
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
  if ((int64_t)p.columns * p.page_size > 0x7fffffffLL) return HA_ERR_TOO_LARGE;
  const int64_t all = (int64_t)p.B * p.n, lines = attn_lines(p);
  if (all == 0) return 0;
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
  if (!p.workspace || (uintptr_t)p.workspace % 16 != 0 || p.workspace_bytes < attn_workspace(p, ctas)) return HA_ERR_WORKSPACE;
  AttnArgs a = {};
  a.c = paged_view(p);
  a.q = (const uint8_t*)p.q;
  a.q_sb = p.q_sb * 2; a.q_sn = p.q_sn * 2; a.q_sh = p.q_sh * 2;
  a.o = p.o; a.lse = p.lse;
  a.n = p.n; a.H = p.H; a.Hk = p.Hk; a.group = p.H / p.Hk; a.blocks = (a.group + ITEM_ROWS - 1) / ITEM_ROWS;
  a.by_n = FastDiv((uint32_t)p.n); a.by_blocks = FastDiv((uint32_t)a.blocks);
  a.scale_log2 = fabsf(p.scale) * LOG2E;
  a.flip = p.scale < 0.f ? 0x80008000u : 0u;
  uint8_t* ws = (uint8_t*)p.workspace;
  a.meta = (int32_t*)ws;
  a.head = (int4*)(ws + 256);
  a.part_stat = (float2*)(ws + 256 + (int64_t)ctas * 16);
  a.part = (float*)(ws + 256 + (int64_t)ctas * (16 + 2 * ITEM_ROWS * 8));
  const cudaStream_t st = (cudaStream_t)stream;
  if (p.dtype == HA_BF16) {
    if (p.d == 64) return p.bits == 16 ? launch_attn<__nv_bfloat16, 64, 16>(a, p, st) : launch_attn<__nv_bfloat16, 64, 4>(a, p, st);
    return p.bits == 16 ? launch_attn<__nv_bfloat16, 128, 16>(a, p, st) : launch_attn<__nv_bfloat16, 128, 4>(a, p, st);
  }
  if (p.d == 64) return p.bits == 16 ? launch_attn<__half, 64, 16>(a, p, st) : launch_attn<__half, 64, 4>(a, p, st);
  return p.bits == 16 ? launch_attn<__half, 128, 16>(a, p, st) : launch_attn<__half, 128, 4>(a, p, st);
}

}  // extern "C"
