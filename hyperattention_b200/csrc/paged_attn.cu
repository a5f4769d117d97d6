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
// A CTA of four warps; each warp takes a quarter of a tile's keys with its own running maximum and sums, which are joined at the item's end.  Tiles
// come by cp.async in a ring of NS stages, across items; queries come with the first tile of an item.
#include <type_traits>

#include "paged.cuh"

namespace ha {

namespace {

constexpr int ITEM_ROWS = 16;
constexpr int MAX_LINES = 416;        // (sequence, token) pairs of one launch: their tiles are summed up in shared memory
constexpr float LN2 = 0.693147180559945309f, LOG2E = 1.44269504088896341f;

struct AttnArgs {
  PagedView c;
  const uint8_t* q;
  int64_t q_sb, q_sn, q_sh;           // bytes
  void* o;
  float* lse;
  int32_t n, H, Hk, group, blocks;    // blocks: items of a (token, K/V head): group / 16, rounded up
  int32_t line0, lines;               // (sequence, token) pairs of this launch
  FastDiv by_n, by_blocks;
  float scale_log2;
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
  static constexpr int SC = BITS == 16 ? 0 : 4 * G;
  static constexpr int V = TK * ROW, KS = 2 * TK * ROW, VS = KS + TK * SC, Q = VS + TK * SC;
  static constexpr int BYTES = Q + ITEM_ROWS * 2 * D;
  static constexpr int NS = BITS == 16 ? (D == 128 ? 3 : 6) : (D == 128 ? 3 : 5);
  static constexpr int CTAS = BITS == 16 ? 2 : 3;
  static constexpr int RING = 2 * TK * (BITS == 16 ? 8 : 16);
  static constexpr int ROUNDS = BITS == 16 ? 1 : 2;          // in which the warps' sums are joined: column ranges that fit a stage
  static constexpr int SMEM = NS * BYTES + RING + 4 * ITEM_ROWS * 8 + (2 * MAX_LINES + 1) * 4 + 32;
  static_assert(4 * ITEM_ROWS * D / ROUNDS * 4 <= Q, "the warps' sums fit a stage");
  static_assert(CTAS * (SMEM + 1024) <= 228 * 1024, "CTAs of an SM");
};

template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_small(uint32_t dst, const void* src, uint32_t src_bytes) {      // 4 or 8 bytes
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(N), "r"(src_bytes) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}
// 16-byte chunk of a row in shared memory: the eight rows that one ldmatrix phase (or one quarter of a 128-bit load) touches lie in different banks
__device__ __forceinline__ int chunk_at(int row, int chunk) { return chunk ^ (row & 7); }
// 4-bit rows of 64 bytes: K lies in the order in which the score columns name keys (column 2c + e is key c + 4e of its eight), V in key order, its 16-byte
// chunks turned so that the four keys c .. of one 64-bit load fill all banks
__device__ __forceinline__ int column_of(int key) { return (key & ~7) | ((key & 3) << 1) | ((key >> 2) & 1); }
template <int D> __device__ __forceinline__ int v4_chunk(int key, int chunk) { return D == 128 ? chunk ^ (((key >> 1) & 1) << 1) : chunk; }

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
  static constexpr float BIAS = 15.f;         // (fp16 weights) of the reference: weights up to 2^15, normal down to 2^-29 of the largest

  // of rows lane / 4 and lane / 4 + 8
  float ref[2], sum[2];
  float acc[D / 8][4];
  uint32_t qf[D / 16][4];
  // 4-bit rows
  float q_unit[2], q_sum[S::G][2];            // score of a code sum; sum of the row's elements of a group, times the softmax scale
  float weight[S::G][4];                      // sums of the rounded weights (every column alike)
  float offset[S::G][2];                      // sum of weights times what a row's middle code stands for
  float v_exp;                                // power of two that no V step so far exceeds

  __device__ __forceinline__ void begin(uint32_t stage, float scale_log2) {
    const int lane = threadIdx.x & 31;
    ref[0] = ref[1] = -INFINITY;
    sum[0] = sum[1] = 0.f;
#pragma unroll
    for (int j = 0; j < D / 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[j][e] = 0.f;
    const uint32_t q = stage + S::Q;
    if constexpr (BITS == 16) {
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        const int row = lane & 15;
        ldmatrix4(qf[ks], q + row * 2 * D + chunk_at(row, 2 * ks + (lane >> 4)) * 16);
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
            const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float2 f = unpack2<T>(ws[j]);
              x[g][8 * u + 2 * j] = f.x;
              x[g][8 * u + 2 * j + 1] = f.y;
              s += f.x + f.y;
              top = max_nan(top, max_nan(fabsf(f.x), fabsf(f.y)));
            }
          }
          q_sum[g][half] = quad_sum(s) * scale_log2;
          weight[g][2 * half] = weight[g][2 * half + 1] = 0.f;
          offset[g][half] = 0.f;
        }
        top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // exponent of the largest element; a row of zeros stays one, one with a NaN or an infinity keeps it through the products
        const int e = max((int)(__float_as_uint(top) >> 23) & 255, 27);
        const float up = __uint_as_float((uint32_t)(127 + 13 + 127 - e) << 23), down = __uint_as_float((uint32_t)(e - 13) << 23);
        // codes are the subnormal fp16 numbers code * 2^-24 (or * 2^-20, against a sixteenth of the query's element)
        q_unit[half] = down * 16777216.f * scale_log2;
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

  // new reference of the rows whose maximum grew; the sums so far follow
  __device__ __forceinline__ void raise(const float (&top)[2], float v_top) {
    float by[2];
    float exp_new = 0.f, exp_old = 0.f;
    if constexpr (BITS == 4) {
      exp_old = v_exp;
#pragma unroll
      for (int s = 1; s < 32; s *= 2) v_top = fmaxf(v_top, __shfl_xor_sync(0xffffffffu, v_top, s));
      v_exp = fmaxf(v_exp, (float)((int)(__float_as_uint(v_top) >> 23) - 126));
      exp_new = v_exp;
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const float now = fmaxf(ref[r], quad_max(top[r]));
      by[r] = now == -INFINITY ? 1.f : fast_exp2((ref[r] - now) + (exp_old - exp_new));
      ref[r] = now;
      sum[r] *= by[r];
    }
#pragma unroll
    for (int j = 0; j < D / 8; ++j) {
      acc[j][0] *= by[0];
      acc[j][1] *= by[0];
      acc[j][2] *= by[1];
      acc[j][3] *= by[1];
    }
    if constexpr (BITS == 4) {
#pragma unroll
      for (int g = 0; g < S::G; ++g) {
        weight[g][0] *= by[0];
        weight[g][2] *= by[1];
        offset[g][0] *= by[0];
        offset[g][1] *= by[1];
      }
    }
  }
  // what is taken off a score's exponent: weights are exp2(x - shift)
  __device__ __forceinline__ float shift(int r) const {
    if (ref[r] == -INFINITY) return 0.f;
    if constexpr (BITS == 4) return ref[r] + v_exp - BIAS;
    else return std::is_same<T, __half>::value ? ref[r] - BIAS : ref[r];
  }

  // One tile: this warp's keys are left .. left + KW - 1 (of the row's `left` that are still to come, counted from this warp's first).
  __device__ __forceinline__ void tile(uint32_t stage, int left, float scale_log2) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = lane & 3;
    float x[NT][4];
    if constexpr (BITS == 16) {
      const int row = warp * 16 + (lane & 7) + ((lane >> 4) << 3);
      const uint32_t k = stage + row * S::ROW;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[t][e] = 0.f;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        uint32_t b[4];
        ldmatrix4(b, k + chunk_at(row, 2 * ks + ((lane >> 3) & 1)) * 16);
        mma16816<T>(x[0], qf[ks], b[0], b[1]);
        mma16816<T>(x[1], qf[ks], b[2], b[3]);
      }
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[t][e] *= scale_log2;
          if (left < S::KW && t * 8 + 2 * c + (e & 1) >= left) x[t][e] = -INFINITY;
        }
    } else {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int at = warp * 32 + t * 8;
        uint32_t w[4];
        if constexpr (D == 128) {
          const uint4 v = lds128(stage + (at + lane / 4) * S::ROW + c * 16);
          w[0] = v.x, w[1] = v.z, w[2] = v.y, w[3] = v.w;                // words of the first group, of the second
        } else {
          const uint2 v = lds64(stage + (at + lane / 4) * S::ROW + c * 8);
          w[0] = v.x, w[1] = v.y;
        }
        float d[S::G][4];
#pragma unroll
        for (int g = 0; g < S::G; ++g) {
#pragma unroll
          for (int e = 0; e < 4; ++e) d[g][e] = 0.f;
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const uint32_t a = w[2 * g + u], b = a >> 8;
            mma16816<__half>(d[g], qf[(g * 2 + u) * 2], a & 0x000f000fu, a & 0x00f000f0u);
            mma16816<__half>(d[g], qf[(g * 2 + u) * 2 + 1], b & 0x000f000fu, b & 0x00f000f0u);
          }
        }
        uint32_t sc[2][S::G];                                            // of this lane's two keys
        if constexpr (D == 128) {
          const uint4 v = lds128(stage + S::KS + (at + 2 * c) * S::SC);
          sc[0][0] = v.x, sc[0][1] = v.y, sc[1][0] = v.z, sc[1][1] = v.w;
        } else {
          const uint2 v = lds64(stage + S::KS + (at + 2 * c) * S::SC);
          sc[0][0] = v.x, sc[1][0] = v.y;
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float y[2] = {0.f, 0.f}, z[2] = {0.f, 0.f};
#pragma unroll
          for (int g = 0; g < S::G; ++g) {
            const float2 f = unpack2<__half>(sc[e][g]);                  // step, value of code 0
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              y[r] = g == 0 ? f.x * d[g][2 * r + e] : fmaf(f.x, d[g][2 * r + e], y[r]);
              z[r] = g == 0 ? f.y * q_sum[g][r] : fmaf(f.y, q_sum[g][r], z[r]);
            }
          }
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            x[t][2 * r + e] = fmaf(y[r], q_unit[r], z[r]);
            if (left < S::KW && t * 8 + c + 4 * e >= left) x[t][2 * r + e] = -INFINITY;
          }
        }
      }
    }

    float top[2] = {fmaxf(x[0][0], x[0][1]), fmaxf(x[0][2], x[0][3])};
#pragma unroll
    for (int t = 1; t < NT; ++t) {
      top[0] = fmax3(top[0], x[t][0], x[t][1]);
      top[1] = fmax3(top[1], x[t][2], x[t][3]);
    }
    uint32_t vsc[NT][2][S::G];
    float v_top = 0.f;
    bool grew = top[0] > ref[0] || top[1] > ref[1];
    if constexpr (BITS == 4) {
      __half2 most = __half2half2(__ushort_as_half(0));
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int at = warp * 32 + t * 8 + 2 * c;
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
      v_top = __low2float(most);
      grew = grew || v_top >= exp2f_int(v_exp);
    }
    if (__any_sync(0xffffffffu, grew)) raise(top, v_top);
    const float sh[2] = {shift(0), shift(1)};
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[t][e] = fast_exp2(x[t][e] - sh[e >> 1]);
        sum[e >> 1] += x[t][e];
      }

    if constexpr (BITS == 16) {
      // Weights as the sum of two numbers of T: the second holds what the first rounds off, so that the output's own rounding is the one that
      // counts.  The products are far from the bound (a second one costs nothing that the loads do not hide).
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const uint32_t w = pack2<T>(x[t][2 * r], x[t][2 * r + 1]);
          const float2 f = unpack2<T>(w);
          hi[2 * t + r] = w;
          lo[2 * t + r] = pack2<T>(x[t][2 * r] - f.x, x[t][2 * r + 1] - f.y);
        }
      const int row = warp * 16 + (lane & 15);
      const uint32_t v = stage + S::V + row * S::ROW;
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        uint32_t b[4];
        ldmatrix4t(b, v + chunk_at(row, 2 * j + (lane >> 4)) * 16);
        mma16816<T>(acc[2 * j], hi, b[0], b[1]);
        mma16816<T>(acc[2 * j + 1], hi, b[2], b[3]);
        mma16816<T>(acc[2 * j], lo, b[0], b[1]);
        mma16816<T>(acc[2 * j + 1], lo, b[2], b[3]);
      }
    } else {
#pragma unroll
      for (int u = 0; u < NT / 2; ++u) {
        // weight times step, rounded to fp16; what the middle code stands for is added in 32 bits, and the rounded weights are summed up by
        // the same products, so that a rounding meets (code - 7.5) and not the code
        uint32_t p[S::G][4];
#pragma unroll
        for (int g = 0; g < S::G; ++g)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int t = 2 * u + h;
            const float2 f0 = unpack2<__half>(vsc[t][0][g]), f1 = unpack2<__half>(vsc[t][1][g]);
            const float m0 = fmaf(7.5f, f0.x, f0.y), m1 = fmaf(7.5f, f1.x, f1.y);
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              p[g][2 * h + r] = pack2<__half>(x[t][2 * r] * f0.x, x[t][2 * r + 1] * f1.x);
              offset[g][r] = fmaf(x[t][2 * r], m0, fmaf(x[t][2 * r + 1], m1, offset[g][r]));
            }
          }
        uint32_t w[4][S::G];                                             // keys c, c + 4 of the first eight, of the second
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const int key = warp * 32 + u * 16 + (y >> 1) * 8 + c + 4 * (y & 1);
          if constexpr (D == 128) {
            const uint2 v = lds64(stage + S::V + key * S::ROW + v4_chunk<D>(key, lane >> 3) * 16 + ((lane >> 2) & 1) * 8);
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
            float(*o)[4] = acc + g * 8 + h * 4;
            mma16816<__half>(o[0], p[g], a & 0x000f000fu, b & 0x000f000fu);
            mma16816<__half>(o[1], p[g], a & 0x00f000f0u, b & 0x00f000f0u);
            mma16816<__half>(o[2], p[g], a8 & 0x000f000fu, b8 & 0x000f000fu);
            mma16816<__half>(o[3], p[g], a8 & 0x00f000f0u, b8 & 0x00f000f0u);
          }
        }
      }
    }
  }
  static __device__ __forceinline__ float exp2f_int(float e) { return __uint_as_float((uint32_t)((int)e + 127) << 23); }

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
          const float mid = offset[g][half] - 7.5f * weight[g][2 * half];
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

template <typename T, int D, int BITS>
__global__ void __launch_bounds__(128, Stage<D, BITS>::CTAS) paged_attn_kernel(const AttnArgs a) {
  using S = Stage<D, BITS>;
  constexpr int NS = S::NS, TK = S::TK;
  extern __shared__ __align__(128) uint8_t smem[];
  int64_t* ring = reinterpret_cast<int64_t*>(smem + NS * S::BYTES);          // [2][TK] offsets of rows, -1: none; 4 bits: [2][TK] of their scales, too
  float2* stat = reinterpret_cast<float2*>(smem + NS * S::BYTES + S::RING);  // [4][ITEM_ROWS]
  int* first = reinterpret_cast<int*>(stat + 4 * ITEM_ROWS);                 // [lines + 1] tiles before a line (of one item)
  int* keys = first + MAX_LINES + 1;                                         // [lines]
  int* warp_sum = keys + MAX_LINES;                                          // [4]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int items = a.Hk * a.blocks;
  chain_begin();

  // keys and tiles of every line: four consecutive lines a thread
  {
    constexpr int PER = (MAX_LINES + 127) / 128;
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
    for (int s = 1; s < 32; s *= 2) {
      const int v = __shfl_up_sync(0xffffffffu, incl, s);
      if (lane >= s) incl += v;
    }
    if (lane == 31) warp_sum[warp] = incl;
    __syncthreads();
    int base = incl - before;
    for (int w = 0; w < warp; ++w) base += warp_sum[w];
#pragma unroll
    for (int u = 0; u < PER; ++u)
      if (tid * PER + u <= a.lines) first[tid * PER + u] = base + mine[u];
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
    for (int e = tid; e < a.H * D / 8; e += 128) o[e] = make_uint4(0, 0, 0, 0);
    for (int h = tid; h < a.H; h += 128) a.lse[((int64_t)b * a.H + h) * a.n + i] = -INFINITY;
  }
  if (begin >= end) return;

  Walk at;                                     // tile that is computed
  {
    int lo = 0, hi = a.lines;                  // the last line whose tiles begin at or before `begin`
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (first[mid] * items <= begin) lo = mid;
      else hi = mid;
    }
    at.line = lo;
    at.settle(first, a.lines);                 // (lines without tiles share their first tile with the next one: the search may stop at such)
    const int off = begin - first[at.line] * items;
    at.item = off / at.tiles;
    at.tile = off - at.item * at.tiles;
  }
  Walk name = at, fetch = at;                  // tile whose rows are looked up next; tile that is fetched next
  int named = begin, fetched = begin;
  const uint32_t base = smem_u32(smem);

  // offset of the row that this thread looks up (every thread up to TK) of tile `name`
  auto look_up = [&](int64_t& off, int64_t& off_s) {
    off = off_s = -1;
    if (named < end && tid < TK) {
      const int key = name.tile * TK + tid;
      if (key < keys[name.line]) {
        const int b = a.by_n(a.line0 + name.line), h = a.by_blocks(name.item);
        int row;
        const int page = paged_slot(a.c, b, key, row);
        if (page >= 0) {
          off = page * a.c.sp + h * a.c.sh + row * a.c.st;
          if (BITS == 4) off_s = page * a.c.ssp + h * a.c.ssh + row * a.c.sst;
        }
      }
    }
  };
  auto keep = [&](int64_t off, int64_t off_s) {
    if (tid < TK) {
      ring[(named & 1) * TK + tid] = off;
      if (BITS == 4) ring[2 * TK + (named & 1) * TK + tid] = off_s;
    }
    if (named < end) name.step(first, a.lines, items);
    ++named;
  };
  auto issue = [&]() {
    if (fetched < end) {
      const uint32_t dst = base + ((fetched - begin) % NS) * S::BYTES;
      const int64_t* offs = ring + (fetched & 1) * TK;
      if constexpr (BITS == 16) {
        constexpr int C = S::ROW / 16, PASS = 128 / C;
        const int chunk = tid % C;
#pragma unroll
        for (int r = tid / C; r < TK; r += PASS) {
          const int64_t off = offs[r];
          const uint32_t bytes = off >= 0 ? 16 : 0, to = dst + r * S::ROW + chunk_at(r, chunk) * 16;
          const int64_t from = (off >= 0 ? off : 0) + chunk * 16;
          cp_async16(to, a.c.k + from, bytes);
          cp_async16(to + S::V, a.c.v + from, bytes);
        }
      } else {
        constexpr int C = S::ROW / 16, PASS = 128 / C;
        const int chunk = tid % C;
#pragma unroll
        for (int r = tid / C; r < TK; r += PASS) {
          const int64_t off = offs[r];
          const uint32_t bytes = off >= 0 ? 16 : 0;
          const int64_t from = (off >= 0 ? off : 0) + chunk * 16;
          cp_async16(dst + column_of(r) * S::ROW + chunk * 16, a.c.k + from, bytes);
          cp_async16(dst + S::V + r * S::ROW + v4_chunk<D>(r, chunk) * 16, a.c.v + from, bytes);
        }
        const int64_t off = offs[2 * TK + tid];
        const uint32_t bytes = off >= 0 ? S::SC : 0;
        const int64_t from = off >= 0 ? off : 0;
        cp_async_small<S::SC == 0 ? 4 : S::SC>(dst + S::KS + column_of(tid) * S::SC, a.c.ks + from, bytes);
        cp_async_small<S::SC == 0 ? 4 : S::SC>(dst + S::VS + column_of(tid) * S::SC, a.c.vs + from, bytes);
      }
      if (fetched == begin || fetch.tile == 0) {
        const int b = a.by_n(a.line0 + fetch.line), i = a.line0 + fetch.line - b * a.n;
        const int h = a.by_blocks(fetch.item), block = fetch.item - h * a.blocks, rows = min(a.group - block * ITEM_ROWS, ITEM_ROWS);
        const uint8_t* q = a.q + b * a.q_sb + i * a.q_sn + (int64_t)(h * a.group + block * ITEM_ROWS) * a.q_sh;
        constexpr int C = 2 * D / 16;
#pragma unroll
        for (int e = tid; e < ITEM_ROWS * C; e += 128) {
          const int r = e / C, chunk = e % C;
          cp_async16(dst + S::Q + r * 2 * D + chunk_at(r, chunk) * 16, q + (r < rows ? r : 0) * a.q_sh + chunk * 16, r < rows ? 16 : 0);
        }
      }
      fetch.step(first, a.lines, items);
    }
    cp_async_commit();
    ++fetched;
  };

  int64_t off, off_s;
#pragma unroll 1
  for (int s = 0; s < NS - 1; ++s) {
    look_up(off, off_s);
    keep(off, off_s);
    __syncthreads();
    issue();
  }
  look_up(off, off_s);
  keep(off, off_s);

  Worker<T, D, BITS> w;
#pragma unroll 1
  for (int it = begin; it < end; ++it) {
    cp_async_wait<NS - 2>();
    __syncthreads();                           // tile `it` is there, its predecessor's stage free, the rows of tile it + NS - 1 named
    issue();
    look_up(off, off_s);                       // (its load is under way during the tile)
    const uint32_t stage = base + ((it - begin) % NS) * S::BYTES;
    if (it == begin || at.tile == 0) w.begin(stage, a.scale_log2);
    w.tile(stage, keys[at.line] - at.tile * TK - warp * S::KW, a.scale_log2);
    if (at.tile == at.tiles - 1 || it == end - 1) {
      // The item ends, or this CTA's part of it: the warps' sums are joined.
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float l = quad_sum(w.sum[r]);
        if (BITS == 4)
#pragma unroll
          for (int g = 0; g < S::G; ++g) w.offset[g][r] = quad_sum(w.offset[g][r]);
        // a warp without keys has no part; one whose scores are all NaN has
        if ((lane & 3) == 0) stat[warp * ITEM_ROWS + lane / 4 + 8 * r] = make_float2(w.ref[r] == -INFINITY && l == 0.f ? -INFINITY : w.shift(r), l);
      }
      const int b = a.by_n(a.line0 + at.line), i = a.line0 + at.line - b * a.n;
      const int h = a.by_blocks(at.item), block = at.item - h * a.blocks, rows = min(a.group - block * ITEM_ROWS, ITEM_ROWS);
      const int item_begin = first[at.line] * items + at.item * at.tiles, item_end = item_begin + at.tiles;
      const bool whole = item_begin >= begin && item_end <= end;
      const int row = tid >> 3;
      constexpr int W = D / S::ROUNDS;
      float* sums = reinterpret_cast<float*>(smem + ((it - begin) % NS) * S::BYTES);
      float part[4], m = -INFINITY, l = 0.f;
#pragma unroll
      for (int round = 0; round < S::ROUNDS; ++round) {
        __syncthreads();                       // the stage has been read (the round before, too); the statistics are there
        w.put(sums + warp * ITEM_ROWS * W, round);
        if (round == 0) {
#pragma unroll
          for (int x = 0; x < 4; ++x) m = fmaxf(m, stat[x * ITEM_ROWS + row].x);
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const float2 st = stat[x * ITEM_ROWS + row];
            part[x] = st.x == -INFINITY ? -1.f : fast_exp2(st.x - m);
            if (!(part[x] < 0.f)) l = fmaf(part[x], st.y, l);
          }
        }
        __syncthreads();
        const float inv = whole ? 1.f / l : 1.f;
        const int64_t out = ((int64_t)(a.line0 + at.line) * a.H + h * a.group + block * ITEM_ROWS + row) * D;
        const int slot = 2 * blockIdx.x + (item_begin <= begin ? 0 : 1);
#pragma unroll
        for (int j = 0; j < W / 32; ++j) {
          const int col = (tid & 7) * 4 + 32 * j;
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const float4 y = *reinterpret_cast<const float4*>(sums + (x * ITEM_ROWS + row) * W + (col ^ ((row & 3) << 3)));
            if (!(part[x] < 0.f)) {
              v.x = fmaf(part[x], y.x, v.x);
              v.y = fmaf(part[x], y.y, v.y);
              v.z = fmaf(part[x], y.z, v.z);
              v.w = fmaf(part[x], y.w, v.w);
            }
          }
          if (row < rows) {
            if (whole)
              *reinterpret_cast<uint2*>((T*)a.o + out + round * W + col) = make_uint2(pack2<T>(v.x * inv, v.y * inv), pack2<T>(v.z * inv, v.w * inv));
            else
              *reinterpret_cast<float4*>(a.part + ((int64_t)slot * ITEM_ROWS + row) * D + round * W + col) = v;
          }
        }
        if (round == 0 && row < rows && (tid & 7) == 0) {
          if (whole) a.lse[((int64_t)b * a.H + h * a.group + block * ITEM_ROWS + row) * a.n + i] = (m + log2f(l)) * LN2;
          else a.part_stat[slot * ITEM_ROWS + row] = make_float2(m, l);
        }
      }
      if (it == end - 1 && tid == 0) a.head[blockIdx.x] = make_int4(item_begin, item_end, a.line0 + at.line, at.item);
    }
    keep(off, off_s);
    at.step(first, a.lines, items);
  }
  cp_async_wait<0>();
}

// Joins the parts of the items that cross from one CTA's list to the next.  Block (c, row): the item that begins in CTA c's list and ends behind it.
template <typename T, int D>
__global__ void __launch_bounds__(128) paged_combine_kernel(const AttnArgs a) {
  __shared__ float red[4][D];
  __shared__ float red_m[4], red_l[4];
  chain_begin();
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

// CTAs of a launch over `lines` lines: as many as are resident at once, and no more than there can be tiles.
int attn_ctas(const ha_paged_params& p, int lines) {
  const int tk = attn_tile(p), items = p.Hk * ((p.H / p.Hk + ITEM_ROWS - 1) / ITEM_ROWS);
  const int64_t most = ((int64_t)p.columns * p.page_size + tk - 1) / tk * items * lines;
  const int resident = sm_count() * (p.bits == 16 ? 2 : 3);
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

int64_t attn_workspace(const ha_paged_params& p, int ctas) { return 256 + (int64_t)ctas * (16 + 2 * ITEM_ROWS * (p.d * 4 + 8)); }

template <typename T, int D, int BITS>
int launch_attn(AttnArgs a, const ha_paged_params& p, cudaStream_t st) {
  using S = Stage<D, BITS>;
  HA_SMEM_ATTR_ONCE((paged_attn_kernel<T, D, BITS>), S::SMEM, "ha_paged_attn");
  const int64_t all = (int64_t)p.B * p.n, most = attn_lines(p);
  for (int64_t line0 = 0; line0 < all; line0 += most) {
    a.line0 = (int)line0;
    a.lines = (int)(all - line0 < most ? all - line0 : most);
    const int ctas = attn_ctas(p, a.lines);
    launch_chained(paged_attn_kernel<T, D, BITS>, ctas, 128, S::SMEM, st, a);
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
  if (p.H < 1) return HA_ERR_INVALID;
  if ((int64_t)p.B * p.n > 0x7fffffffLL - 65536 || (int64_t)p.H * p.d > 1 << 24) return HA_ERR_TOO_LARGE;
  if (p.B > 0 && p.n > 0 && attn_lines(p) < 1) return HA_ERR_TOO_LARGE;
  return HA_OK;
}

}  // namespace
}  // namespace ha

using namespace ha;

extern "C" {

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
  a.scale_log2 = p.scale * LOG2E;
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
