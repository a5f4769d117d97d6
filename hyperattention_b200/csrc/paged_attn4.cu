// Attention over 4-bit pages (the scheme of paged_attn.cu: items, list of tiles, parts).
//
// A quarter of the bytes, so that the work on a value counts: at the memory's rate an SM has some three instructions a value.  Codes become operands without
// arithmetic: code * 2^-24, 2^-22, 2^-20 and 2^-18 are fp16 numbers (subnormal ones) whose bits are the code's own, so that one mask makes a
// pair; steps and offsets are applied to the products.  Tensor cores cut products off as if a subnormal factor were as large as 2^-14: K's codes of the
// words shifted by six stand higher up and lose less, and those of one place go into one product (score of one key, fp16 queries: error 2.3e-6
// with the places 2^-24 and 2^-20 side by side, 1.2e-6 so; bf16: 9e-7 and 5e-7.  V's products have the weights' rounding above that).  With s, m of a group (a row's 64 elements):
//   q . k = sum over groups of s (q . code) + m sum(q),      o = sum p (s code + m) = sum (p s) (code - 7.5) + sum p (m + 7.5 s)
// Both products are taken transposed, keys (and then V's elements) as the 16 rows and queries as the 8 columns of mma.sync.m16n8k16: eight query heads
// cost half of what sixteen do, in products and in everything done per score.
//
// A CTA of four warps, each a quarter of a tile's keys and a ring of its own of NS stages, which it fills itself when it is done with one: between an item's
// begin and its end the warps do not wait for one another.  cp.async, whose copies of a warp's 32 or 64 neighbouring rows need two addresses: bulk copies,
// of which a warp's part of a tile takes four, cost some 100 instructions where these cost 40.
//
// Bound by instructions: batch of 64 x up to 32768, two K/V heads x 128, 16 query heads each: 81 us, 2.6 TB/s; without the copies 84, the copies alone 50.  1 x 262144, 32 heads
// x 64: 136 to 148 us from machine to machine, 4.1 to 4.4 TB/s; 124 and 97 on the first of them.  (Queries as the sixteen rows of the products and tiles fetched by
// a fifth warp took 105 and 323 us.)
#include <type_traits>

#include "paged_attn.cuh"

namespace ha {

namespace {


template <int D, int NQ>
struct Stage4 {
  static constexpr int NB = 2;                              // sixteens of keys that a warp takes at once
  static constexpr int KW = 16 * NB, TK = attn4_tile(D), WK = TK / 4;      // those keys; keys of a tile, a warp's of them
  static constexpr int ROW = D / 2, G = D / PAGED_GROUP, SC = 4 * G, ROWS = 8 * NQ;        // bytes of a row, of its scales; queries
  static constexpr int RUN = 512 / ROW;                      // rows of a copy of the warp
  static constexpr int V = WK * ROW, KS = 2 * WK * ROW, VS = KS + WK * SC, BYTES = VS + WK * SC;       // a warp's stage
  // (16 rows x 128: 170 registers a thread; for a fourth CTA sums would be spilled, 80 -> 107 us at 64 x 32768 tokens.  8 rows gain by it: 59.0 -> 57.1)
  static constexpr int CTAS = D == 128 && NQ == 2 ? 3 : 4, NS = 2;
  static constexpr int QF = (NQ == 2 ? D * 32 : 0) + (1 + G) * ROWS * 4;   // a warp's query operands (16 rows); units and sums of the queries
  static constexpr int WARP = NS * BYTES + QF + NS * 16 + 64;          // of a warp, too: what its stages hold, and its place in the list
  static constexpr int PARTS = ROWS * (D * 4 + 8);           // with clusters: the CTA's part
  static constexpr int SMEM = 4 * WARP + PARTS + 4 * ITEM_ROWS * 8 + (2 * MAX_LINES + 8) * 4 + 32 + MAX_LINES;
  static constexpr int ROUNDS = NQ;                          // in which the warps' sums are joined: column ranges that fit a stage
  static_assert(ROWS * D / ROUNDS * 4 <= BYTES, "a warp's sums fit a stage");
  static_assert(WK * ROW == 2048 && WK * SC == 256 && RUN * SC == 64 && WARP % 16 == 0, "copies of a warp's rows and scales");
  static_assert(CTAS * (SMEM + 1024) <= 228 * 1024, "CTAs of an SM");
};

// Row r (and r + 8) of a score fragment is key key_of(r) of its eight, so that the four pairs of keys that a load of V takes, 2c and 2c + 1 as the
// products count, are c and c + 4: neighbours, two to a bank instead of four.
__device__ __forceinline__ int key_of(int row) { return (row >> 1) | ((row & 1) << 2); }

// 8 x 8 matrix of 16-bit elements, a row's neighbours in a register: transposed
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float column_max(float v) {       // over the lanes that hold the same columns
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
}
__device__ __forceinline__ float column_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 4);
  v += __shfl_xor_sync(0xffffffffu, v, 8);
  return v + __shfl_xor_sync(0xffffffffu, v, 16);
}

template <typename T, int D, int NQ, bool PACKED>
struct Worker4 {
  using S = Stage4<D, NQ>;
  static constexpr int G = S::G, ROWS = S::ROWS, ROUNDS = S::ROUNDS, STEPS = D / 16, NB = S::NB, KW = S::KW;
  static constexpr float BIAS = 15.f - SLACK;  // weights times steps reach up to 2^15 and stay normal down to 2^-23 of that of the reference

  // Of queries 2c, 2c + 1 (c = lane % 4) of each eight.  Weights are exp2(score - shift), shift = ref + log2 v_top - BIAS, ref the largest score when it was last
  // looked for: when one came whose weight's exponent is above limit (the same for all queries; -inf while one has no score).
  float ref[NQ][2], limit;
  uint64_t below[NQ];                         // -shift
  uint64_t sum[NQ];
  uint64_t offset[G][NQ];                     // sums of weights times what a row's middle code stands for, less what the products count too much
  float acc[NQ][D / 16][4];
  float v_top;                                // power of two that no V step so far reaches
  uint32_t qf[NQ == 1 ? STEPS : 1][2];
  int k_at, s_at, v_at;                       // in a stage: this lane's codes of K and scales of key key_of(lane / 4), codes of V of key lane % 4
  uint4* qs;                                  // 16 queries: this warp's operands, [STEPS][32], in shared memory
  float* q_unit;                              // ... of each query: score of a code sum; [G] sums of its elements of a group, times the softmax scale
  int lane;

  // Query operands: fp16, every query times the power of two that brings its largest element to 2^13 .. 2^14.  Lane c of a query's four holds elements
  // 16 c .. 16 c + 15 of each group, paired as the codes come out of their words: (0, 4), (1, 5) / 16, (2, 6) / 4, (3, 7) / 64.
  __device__ __forceinline__ void begin(const AttnArgs& a, int line, int item) {
    const int c = lane & 3;
    const uint8_t* q = query_of(a, line, item);
    v_top = 0x1p-24f;
    limit = -INFINITY;
    uint32_t f[STEPS][2 * NQ];
    __syncwarp();                             // (the operands of the item before have been read)
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const int row = lane / 4 + 8 * n;
      const bool there = row_at<PACKED>(a, line, item, row).there;
      const uint8_t* from = q + (there ? query_row<PACKED>(a, row) : 0);
      float x[G][16], top = 0.f, s[G];
#pragma unroll
      for (int g = 0; g < G; ++g) {
        s[g] = 0.f;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const uint4 w = there ? *reinterpret_cast<const uint4*>(from + (8 * g + 2 * c + u) * 16) : make_uint4(0, 0, 0, 0);
          const uint32_t ws[4] = {w.x ^ a.flip, w.y ^ a.flip, w.z ^ a.flip, w.w ^ a.flip};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 v = unpack2<T>(ws[j]);
            x[g][8 * u + 2 * j] = v.x;
            x[g][8 * u + 2 * j + 1] = v.y;
            s[g] += v.x + v.y;
            top = max_nan(top, max_nan(fabsf(v.x), fabsf(v.y)));
          }
        }
        s[g] = quad_sum(s[g]) * a.scale_log2;
        if (c == 0) q_unit[(1 + g) * ROWS + row] = s[g];
        offset[g][n] = 0;
      }
      top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // exponent of the largest element; a query of zeros stays one, one with a NaN or an infinity keeps it through the products
      const int e = max((int)(__float_as_uint(top) >> 23) & 255, 27);
      const float up = __uint_as_float((uint32_t)(127 + 13 + 127 - e) << 23), down = __uint_as_float((uint32_t)(e - 13) << 23);
      if (c == 0) q_unit[row] = down * 16777216.f * a.scale_log2;
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const float by = up * (y == 0 ? 1.f : y == 1 ? 0x1p-4f : y == 2 ? 0x1p-2f : 0x1p-6f);
#pragma unroll
          for (int u = 0; u < 2; ++u) f[g * 4 + y][2 * n + u] = pack2<__half>(x[g][8 * u + y] * by, x[g][8 * u + y + 4] * by);
        }
      ref[n][0] = ref[n][1] = -INFINITY;
      below[n] = 0;
      sum[n] = 0;
    }
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int j = 0; j < D / 16; ++j)
#pragma unroll
        for (int y = 0; y < 4; ++y) acc[n][j][y] = 0.f;
    if constexpr (NQ == 1) {
#pragma unroll
      for (int y = 0; y < STEPS; ++y) qf[y][0] = f[y][0], qf[y][1] = f[y][1];
    } else {
#pragma unroll
      for (int y = 0; y < STEPS; ++y) qs[y * 32 + lane] = make_uint4(f[y][0], f[y][1], f[y][2], f[y][3]);
    }
    __syncwarp();
  }

  // New references; the sums so far follow, and the scores of this tile (less shift).
  __device__ __forceinline__ void raise(uint64_t (&x)[NB][2][NQ], float step) {
#pragma unroll
    for (int y = 1; y < 32; y *= 2) step = fmaxf(step, __shfl_xor_sync(0xffffffffu, step, y));
    v_top = fmaxf(v_top, __uint_as_float((__float_as_uint(step) & 0x7f800000u) + 0x800000u));
    const float v_exp = (float)((int)(__float_as_uint(v_top) >> 23) - 127);
    limit = BIAS - v_exp + SLACK;
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      float old[2], by[2], less[2], v[2] = {-INFINITY, -INFINITY};
      unpack_f2(below[n], old[0], old[1]);
#pragma unroll
      for (int y = 0; y < 2 * NB; ++y) {
        float u, w;
        unpack_f2(x[y >> 1][y & 1][n], u, w);
        v[0] = fmaxf(v[0], u);
        v[1] = fmaxf(v[1], w);
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float top = v[e] - old[e];
        const bool empty = ref[n][e] == -INFINITY;
        ref[n][e] = fmaxf(ref[n][e], column_max(top));
        if (ref[n][e] == -INFINITY) limit = -INFINITY;
        less[e] = ref[n][e] == -INFINITY ? 0.f : -ref[n][e] - (v_exp - BIAS);
        by[e] = empty ? 0.f : fast_exp2(less[e] - old[e]);             // (sums of a query without a score so far are zeros, or NaN)
      }
      const uint64_t by2 = pack_f2(by[0], by[1]), more = pack_f2(less[0] - old[0], less[1] - old[1]);
      below[n] = pack_f2(less[0], less[1]);
      sum[n] = fmul2(sum[n], by2);
#pragma unroll
      for (int y = 0; y < 2 * NB; ++y) x[y >> 1][y & 1][n] = fadd2(x[y >> 1][y & 1][n], more);
#pragma unroll
      for (int j = 0; j < D / 16; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[n][j][e] *= by[e & 1];
#pragma unroll
      for (int g = 0; g < G; ++g) offset[g][n] = fmul2(offset[g][n], by2);
    }
  }

  // Scales of V rows behind the last key hold anything: zeros instead.
  __device__ __forceinline__ void clear_tail(uint8_t* stage, int left) {
    for (int e = max(left, 0) * G + lane; e < S::WK * G; e += 32) *reinterpret_cast<uint32_t*>(stage + S::VS + e * 4) = 0;
    __syncwarp();
  }

  // words of a row (of its groups in turn), or scales: 2 G or G registers
  template <int N>
  static __device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&w)[N]) {
    if constexpr (N == 4) {
      const uint4 v = lds128(p);
      w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    } else if constexpr (N == 2) {
      const uint2 v = lds64(p);
      w[0] = v.x, w[1] = v.y;
    } else {
      w[0] = lds32(p);
    }
  }

  // KW keys of a tile from this warp's key `base` on, of which the line's last token, the `last`-th of its pack, sees the first `left`.
  __device__ __forceinline__ void keys(const AttnArgs& a, const uint8_t* stage, int base, int left, int last) {
    const int c = lane & 3, r = lane >> 2;
    const uint8_t *kp = stage + k_at + base * S::ROW, *sp = stage + s_at + base * S::SC, *vp = stage + v_at + base * S::ROW;
    constexpr uint32_t M0 = 0x000f000fu, M1 = 0x00f000f0u;
    uint64_t x[NB][2][NQ];                    // [16 keys][first, second eight]: scores less shift of two queries
#pragma unroll
    for (int blk = 0; blk < NB; ++blk) {
      uint32_t w[2][2 * G], sc[2][G];
      float d[G][NQ][4];
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        load_words(kp + (16 * blk + 8 * y) * S::ROW, w[y]);
        load_words(sp + S::KS + (16 * blk + 8 * y) * S::SC, sc[y]);
      }
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) d[g][n][e] = 0.f;
#pragma unroll
      for (int y = 0; y < 4; ++y)             // elements y, y + 4 of the words
#pragma unroll
        for (int g = 0; g < G; ++g) {
          constexpr uint32_t M[4] = {0x000f000fu, 0x00f000f0u, 0x003c003cu, 0x03c003c0u};
          const int by = y < 2 ? 0 : 6, step = g * 4 + y;
          const uint32_t k[4] = {(w[0][g] >> by) & M[y], (w[1][g] >> by) & M[y], (w[0][G + g] >> by) & M[y], (w[1][G + g] >> by) & M[y]};
          if constexpr (NQ == 1) {
            mma16816<__half>(d[g][0], k, qf[step][0], qf[step][1]);
          } else {
            const uint4 q = qs[step * 32 + lane];
            mma16816<__half>(d[g][0], k, q.x, q.y);
            mma16816<__half>(d[g][1], k, q.z, q.w);
          }
        }
      uint64_t unit[NQ], qsum[G][NQ];
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        unit[n] = *reinterpret_cast<const uint64_t*>(q_unit + 8 * n + 2 * c);
#pragma unroll
        for (int g = 0; g < G; ++g) qsum[g][n] = *reinterpret_cast<const uint64_t*>(q_unit + (1 + g) * ROWS + 8 * n + 2 * c);
      }
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        float2 f[G];
#pragma unroll
        for (int g = 0; g < G; ++g) f[g] = unpack2<__half>(sc[y][g]);                // step, value of code 0
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          uint64_t p, z = below[n];
#pragma unroll
          for (int g = 0; g < G; ++g) {
            const uint64_t dd = pack_f2(d[g][n][2 * y], d[g][n][2 * y + 1]);
            p = g == 0 ? fmul2(dup_f2(f[g].x), dd) : ffma2(dup_f2(f[g].x), dd, p);
            z = ffma2(dup_f2(f[g].y), qsum[g][n], z);
          }
          x[blk][y][n] = ffma2(p, unit[n], z);
        }
      }
    }
    const bool mixed = left - last < KW;
    if (mixed) {
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        const int sees[2] = {left - keys_short<PACKED>(a, 8 * n + 2 * c, last), left - keys_short<PACKED>(a, 8 * n + 2 * c + 1, last)};
#pragma unroll
        for (int blk = 0; blk < NB; ++blk)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const int key = blk * 16 + y * 8 + key_of(r);
            float u, v;
            unpack_f2(x[blk][y][n], u, v);
            x[blk][y][n] = pack_f2(key < sees[0] ? u : -INFINITY, key < sees[1] ? v : -INFINITY);
          }
      }
    }
    float top = -INFINITY;
#pragma unroll
    for (int y = 0; y < 2 * NB; ++y)
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        float u, v;
        unpack_f2(x[y >> 1][y & 1][n], u, v);
        top = fmax3(top, u, v);
      }
    uint32_t vs[NB][2][G];
    __half2 most = __half2half2(__ushort_as_half(0));
#pragma unroll
    for (int blk = 0; blk < NB; ++blk)
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        load_words(sp + S::VS + (16 * blk + 8 * y) * S::SC, vs[blk][y]);
#pragma unroll
        for (int g = 0; g < G; ++g) most = __hmax2(most, __habs2(*reinterpret_cast<const __half2*>(&vs[blk][y][g])));
      }
    const float step = __low2float(most);
    if (__any_sync(0xffffffffu, top > limit || step >= v_top)) raise(x, step);
    // Weights times steps are rounded to fp16.  What the middle code stands for is added in 32 bits, and the rounded weights are summed up by the same
    // products, so that a rounding meets (code - 7.5) and not the code.  Odd keys (as the products count) enter as 15 - code with the weight's
    // sign turned: the sums stay near the middle, where tensor cores, which cut sums off instead of rounding them, lose nothing that counts
    // (262144 keys, fp16 output: error 1.3e-3 with plain codes, 2.4e-4 with these; the output's own rounding is 2.0e-4).
    const uint32_t sign = (r & 1) ? 0x8000u : 0u;
    const float mid = (r & 1) ? -7.5f : 7.5f;
#pragma unroll
    for (int blk = 0; blk < NB; ++blk) {
      uint32_t pb[G][NQ][2];
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        uint64_t p[NQ];
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          float u, v;
          unpack_f2(x[blk][y][n], u, v);
          p[n] = pack_f2(fast_exp2(u), fast_exp2(v));
          sum[n] = fadd2(sum[n], p[n]);
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const float2 f = unpack2<__half>(vs[blk][y][g] ^ sign);
          const float m = fmaf(f.x, mid, f.y);
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
            float u, v;
            uint64_t mids = dup_f2(m);
            unpack_f2(fmul2(p[n], dup_f2(f.x)), u, v);
            if (PACKED && mixed) {            // (a group that stands for no number counts for the queries that see its key, and for no others)
              float pu, pv;
              unpack_f2(p[n], pu, pv);
              if (pu == 0.f) u = 0.f;
              if (pv == 0.f) v = 0.f;
              mids = pack_f2(pu == 0.f ? 0.f : m, pv == 0.f ? 0.f : m);
            }
            pb[g][n][y] = transposed(pack2<__half>(u, v));
            offset[g][n] = ffma2(p[n], mids, offset[g][n]);
          }
        }
      }
      uint32_t w[4][G];                       // keys c, c + 4 of the first eight, of the second
#pragma unroll
      for (int y = 0; y < 4; ++y) load_words(vp + S::V + (16 * blk + (y >> 1) * 8 + 4 * (y & 1)) * S::ROW, w[y]);
      const uint32_t ones[4] = {0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u};
      constexpr uint32_t X0 = 0x000f0000u, X1 = 0x00f00000u;
#pragma unroll
      for (int g = 0; g < G; ++g) {
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          float sums[4] = {0.f, 0.f, 0.f, 0.f};
          mma16816<__half>(sums, ones, pb[g][n][0], pb[g][n][1]);
          offset[g][n] = ffma2(pack_f2(sums[0], sums[1]), lane < 4 ? dup_f2(-7.5f) : 0, offset[g][n]);      // (every row of the product alike)
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {         // elements 2j, 2j + 1 of the words
          const uint32_t sel = j & 2 ? 0x7632u : 0x5410u;
          const uint32_t a = __byte_perm(w[0][g], w[1][g], sel) >> (8 * (j & 1)), b = __byte_perm(w[2][g], w[3][g], sel) >> (8 * (j & 1));
          const uint32_t v[4] = {and_xor(a, M0, X0), and_xor(a, M1, X1), and_xor(b, M0, X0), and_xor(b, M1, X1)};
#pragma unroll
          for (int n = 0; n < NQ; ++n) mma16816<__half>(acc[n][g * 4 + j], v, pb[g][n][0], pb[g][n][1]);
        }
      }
    }
  }

  // (shift, denominator) of the queries; a warp without keys has no part, one whose scores are all NaN has
  __device__ __forceinline__ void statistics(float2* stat) {
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      float l[2], less[2];
      unpack_f2(sum[n], l[0], l[1]);
      unpack_f2(below[n], less[0], less[1]);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        l[e] = column_sum(l[e]);
        if (lane < 4) stat[8 * n + 2 * lane + e] = make_float2(ref[n][e] == -INFINITY && l[e] == 0.f ? -INFINITY : -less[e], l[e]);
      }
#pragma unroll
      for (int g = 0; g < G; ++g) {
        float u, v;
        unpack_f2(offset[g][n], u, v);
        offset[g][n] = pack_f2(column_sum(u), column_sum(v));
      }
    }
  }
  // This warp's sums of columns [round * D / ROUNDS ..), rows of D / ROUNDS floats; columns of 8 turned by the row.
  static __device__ __forceinline__ int turn(int row) { return ((row >> 1) & 3) << 3; }
  __device__ __forceinline__ void put(float* to, int round) {
    const int c = lane & 3, r = lane >> 2;
    constexpr int W = D / ROUNDS;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const int col = 64 * g + 8 * r;         // this lane's eight elements
      if (ROUNDS > 1 && col / W != round) continue;
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        float m[2];
        unpack_f2(offset[g][n], m[0], m[1]);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int row = 8 * n + 2 * c + e;
          const float mid = m[e];
          float* line = to + row * W + ((col % W) ^ turn(row));
          float4 v;
#pragma unroll
          for (int j = 0; j < 4; j += 2) {
            const float(*o)[4] = &acc[n][g * 4 + j];
            v.x = fmaf(o[0][e], 16777216.f, mid);
            v.y = fmaf(o[0][2 + e], 1048576.f, mid);
            v.z = fmaf(o[1][e], 16777216.f, mid);
            v.w = fmaf(o[1][2 + e], 1048576.f, mid);
            *reinterpret_cast<float4*>(line + 2 * j) = v;
          }
        }
      }
    }
  }
};

// Where a warp's fetching stands, for one lane: what changes from tile to tile, and what an item's tiles have in common.
struct alignas(16) Place {
  int line, item, tile, tiles;
  const int32_t* table;               // of the sequence
  int64_t head, head_s;               // offsets of the K/V head in a page, of its scales
  int keys;
};

template <typename T, int D, int NQ, bool CLUSTER, bool PACKED>
__global__ void __launch_bounds__(128, (Stage4<D, NQ>::CTAS)) paged_attn4_kernel(const __grid_constant__ AttnArgs a) {
  using S = Stage4<D, NQ>;
  constexpr int NS = S::NS, TK = S::TK, KW = S::KW, WK = S::WK;
  extern __shared__ __align__(1024) uint8_t smem[];
  float* cluster_sums = reinterpret_cast<float*>(smem + 4 * S::WARP);        // [ROWS][D]
  float2* cluster_stat = reinterpret_cast<float2*>(cluster_sums + S::ROWS * D);
  float2* stat = cluster_stat + S::ROWS;                                     // [4][ITEM_ROWS]
  int* first = reinterpret_cast<int*>(stat + 4 * ITEM_ROWS);                 // [lines + 1]
  int* abort_flag = first + MAX_LINES + 3;
  int* keys = first + MAX_LINES + 4;                                         // [lines]
  const uint32_t join_bar = smem_u32(keys + MAX_LINES);
  int* warp_sum = keys + MAX_LINES + 2;                                      // [4]
  uint8_t* lasts = reinterpret_cast<uint8_t*>(warp_sum + 4);                 // [lines]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int items = a.Hk * a.blocks;
  if (tid == 0) {
    mbar_init(join_bar, 4);
    mbar_fence_init();
    *abort_flag = 0;
  }
  if (CLUSTER) chain_release();              // (as in paged_attn.cu: the kernel behind is let in at the end, or at once)
  chain_wait();
  int begin, end, line0;
  const Walk start = take_part<T, D, CLUSTER>(a, TK, 1, first, keys, lasts, warp_sum, items, begin, end, line0);
  const int lines = CLUSTER ? 1 : a.lines;
  if (begin >= end && (!CLUSTER || keys[0] == 0)) return;

  uint8_t* mine = smem + warp * S::WARP;                                     // stages, query operands, what the stages hold
  int4* what = reinterpret_cast<int4*>(mine + NS * S::BYTES + S::QF);
  Place* place = reinterpret_cast<Place*>(what + NS);
  const uint32_t base = smem_u32(mine);
  auto settle = [&](const Walk& f) {
    const int h = a.by_blocks(f.item);
    place->table = a.c.table + a.by_packs(line0 + f.line) * a.c.table_sb;
    place->head = h * a.c.sh;
    place->head_s = h * a.c.ssh;
    place->keys = keys[f.line];
  };
  // This warp's keys of the next tile into stage s.
  auto fetch = [&](int s) {
    const Place f = *place;
    const int key0 = f.tile * TK + warp * WK, left = f.keys - key0;
    const uint32_t dst = base + s * S::BYTES;
    if (a.runs == 2) {
      // rows that lie together, and their scales (of all WK, whatever they are behind the last key: the page has them)
      if (left > 0) {
        const int col = a.c.by_page(key0), slot = key0 - col * a.c.page_size, page = f.table[col];
        if (paged_checked(a.c, page)) {
          const int64_t off = page * a.c.sp + f.head + (int64_t)slot * S::ROW + lane * 16, off_s = page * a.c.ssp + f.head_s + (int64_t)slot * S::SC + (lane & 15) * 16;
          const uint8_t *k = a.c.k + off, *v = a.c.v + off, *sc = (lane < 16 ? a.c.ks : a.c.vs) + off_s;
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            cp_async16(dst + lane * 16 + 512 * y, k + 512 * y, 16);
            cp_async16(dst + lane * 16 + S::V + 512 * y, v + 512 * y, 16);
          }
          cp_async16(dst + S::KS + lane * 16, sc, 16);
        }
      }
    } else if (a.runs == 1) {
      // ... in runs of RUN, one a copy of the warp; scales by the lanes that look the run up (64 x 32768 tokens, pages of 16: 97 us row by row, 86 so, 81 where pages hold the
      // whole part; 1 x 262144, 32 heads x 64, pages of 32: 179, 149, 137)
      constexpr int RUN = S::RUN;
      const int first_row = RUN * ((lane & 15) >> 2);
      int64_t off = -1, off_s = 0;
      if (first_row < left) {
        const int col = a.c.by_page(key0 + first_row), slot = key0 + first_row - col * a.c.page_size, page = f.table[col];
        if (paged_checked(a.c, page)) {
          off = page * a.c.sp + f.head + (int64_t)slot * S::ROW;
          off_s = page * a.c.ssp + f.head_s + (int64_t)slot * S::SC;
        }
      }
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const int64_t from = __shfl_sync(0xffffffffu, off, 4 * y);
        if (from >= 0) {
          cp_async16(dst + lane * 16 + 512 * y, a.c.k + from + lane * 16, 16);
          cp_async16(dst + lane * 16 + S::V + 512 * y, a.c.v + from + lane * 16, 16);
        }
      }
      if (off >= 0) cp_async16(dst + S::KS + lane * 16, (lane < 16 ? a.c.ks : a.c.vs) + off_s + (lane & 3) * 16, 16);
    } else {
      constexpr int C = S::ROW / 16;
      for (int e = lane; e < WK * C; e += 32) {
        const int row = e / C, chunk = e % C;
        int slot = 0, page = -1;
        if (row < left) {
          const int col = a.c.by_page(key0 + row);
          slot = key0 + row - col * a.c.page_size;
          page = f.table[col];
          if (!paged_checked(a.c, page)) page = -1;
        }
        if (page >= 0) {
          const int64_t off = page * a.c.sp + f.head + slot * a.c.st + chunk * 16;
          cp_async16(dst + e * 16, a.c.k + off, 16);
          cp_async16(dst + S::V + e * 16, a.c.v + off, 16);
          if (chunk == 0) {
            const int64_t off_s = page * a.c.ssp + f.head_s + slot * a.c.sst;
            cp_async_small<S::SC>(dst + S::KS + row * S::SC, a.c.ks + off_s, S::SC);
            cp_async_small<S::SC>(dst + S::VS + row * S::SC, a.c.vs + off_s, S::SC);
          }
        }
      }
    }
    __syncwarp();
    if (lane == 0) {
      what[s] = make_int4(left, f.line, f.item, f.tile);
      if (f.tile + 1 < f.tiles) {
        place->tile = f.tile + 1;
      } else {
        Walk next = {f.line, f.item, f.tile, f.tiles};
        next.step(first, lines, items);
        place->line = next.line, place->item = next.item, place->tile = next.tile, place->tiles = next.tiles;
        if (next.line < lines) settle(next);
      }
    }
    __syncwarp();
  };

  Worker4<T, D, NQ, PACKED> w;
  w.lane = lane;
  w.qs = reinterpret_cast<uint4*>(mine + NS * S::BYTES);
  w.q_unit = reinterpret_cast<float*>(mine + NS * S::BYTES + (NQ == 2 ? D * 32 : 0));
  w.k_at = key_of(lane >> 2) * S::ROW + (lane & 3) * (8 * S::G);
  w.s_at = key_of(lane >> 2) * S::SC;
  w.v_at = (lane & 3) * S::ROW + (lane >> 2) * (4 * S::G);
  uint32_t joined = 0;
  auto join = [&]() {
    __syncwarp();
    if (lane == 0) mbar_arrive(join_bar);
    return mbar_wait_or_abort(join_bar, joined++ & 1, abort_flag);
  };
  if (lane == 0) {
    place->line = start.line, place->item = start.item, place->tile = start.tile, place->tiles = start.tiles;
    settle(start);
  }
  __syncwarp();
#pragma unroll 1
  for (int y = 0; y < NS; ++y) {
    if (begin + y < end) fetch(y);
    cp_async_commit();
  }
  int s = 0;
  bool ok = true;
#pragma unroll 1
  for (int it = begin; it < end; ++it) {
    uint8_t* stage = mine + s * S::BYTES;
    cp_async_wait<NS - 1>();
    __syncwarp();
    const int4 t = what[s];
    if (it == begin || t.w == 0) {
      w.begin(a, line0 + t.y, t.z);
    }
    const int last = PACKED ? lasts[t.y] : 0;
    if (t.x < WK) w.clear_tail(stage, t.x);
#pragma unroll
    for (int y = 0; y < WK; y += KW) w.keys(a, stage, y, t.x - y, last);
    if (t.x + warp * WK <= TK || it == end - 1) {
      const Walk at = {t.y, t.z, t.w, first[t.y + 1] - first[t.y]};
      ok = finish_item<T, D, S::WARP / 4, CLUSTER, PACKED>(a, w, stat, reinterpret_cast<float*>(smem + s * S::BYTES), at, first, items, begin, end, it == end - 1, line0, keys[t.y],
                                                              last, cluster_sums, cluster_stat, join) &&
           join();
      if (!ok) break;
    }
    __syncwarp();
    if (it + NS < end) fetch(s);
    cp_async_commit();
    if (++s == NS) s = 0;
  }
  if constexpr (CLUSTER) {
    if (begin >= end || !ok) {
      if (tid < S::ROWS) cluster_stat[tid] = make_float2(-INFINITY, -1.f);
    }
    __syncwarp();
    cluster_finish<T, D, PACKED>(a, cluster_sums, cluster_stat, line0, start.item, keys[0], lasts[0]);
  }
  if (!ok && !CLUSTER && tid == 0) a.head[blockIdx.x] = make_int4(0, 0, 0, 0);       // nothing to join from here
  if (!ok && lane == 0) report_timeout(a.c.status, a.c.status_host);
  cp_async_wait<0>();
  chain_release();
}

template <typename T, int D, int NQ>
int launch4(const AttnArgs& a, int ctas, cudaStream_t st) {
  using S = Stage4<D, NQ>;
  auto launch = [&](auto kernel) {
    if (a.cluster > 0) launch_chained_clusters(kernel, ctas, 128, S::SMEM, a.cluster, st, a);
    else launch_chained(kernel, ctas, 128, S::SMEM, st, a);
  };
#define HA_PAGED_VARIANT(cluster, packed)                                                          \
  do {                                                                                             \
    HA_SMEM_ATTR_ONCE((paged_attn4_kernel<T, D, NQ, cluster, packed>), S::SMEM, "ha_paged_attn");  \
    if (cluster) HA_ATTR_ONCE((paged_attn4_kernel<T, D, NQ, cluster, packed>), cudaFuncAttributeNonPortableClusterSizeAllowed, 1, "ha_paged_attn"); \
    launch(paged_attn4_kernel<T, D, NQ, cluster, packed>);                                         \
  } while (0)
  if (a.cluster > 0 && a.pack > 1) HA_PAGED_VARIANT(true, true);
  else if (a.cluster > 0) HA_PAGED_VARIANT(true, false);
  else if (a.pack > 1) HA_PAGED_VARIANT(false, true);
  else HA_PAGED_VARIANT(false, false);
#undef HA_PAGED_VARIANT
  HA_LAUNCHED("ha_paged_attn");
  return HA_OK;
}

}  // namespace

int attn4_resident(int d, int rows) {
  if (d == 128) return rows > 8 ? Stage4<128, 2>::CTAS : Stage4<128, 1>::CTAS;
  return rows > 8 ? Stage4<64, 2>::CTAS : Stage4<64, 1>::CTAS;
}

int attn4_launch(AttnArgs a, int dtype, int d, int ctas, cudaStream_t st) {
  const bool bf = dtype == HA_BF16, many = a.group * a.pack > 8;
  if (d == 128) {
    if (many) return bf ? launch4<__nv_bfloat16, 128, 2>(a, ctas, st) : launch4<__half, 128, 2>(a, ctas, st);
    return bf ? launch4<__nv_bfloat16, 128, 1>(a, ctas, st) : launch4<__half, 128, 1>(a, ctas, st);
  }
  if (many) return bf ? launch4<__nv_bfloat16, 64, 2>(a, ctas, st) : launch4<__half, 64, 2>(a, ctas, st);
  return bf ? launch4<__nv_bfloat16, 64, 1>(a, ctas, st) : launch4<__half, 64, 1>(a, ctas, st);
}

}  // namespace ha
