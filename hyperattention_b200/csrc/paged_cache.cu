// Writing rows to the paged key/value cache (position rotation and 4-bit coding on the way) and reading them back as dense tensors.
#include "paged.cuh"

namespace ha {

constexpr int PART = 16;           // elements of a row that a lane takes

// Sixteen neighbouring elements of a row, as they lie (two or eight loads' worth).
template <typename T, bool WIDE>
__device__ __forceinline__ void load_raw(const T* src, uint4 (&r)[2]) {
  if (WIDE) {
    r[0] = __ldg(reinterpret_cast<const uint4*>(src));
    r[1] = __ldg(reinterpret_cast<const uint4*>(src) + 1);
  } else {
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint16_t lo = __ldg(reinterpret_cast<const uint16_t*>(src) + 2 * j), hi = __ldg(reinterpret_cast<const uint16_t*>(src) + 2 * j + 1);
      w[j] = lo | (uint32_t)hi << 16;
    }
    r[0] = make_uint4(w[0], w[1], w[2], w[3]);
    r[1] = make_uint4(w[4], w[5], w[6], w[7]);
  }
}
template <typename T>
__device__ __forceinline__ void unpack16(const uint4 (&r)[2], float (&x)[PART]) {
  const uint32_t w[8] = {r[0].x, r[0].y, r[0].z, r[0].w, r[1].x, r[1].y, r[1].z, r[1].w};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float2 f = unpack2<T>(w[j]);
    x[2 * j] = f.x;
    x[2 * j + 1] = f.y;
  }
}
template <typename T>
__device__ __forceinline__ void store16(void* dst, const float (&x)[PART]) {
  uint4* d = reinterpret_cast<uint4*>(dst);
#pragma unroll
  for (int y = 0; y < 2; ++y)
    d[y] = make_uint4(pack2<T>(x[8 * y], x[8 * y + 1]), pack2<T>(x[8 * y + 2], x[8 * y + 3]), pack2<T>(x[8 * y + 4], x[8 * y + 5]), pack2<T>(x[8 * y + 6], x[8 * y + 7]));
}

struct AppendArgs {
  PagedView c;
  const void *q, *k, *v;
  int64_t q_sb, q_sn, q_sh, k_sb, k_sn, k_sh, v_sb, v_sn, v_sh;
  const void* rope;
  int32_t n, H, Hk, rot, rope_rows, rope_f32, rope_wide;      // rope_wide: a lane's cosines and sines are all there or none, on 16-byte boundaries
  int64_t tokens;
  FastDiv by_n;
  void *q_out, *k_out;
};

// A lane's share of a position's rotation: cosines and sines of its eight pairs, as far as they are rotated.
struct Turn {
  float cs[8], sn[8];
  int pairs;
  // Products and sums are rounded one by one (no fused multiply-add), so that the results, and with them the 4-bit codes, are those of the
  // formula in 32 bits, whoever evaluates it.
  __device__ __forceinline__ void pair(float (&x)[PART], int j) const {
    const float x0 = x[2 * j], x1 = x[2 * j + 1];
    x[2 * j] = __fsub_rn(__fmul_rn(x0, cs[j]), __fmul_rn(x1, sn[j]));
    x[2 * j + 1] = __fadd_rn(__fmul_rn(x1, cs[j]), __fmul_rn(x0, sn[j]));
  }
  __device__ __forceinline__ void operator()(float (&x)[PART]) const {
    if (pairs == 8) {
#pragma unroll
      for (int j = 0; j < 8; ++j) pair(x, j);
    } else if (pairs > 0) {
#pragma unroll
      for (int j = 0; j < 7; ++j)
        if (j < pairs) pair(x, j);
    }
  }
};

// smallest and largest of three; a NaN among them stays one
__device__ __forceinline__ float min3_nan(float a, float b, float c) {
  float d;
  asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Sixteen elements of a 64-element group that four neighbouring lanes hold, as two words of codes; the group's step and offset to all of them.
__device__ __forceinline__ uint2 quantise(const float (&x)[PART], __half2& scale) {
  const uint32_t four = 0xfu << (threadIdx.x & 28);
  float lo = min3_nan(x[0], x[1], x[2]), hi = max3_nan(x[0], x[1], x[2]);
#pragma unroll
  for (int j = 3; j < 15; j += 2) {
    lo = min3_nan(lo, x[j], x[j + 1]);
    hi = max3_nan(hi, x[j], x[j + 1]);
  }
  lo = min3_nan(lo, x[15], x[15]);
  hi = max3_nan(hi, x[15], x[15]);
#pragma unroll
  for (int s = 1; s < 4; s *= 2) {
    const float u = __shfl_xor_sync(four, lo, s), v = __shfl_xor_sync(four, hi, s);
    lo = min3_nan(lo, u, u);
    hi = max3_nan(hi, v, v);
  }
  // (hi - lo) / 15, rounded once: the quotient of a product with the rounded reciprocal, corrected by its exact remainder (Markstein, 1990).  Where the
  // span is infinite, or the difference of infinities, it becomes NaN.
  const float span = __fsub_rn(hi, lo), q0 = __fmul_rn(span, 1.f / 15.f), q1 = fmaf(fmaf(-15.f, q0, span), 1.f / 15.f, q0);
  __half2 sm = __floats2half2_rn(q1, lo);
  // neither may be infinite or no number: the exponent's bits all set
  const uint32_t bits = *reinterpret_cast<const uint32_t*>(&sm);
  if ((bits & 0x7c00u) == 0x7c00u || (bits & 0x7c000000u) == 0x7c000000u) {
    scale = __halves2half2(__ushort_as_half(0), __ushort_as_half(0x7fff));
    return make_uint2(0, 0);
  }
  scale = sm;
  const float2 step = unpack2<__half>(bits);
  const float s = step.x, m = step.y;
  if (!(s > 0.f)) return make_uint2(0, 0);
  // The code is rint of the rounded quotient (x - m) / s, between 0 and 15.  x * (1 / s) - m * (1 / s) is within 2^-21 (|m / s| + 16) of it; where that leaves
  // the nearest number open, or the offset's own rounding puts an extreme out of the range, and there alone, the quotient itself is taken.
  const float inv = __fdividef(1.f, s), low = -m * inv, magic = 12582912.f;      // 1.5 * 2^23: adding it rounds to a whole number
  const float open = 0.5f - (fabsf(low) + 16.f) * 0x1p-20f;
  float off = 0.f;
  uint64_t c[PART / 2];              // pairs of neighbours
#pragma unroll
  for (int j = 0; j < PART / 2; ++j) {
    const uint64_t t = ffma2(pack_f2(x[2 * j], x[2 * j + 1]), dup_f2(inv), dup_f2(low));
    c[j] = fadd2(fadd2(t, dup_f2(magic)), dup_f2(-magic));
    float u, v;
    unpack_f2(ffma2(c[j], dup_f2(-1.f), t), u, v);
    off = fmax3(off, fabsf(u), fabsf(v));
  }
  if (off > open || fmaf(hi, inv, low) > 15.25f || fmaf(lo, inv, low) < -0.25f) {
#pragma unroll
    for (int j = 0; j < PART / 2; ++j) {
      const float u = rintf(__fdiv_rn(__fsub_rn(x[2 * j], m), s)), v = rintf(__fdiv_rn(__fsub_rn(x[2 * j + 1], m), s));
      c[j] = pack_f2(fminf(fmaxf(u, 0.f), 15.f), fminf(fmaxf(v, 0.f), 15.f));
    }
  }
  // (sums of four codes are whole numbers below 2^16)
  uint32_t w[4];
#pragma unroll
  for (int y = 0; y < 4; ++y) {
    float u, v;
    unpack_f2(ffma2(c[2 * y + 1], dup_f2(256.f), c[2 * y]), u, v);
    w[y] = (uint32_t)fmaf(v, 16.f, u);
  }
  return make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
}

// One block a token, D / 16 lanes a row, sixteen elements a lane, which keeps its cosines and sines for all the heads that it meets; two rows of a
// lane under way at once.  Bound by the bytes of q, k and v for long prompts, by the chain length -> page -> store for single tokens.  32768 tokens, 32 + 2 + 2
// heads x 128: 97 to 103 us from machine to machine, 5.9 to 6.3 TB/s; 2 x 8191 tokens, 32 + 32 + 32 heads x 64, into 4 bits: 77 to 80 us, 3.8 to 4.0 TB/s: a block's
// rounds of loads one after another, with the codes' arithmetic between them; one token of 32 sequences: 2.4 us.  (16 bits: 20 warps an SM, 96 registers:
// 24 x 2319 tokens, 12 + 2 + 2 heads x 128, 82.8 -> 75.3 us; 24 warps spill.  4 bits: 16 warps, 120 of their 128 registers: by 18 or 20 with spilled ones
// 107 -> 114 us, by fewer with more 124.)
template <typename T, int D, int BITS, bool WIDE, int THREADS>
__global__ void __launch_bounds__(THREADS, (BITS == 16 ? 640 : 512) / THREADS) paged_append_kernel(const AppendArgs a) {
  chain_begin();
  constexpr int LANES = D / PART, GROUPS = THREADS / LANES;
  const int lane = threadIdx.x % LANES, grp = threadIdx.x / LANES;
  for (int64_t tok = blockIdx.x; tok < a.tokens; tok += gridDim.x) {
    const int b = a.by_n((int)tok), i = (int)(tok - (int64_t)b * a.n);
    // the rows, the first of a lane before anything is known of their place: those loads and the chain of the others are under way together
    const T* src = (const T*)a.q + b * a.q_sb + i * a.q_sn + lane * PART;
    const T *ksrc = (const T*)a.k + b * a.k_sb + i * a.k_sn + lane * PART, *vsrc = (const T*)a.v + b * a.v_sb + i * a.v_sn + lane * PART;
    uint4 qraw[2][2], kraw[2], vraw[2];
    auto load_q = [&](int h) {
      if (h < a.H) load_raw<T, WIDE>(src + h * a.q_sh, qraw[0]);
      if (h + GROUPS < a.H) load_raw<T, WIDE>(src + (h + GROUPS) * a.q_sh, qraw[1]);
    };
    auto load_kv = [&](int h) {
      if (h < a.Hk) {
        load_raw<T, WIDE>(ksrc + h * a.k_sh, kraw);
        load_raw<T, WIDE>(vsrc + h * a.v_sh, vraw);
      }
    };
    load_q(grp);
    load_kv(grp);
    const int len = a.c.lengths[b];
    const bool live = i < (a.c.counts ? a.c.counts[b] : a.n);
    const bool ok = live && len >= 0 && len < a.c.capacity - i && (!a.rope || len < a.rope_rows - i);
    if (live && !ok && threadIdx.x == 0) report_status(a.c.status, a.c.status_host, HA_DEV_BAD_INDEX);
    const int pos = ok ? len + i : 0;
    int row = 0, page = -1;
    if (ok) page = paged_entry(a.c, b, pos, row);
    if (!live) {                                      // padding: zeros, and nothing to keep
      const uint4 zero = make_uint4(0, 0, 0, 0);
      if (a.q)
        for (int e = threadIdx.x; e < a.H * D / 8; e += THREADS) reinterpret_cast<uint4*>((T*)a.q_out + tok * a.H * D)[e] = zero;
      if (a.k_out)
        for (int e = threadIdx.x; e < a.Hk * D / 8; e += THREADS) reinterpret_cast<uint4*>((T*)a.k_out + tok * a.Hk * D)[e] = zero;
      continue;
    }
    Turn turn;
    turn.pairs = 0;
    if (a.rope && ok) {
      const int pairs = a.rot / 2 - lane * 8;
      turn.pairs = pairs < 0 ? 0 : pairs > 8 ? 8 : pairs;
      const int64_t at = ((int64_t)pos * (a.rot / 2) + lane * 8) * 2;
      if (a.rope_wide && turn.pairs == 8) {
        if (a.rope_f32) {
          const float4* src = reinterpret_cast<const float4*>((const float*)a.rope + at);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float4 u = __ldg(src + j);
            turn.cs[2 * j] = u.x, turn.sn[2 * j] = u.y, turn.cs[2 * j + 1] = u.z, turn.sn[2 * j + 1] = u.w;
          }
        } else {
          uint4 raw[2];
          float x[PART];
          load_raw<T, true>((const T*)a.rope + at, raw);
          unpack16<T>(raw, x);
#pragma unroll
          for (int j = 0; j < 8; ++j) turn.cs[j] = x[2 * j], turn.sn[j] = x[2 * j + 1];
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (j < turn.pairs) {
            turn.cs[j] = a.rope_f32 ? ((const float*)a.rope)[at + 2 * j] : to_f32<T>(((const T*)a.rope)[at + 2 * j]);
            turn.sn[j] = a.rope_f32 ? ((const float*)a.rope)[at + 2 * j + 1] : to_f32<T>(((const T*)a.rope)[at + 2 * j + 1]);
          }
      }
    }
    T* dst = (T*)a.q_out + tok * a.H * D + lane * PART;
    for (int h = grp; h < a.H; h += 2 * GROUPS) {
      if (h != grp) load_q(h);
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        if (h + y * GROUPS >= a.H) break;
        float x[PART];
        unpack16<T>(qraw[y], x);
        turn(x);
        store16<T>(dst + (h + y * GROUPS) * D, x);
      }
    }
    if (ok && !paged_checked(a.c, page)) page = -1;
    const int64_t off = page * a.c.sp + row * a.c.st, off_s = page * a.c.ssp + row * a.c.sst;
    // key and value of a head by the same lanes
    for (int h = grp; h < a.Hk; h += GROUPS) {
      if (h != grp) load_kv(h);
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        uint8_t* dst = (y ? a.c.v : a.c.k) + off + h * a.c.sh;
        float x[PART];
        if (BITS == 4 || y == 0) unpack16<T>(y ? vraw : kraw, x);
        if (y == 0) {
          turn(x);
          if (a.k_out) store16<T>((T*)a.k_out + (tok * a.Hk + h) * D + lane * PART, x);
        }
        if (BITS == 16) {
          if (page < 0) continue;
          if (y == 0) {
            store16<T>(dst + lane * 32, x);
          } else {
            reinterpret_cast<uint4*>(dst + lane * 32)[0] = vraw[0];
            reinterpret_cast<uint4*>(dst + lane * 32)[1] = vraw[1];
          }
        } else {
          __half2 scale;
          const uint2 w = quantise(x, scale);
          if (page < 0) continue;
          constexpr int G = D / PAGED_GROUP;
          const int g = lane / 4, first = (lane % 4) * 2 * G + g;       // words of the groups in turn
          *reinterpret_cast<uint32_t*>(dst + 4 * first) = w.x;
          *reinterpret_cast<uint32_t*>(dst + 4 * (first + G)) = w.y;
          if (lane % 4 == 0) *reinterpret_cast<__half2*>((y ? a.c.vs : a.c.ks) + off_s + h * a.c.ssh + 4 * g) = scale;
        }
      }
    }
  }
}

struct GatherArgs {
  PagedView c;
  int32_t Hk, rows;
  FastDiv by_blocks, by_heads;
  void *k_out, *v_out;
};

// Eight codes as numbers code * step + offset, in T.  The product is exact in 32 bits (4 and 11 bits), so that the sum is the value's one rounding before T's.
template <typename T>
__device__ __forceinline__ uint4 values8(uint32_t w, float2 f) {
  float x[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    // 1024 + code as fp16 numbers, codes j and j + 4; less 1024
    const uint32_t u = ((w >> (4 * j)) & 0x000f000fu) | 0x64006400u;
    const float2 c = __half22float2(__hsub2(*reinterpret_cast<const __half2*>(&u), __half2half2(__ushort_as_half(0x6400))));
    x[j] = fmaf(c.x, f.x, f.y);
    x[j + 4] = fmaf(c.y, f.x, f.y);
  }
  return make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
}

// D / 16 lanes a row, eight elements of each half of it a lane; ROWS rows of K and V a thread, whose loads are under way together.  Bound by the bytes written: 2 x 8322
// rows, 32 heads x 64, from 4 bits: 30 to 31 us, 5.6 to 5.9 TB/s.
template <typename T, int D, int BITS>
__global__ void __launch_bounds__(256) paged_gather_kernel(const GatherArgs a) {
  chain_begin();
  constexpr int LANES = D / 16, PER = 256 / LANES, ROWS = 2, G = D / PAGED_GROUP;
  const int lane = threadIdx.x % LANES;
  const int bh = a.by_blocks((int)blockIdx.x), b = a.by_heads(bh), h = bh - b * a.Hk;
  const int blocks = (a.rows + PER * ROWS - 1) / (PER * ROWS);
  const int first = (blockIdx.x - bh * blocks) * PER * ROWS + threadIdx.x / LANES;
  int len = a.c.lengths[b];
  if (len > a.c.capacity) {
    if (threadIdx.x == 0) report_status(a.c.status, a.c.status_host, HA_DEV_BAD_INDEX);
    len = a.c.capacity;
  }
  uint4 w[2][ROWS][2];          // 16 bits: the elements; 4 bits: two words, then their scales
#pragma unroll
  for (int u = 0; u < ROWS; ++u) {
    const int r = first + u * PER;
    int row = 0, page = -1;
    if (r < len && r < a.rows) page = paged_slot(a.c, b, r, row);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      w[s][u][0] = w[s][u][1] = make_uint4(0, 0, 0, 0);
      if (page < 0) continue;
      const uint8_t* src = (s ? a.c.v : a.c.k) + page * a.c.sp + h * a.c.sh + row * a.c.st;
      if (BITS == 16) {
        w[s][u][0] = *reinterpret_cast<const uint4*>(src + lane * 16);
        w[s][u][1] = *reinterpret_cast<const uint4*>(src + D + lane * 16);
      } else {
        const uint8_t* sc = (s ? a.c.vs : a.c.ks) + page * a.c.ssp + h * a.c.ssh + row * a.c.sst;
        if (G == 2) {
          const uint2 c = *reinterpret_cast<const uint2*>(src + 8 * lane);
          w[s][u][0].x = c.x;
          w[s][u][0].y = c.y;
        } else {
          w[s][u][0].x = *reinterpret_cast<const uint32_t*>(src + 4 * lane);
          w[s][u][0].y = *reinterpret_cast<const uint32_t*>(src + 16 + 4 * lane);
        }
        w[s][u][0].z = *reinterpret_cast<const uint32_t*>(sc);
        if (G == 2) w[s][u][0].w = *reinterpret_cast<const uint32_t*>(sc + 4);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < ROWS; ++u) {
    const int r = first + u * PER;
    if (r >= a.rows) continue;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      T* dst = (T*)(s ? a.v_out : a.k_out) + ((int64_t)bh * a.rows + r) * D;
      if (BITS == 16) {
        *reinterpret_cast<uint4*>(dst + lane * 8) = w[s][u][0];
        *reinterpret_cast<uint4*>(dst + D / 2 + lane * 8) = w[s][u][1];
      } else {
        const uint4 c = w[s][u][0];
        const float2 f0 = unpack2<__half>(c.z), f1 = unpack2<__half>(G == 2 ? c.w : c.z);
        *reinterpret_cast<uint4*>(dst + lane * 8) = values8<T>(c.x, f0);
        *reinterpret_cast<uint4*>(dst + D / 2 + lane * 8) = values8<T>(c.y, f1);
      }
    }
  }
}

template <typename T, int D, int BITS, int THREADS>
static void launch_append_block(const AppendArgs& a, bool wide, unsigned grid, cudaStream_t st) {
  if (wide) launch_chained(paged_append_kernel<T, D, BITS, true, THREADS>, grid, THREADS, 0, st, a);
  else launch_chained(paged_append_kernel<T, D, BITS, false, THREADS>, grid, THREADS, 0, st, a);
}
// Threads of a block, which takes a token.  Fewer make more tokens resident, whose chains hide one another: 64 where there are more tokens than blocks of 128 are resident
// (five an SM), or 32 where the query rows are few, too.  32768 tokens, 32 + 2 + 2 heads x 128: 107.7 us by 128 threads, 97.8 by 64, 102.1 by 32; 55656 tokens, 12 + 2 + 2
// heads: 127.7, 87.8, 75.3; 2 x 8191 tokens into 4 bits, 32 + 32 + 32 heads x 64, and back: 122.9, 109.8, 107.5; 32 tokens: 2.4, 2.9, 3.8.
template <typename T, int D, int BITS>
static int launch_append(const AppendArgs& a, bool wide, cudaStream_t st) {
  const int64_t sms = sm_count(), most = sms * 512;
  const unsigned grid = (unsigned)(a.tokens < most ? a.tokens : most);
  if (a.tokens <= 5 * sms) launch_append_block<T, D, BITS, 128>(a, wide, grid, st);
  else if (a.H * (D / PART) > 128) launch_append_block<T, D, BITS, 64>(a, wide, grid, st);
  else launch_append_block<T, D, BITS, 32>(a, wide, grid, st);
  HA_LAUNCHED("ha_paged_append");
  return HA_OK;
}
template <typename T, int D, int BITS>
static int launch_gather(const GatherArgs& a, unsigned grid, cudaStream_t st) {
  launch_chained(paged_gather_kernel<T, D, BITS>, grid, 256, 0, st, a);
  HA_LAUNCHED("ha_paged_gather");
  return HA_OK;
}

#define HA_PAGED_DISPATCH(fn, ...)                                                                      \
  do {                                                                                                  \
    if (p.dtype == HA_BF16) {                                                                           \
      if (p.d == 64) return p.bits == 16 ? fn<__nv_bfloat16, 64, 16>(__VA_ARGS__) : fn<__nv_bfloat16, 64, 4>(__VA_ARGS__);    \
      return p.bits == 16 ? fn<__nv_bfloat16, 128, 16>(__VA_ARGS__) : fn<__nv_bfloat16, 128, 4>(__VA_ARGS__);                 \
    }                                                                                                   \
    if (p.d == 64) return p.bits == 16 ? fn<__half, 64, 16>(__VA_ARGS__) : fn<__half, 64, 4>(__VA_ARGS__); \
    return p.bits == 16 ? fn<__half, 128, 16>(__VA_ARGS__) : fn<__half, 128, 4>(__VA_ARGS__);           \
  } while (0)

}  // namespace ha

using namespace ha;

extern "C" {

int ha_paged_append(const ha_paged_params* pp, void* stream) {
  if (!pp) return HA_ERR_INVALID;
  const ha_paged_params& p = *pp;
  const int rc = paged_check(p);
  if (rc != HA_OK) return rc;
  if (p.rope && (p.rot < 0 || p.rot > p.d || p.rot % 2 != 0 || p.rope_rows < 0 || (p.rope_dtype != HA_FP32 && p.rope_dtype != p.dtype))) return HA_ERR_INVALID;
  const int64_t tokens = (int64_t)p.B * p.n;
  if (tokens == 0) return HA_OK;
  if (tokens > 0x7fffffffLL || (int64_t)p.H + 2 * (int64_t)p.Hk > 1 << 20) return HA_ERR_TOO_LARGE;
  if (!p.k || !p.v || (p.q_out && !p.q) || (p.q && !p.q_out)) return HA_ERR_INVALID;
  if (((uintptr_t)p.q_out | (uintptr_t)p.k_out) % 16 != 0) return HA_ERR_INVALID;
  AppendArgs a = {};
  a.c = paged_view(p);
  a.q = p.q; a.k = p.k; a.v = p.v;
  a.q_sb = p.q_sb; a.q_sn = p.q_sn; a.q_sh = p.q_sh;
  a.k_sb = p.k_sb; a.k_sn = p.k_sn; a.k_sh = p.k_sh;
  a.v_sb = p.v_sb; a.v_sn = p.v_sn; a.v_sh = p.v_sh;
  a.rope = p.rope; a.rot = p.rope ? p.rot : 0; a.rope_rows = p.rope_rows; a.rope_f32 = p.rope_dtype == HA_FP32;
  a.rope_wide = a.rot % 16 == 0 && (uintptr_t)p.rope % 16 == 0;
  a.n = p.n; a.H = p.q ? p.H : 0; a.Hk = p.Hk;
  a.tokens = tokens; a.by_n = FastDiv((uint32_t)p.n);
  a.q_out = p.q_out; a.k_out = p.k_out;
  bool wide = (((uintptr_t)p.k | (uintptr_t)p.v) % 16 == 0) && ((p.k_sb | p.k_sn | p.k_sh | p.v_sb | p.v_sn | p.v_sh) % 8 == 0);
  if (p.q) wide = wide && (uintptr_t)p.q % 16 == 0 && (p.q_sb | p.q_sn | p.q_sh) % 8 == 0;
  HA_PAGED_DISPATCH(launch_append, a, wide, (cudaStream_t)stream);
}

int ha_paged_gather(const ha_paged_params* pp, void* stream) {
  if (!pp) return HA_ERR_INVALID;
  const ha_paged_params& p = *pp;
  const int rc = paged_check(p);
  if (rc != HA_OK) return rc;
  if (p.rows < 0) return HA_ERR_INVALID;
  const int per = 256 / (p.d / 16) * 2;          // rows of a block
  const int64_t blocks = ((int64_t)p.rows + per - 1) / per, grid = blocks * p.B * p.Hk;
  if (grid == 0) return HA_OK;
  if (grid > 0x7fffffffLL) return HA_ERR_TOO_LARGE;
  if (!p.k_out || !p.v_out || ((uintptr_t)p.k_out | (uintptr_t)p.v_out) % 16 != 0) return HA_ERR_INVALID;
  GatherArgs a = {};
  a.c = paged_view(p);
  a.Hk = p.Hk; a.rows = p.rows;
  a.by_blocks = FastDiv((uint32_t)blocks); a.by_heads = FastDiv((uint32_t)p.Hk);
  a.k_out = p.k_out; a.v_out = p.v_out;
  HA_PAGED_DISPATCH(launch_gather, a, (unsigned)grid, (cudaStream_t)stream);
}

}  // extern "C"
