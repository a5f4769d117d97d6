// Writing rows to the paged key/value cache (position rotation and 4-bit coding on the way) and reading them back as dense tensors.
#include "paged.cuh"

namespace ha {

// eight neighbouring elements of a row in 32 bits
template <typename T, bool WIDE>
__device__ __forceinline__ void load8(const T* src, float (&x)[8]) {
  if (WIDE) {
    const uint4 w = *reinterpret_cast<const uint4*>(src);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack2<T>(u[i]);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f32<T>(src[i]);
  }
}
template <typename T>
__device__ __forceinline__ void store8(void* dst, const float (&x)[8]) {
  *reinterpret_cast<uint4*>(dst) = make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
}

struct AppendArgs {
  PagedView c;
  const void *q, *k, *v;
  int64_t q_sb, q_sn, q_sh, k_sb, k_sn, k_sh, v_sb, v_sn, v_sh;
  const void* rope;
  int32_t n, H, Hk, rot, rope_rows, rope_f32;
  int64_t tokens;
  FastDiv by_n;
  void *q_out, *k_out;
};

// One block a token, D / 8 lanes a row, eight elements a lane: a lane keeps its cosines and sines for all the heads of the token that it meets.
// Bound by the bytes of q, k and v for prompts, by the chain length -> page -> store for single tokens.
// The rotation's products and sums are rounded one by one (no fused multiply-add), so that its results, and with them the 4-bit codes, are
// those of the formula in 32 bits, whoever evaluates it.
template <typename T, int D, int BITS, bool WIDE>
__global__ void __launch_bounds__(128) paged_append_kernel(const AppendArgs a) {
  chain_begin();
  constexpr int LANES = D / 8, GROUPS = 128 / LANES, UNROLL = 4;
  const int lane = threadIdx.x % LANES, grp = threadIdx.x / LANES;
  const int tasks = a.H + 2 * a.Hk;
  for (int64_t tok = blockIdx.x; tok < a.tokens; tok += gridDim.x) {
    const int b = a.by_n((int)tok), i = (int)(tok - (int64_t)b * a.n);
    const int len = a.c.lengths[b];
    const bool live = i < (a.c.counts ? a.c.counts[b] : a.n);
    const bool ok = live && len >= 0 && len < a.c.capacity - i && (!a.rope || len < a.rope_rows - i);
    const int pos = ok ? len + i : 0;
    if (live && !ok && threadIdx.x == 0) report_status(a.c.status, a.c.status_host, HA_DEV_BAD_INDEX);
    int row = 0, page = -1;
    if (ok) page = paged_slot(a.c, b, pos, row);
    float cs[4], sn[4];                        // of this lane's four pairs
    int turned = 0;                            // pairs of them that are rotated
    if (a.rope && ok) {
      const int pairs = a.rot / 2 - lane * 4;
      turned = pairs < 0 ? 0 : pairs > 4 ? 4 : pairs;
      const int64_t at = ((int64_t)pos * (a.rot / 2) + lane * 4) * 2;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < turned) {
          cs[j] = a.rope_f32 ? ((const float*)a.rope)[at + 2 * j] : to_f32<T>(((const T*)a.rope)[at + 2 * j]);
          sn[j] = a.rope_f32 ? ((const float*)a.rope)[at + 2 * j + 1] : to_f32<T>(((const T*)a.rope)[at + 2 * j + 1]);
        }
    }
    for (int first = 0; first < tasks; first += GROUPS * UNROLL) {
      float x[UNROLL][8];
      // task: query heads, then key heads, then value heads
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        const int t = first + u * GROUPS + grp;
        const T* src = nullptr;
        if (t < a.H) src = a.q ? (const T*)a.q + b * a.q_sb + i * a.q_sn + t * a.q_sh : nullptr;
        else if (t < a.H + a.Hk) src = (const T*)a.k + b * a.k_sb + i * a.k_sn + (t - a.H) * a.k_sh;
        else if (t < tasks) src = (const T*)a.v + b * a.v_sb + i * a.v_sn + (t - a.H - a.Hk) * a.v_sh;
        if (src && live) load8<T, WIDE>(src + lane * 8, x[u]);
        else
#pragma unroll
          for (int j = 0; j < 8; ++j) x[u][j] = 0.f;
      }
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        const int t = first + u * GROUPS + grp;
        const bool is_q = t < a.H, is_v = t >= a.H + a.Hk;
        const int h = is_q ? t : is_v ? t - a.H - a.Hk : t - a.H;
        if (!is_v)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (j < turned) {
              const float x0 = x[u][2 * j], x1 = x[u][2 * j + 1];
              x[u][2 * j] = __fsub_rn(__fmul_rn(x0, cs[j]), __fmul_rn(x1, sn[j]));
              x[u][2 * j + 1] = __fadd_rn(__fmul_rn(x1, cs[j]), __fmul_rn(x0, sn[j]));
            }
        if (is_q) {
          if (a.q_out) store8<T>((T*)a.q_out + (tok * a.H + h) * D + lane * 8, x[u]);
        } else if (!is_v && t < tasks && a.k_out) {
          store8<T>((T*)a.k_out + (tok * a.Hk + h) * D + lane * 8, x[u]);
        }
        if (BITS == 16) {
          if (!is_q && t < tasks && page >= 0)
            store8<T>((is_v ? a.c.v : a.c.k) + page * a.c.sp + h * a.c.sh + row * a.c.st + lane * 16, x[u]);
        } else {
          // extremes of the 64 elements that eight neighbouring lanes hold; a NaN among them stays one
          float lo = x[u][0], hi = x[u][0];
#pragma unroll
          for (int j = 1; j < 8; ++j) {
            hi = max_nan(hi, x[u][j]);
            lo = -max_nan(-lo, -x[u][j]);
          }
#pragma unroll
          for (int s = 1; s < 8; s *= 2) {
            hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, s));
            lo = -max_nan(-lo, -__shfl_xor_sync(0xffffffffu, lo, s));
          }
          __half s16 = __float2half_rn(__fdiv_rn(__fsub_rn(hi, lo), 15.f)), m16 = __float2half_rn(lo);
          if (__hisinf(s16) || __hisnan(s16) || __hisinf(m16) || __hisnan(m16)) {
            s16 = __ushort_as_half(0);
            m16 = __ushort_as_half(0x7fff);
          }
          const float s = __half2float(s16), m = __half2float(m16);
          uint32_t word = 0;
          if (s > 0.f)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float c = fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(x[u][j], m), s)), 0.f), 15.f);
              word |= (uint32_t)(int)c << (4 * j);
            }
          if (!is_q && t < tasks && page >= 0) {
            const int g = lane / 8, w = (lane % 8) * (D / PAGED_GROUP) + g;
            uint8_t* dst = (is_v ? a.c.v : a.c.k) + page * a.c.sp + h * a.c.sh + row * a.c.st;
            *reinterpret_cast<uint32_t*>(dst + 4 * w) = word;
            if (lane % 8 == 0) {
              uint8_t* sc = (is_v ? a.c.vs : a.c.ks) + page * a.c.ssp + h * a.c.ssh + row * a.c.sst;
              *reinterpret_cast<__half2*>(sc + 4 * g) = __halves2half2(s16, m16);
            }
          }
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

// D / 8 lanes a row, ROWS rows of K and V a thread: their loads are under way together.  Bound by the bytes written.
template <typename T, int D, int BITS>
__global__ void __launch_bounds__(256) paged_gather_kernel(const GatherArgs a) {
  chain_begin();
  constexpr int LANES = D / 8, PER = 256 / LANES, ROWS = 4;
  const int lane = threadIdx.x % LANES;
  const int bh = a.by_blocks((int)blockIdx.x), b = a.by_heads(bh), h = bh - b * a.Hk;
  const int blocks = (a.rows + PER * ROWS - 1) / (PER * ROWS);
  const int first = (blockIdx.x - bh * blocks) * PER * ROWS + threadIdx.x / LANES;
  int len = a.c.lengths[b];
  if (len > a.c.capacity) {
    if (threadIdx.x == 0) report_status(a.c.status, a.c.status_host, HA_DEV_BAD_INDEX);
    len = a.c.capacity;
  }
  uint4 w[2][ROWS];
  uint32_t sc[2][ROWS];
#pragma unroll
  for (int u = 0; u < ROWS; ++u) {
    const int r = first + u * PER;
    int row = 0, page = -1;
    if (r < len && r < a.rows) page = paged_slot(a.c, b, r, row);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      w[s][u] = make_uint4(0, 0, 0, 0);
      sc[s][u] = 0;
      if (page < 0) continue;
      const uint8_t* src = (s ? a.c.v : a.c.k) + page * a.c.sp + h * a.c.sh + row * a.c.st;
      if (BITS == 16) {
        w[s][u] = *reinterpret_cast<const uint4*>(src + lane * 16);
      } else {
        const int g = lane / 8;
        w[s][u].x = *reinterpret_cast<const uint32_t*>(src + 4 * ((lane % 8) * (D / PAGED_GROUP) + g));
        sc[s][u] = *reinterpret_cast<const uint32_t*>((s ? a.c.vs : a.c.ks) + page * a.c.ssp + h * a.c.ssh + row * a.c.sst + 4 * g);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < ROWS; ++u) {
    const int r = first + u * PER;
    if (r >= a.rows) continue;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      T* dst = (T*)(s ? a.v_out : a.k_out) + ((int64_t)bh * a.rows + r) * D + lane * 8;
      if (BITS == 16) {
        *reinterpret_cast<uint4*>(dst) = w[s][u];
      } else {
        // code * step is exact in 32 bits (4 and 11 bits), so that the sum is the value's one rounding before T's
        const float2 f = unpack2<__half>(sc[s][u]);
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = fmaf((float)((w[s][u].x >> (4 * j)) & 15u), f.x, f.y);
        store8<T>(dst, x);
      }
    }
  }
}

template <typename T, int D, int BITS>
static int launch_append(const AppendArgs& a, bool wide, cudaStream_t st) {
  const int64_t most = (int64_t)sm_count() * 512;
  const unsigned grid = (unsigned)(a.tokens < most ? a.tokens : most);
  if (wide) launch_chained(paged_append_kernel<T, D, BITS, true>, grid, 128, 0, st, a);
  else launch_chained(paged_append_kernel<T, D, BITS, false>, grid, 128, 0, st, a);
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
  const int per = 256 / (p.d / 8) * 4;
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
