// Shared by the kernels of the paged key/value cache: argument checks, and where a token's row lies.
#pragma once
#include "common.cuh"

namespace ha {

constexpr int PAGED_GROUP = 64;      // elements that share a scale in a 4-bit row
constexpr long long PAGED_MOST = 0x7fffffffLL - 65536;      // positions of a sequence: 32-bit numbers, with room for a tile behind the last

// What every entry point of the cache asks of its arguments.
inline int paged_check(const ha_paged_params& p) {
  if (p.dtype != HA_BF16 && p.dtype != HA_FP16) return HA_ERR_DTYPE;
  if ((p.bits != 16 && p.bits != 4) || (p.d != 64 && p.d != 128)) return HA_ERR_INVALID;
  if (p.B < 0 || p.n < 0 || p.Hk < 1 || p.H < 0 || p.H % p.Hk != 0) return HA_ERR_INVALID;
  if (p.pages < 0 || p.page_size < 1 || p.columns < 0 || p.table_sb < 0) return HA_ERR_INVALID;
  if ((long long)p.columns * p.page_size > PAGED_MOST) return HA_ERR_TOO_LARGE;
  if (p.page_sp < 0 || p.page_sh < 0 || p.page_st < 0 || p.scale_sp < 0 || p.scale_sh < 0 || p.scale_st < 0) return HA_ERR_INVALID;
  if (p.B > 0 && (!p.lengths || (p.columns > 0 && !p.table))) return HA_ERR_INVALID;
  if (p.pages > 0) {
    const int bytes = p.bits == 16 ? 2 : 1, sc = p.d / PAGED_GROUP * 4;
    if (!p.k_pages || !p.v_pages) return HA_ERR_INVALID;
    if (((uintptr_t)p.k_pages | (uintptr_t)p.v_pages) % 16 != 0) return HA_ERR_INVALID;
    if (((p.page_sp | p.page_sh | p.page_st) * bytes) % 16 != 0) return HA_ERR_INVALID;
    if (p.bits == 4) {
      if (!p.k_scales || !p.v_scales || ((uintptr_t)p.k_scales | (uintptr_t)p.v_scales) % sc != 0) return HA_ERR_INVALID;
      if (((p.scale_sp | p.scale_sh | p.scale_st) * 2) % sc != 0) return HA_ERR_INVALID;
    }
  }
  return HA_OK;
}

// The pool, the table and the lengths, as kernels take them.
struct PagedView {
  uint8_t *k, *v;                    // rows: 16-bit elements or packed codes; strides in bytes
  int64_t sp, sh, st;
  uint8_t *ks, *vs;                  // scales, strides in bytes
  int64_t ssp, ssh, sst;
  const int32_t* table;
  int64_t table_sb;
  const int32_t *lengths, *counts;
  int32_t pages, page_size, capacity;
  FastDiv by_page;
  int32_t *status, *status_host;
};

inline PagedView paged_view(const ha_paged_params& p) {
  PagedView v;
  const int bytes = p.bits == 16 ? 2 : 1;
  v.k = (uint8_t*)p.k_pages; v.v = (uint8_t*)p.v_pages;
  v.sp = p.page_sp * bytes; v.sh = p.page_sh * bytes; v.st = p.page_st * bytes;
  v.ks = (uint8_t*)p.k_scales; v.vs = (uint8_t*)p.v_scales;
  v.ssp = p.scale_sp * 2; v.ssh = p.scale_sh * 2; v.sst = p.scale_st * 2;
  v.table = p.table; v.table_sb = p.table_sb;
  v.lengths = p.lengths; v.counts = p.counts;
  v.pages = p.pages; v.page_size = p.page_size; v.capacity = p.columns * p.page_size;
  v.by_page = FastDiv((uint32_t)p.page_size);
  v.status = p.status; v.status_host = p.status_host;
  return v;
}

// The table's entry for position `pos` (0 <= pos < capacity) of sequence b, whatever it is, and the row within the page: the load alone, so that a kernel can
// look ahead; paged_checked when the page is used.
__device__ __forceinline__ int paged_entry(const PagedView& v, int b, int pos, int& row) {
  const int col = v.by_page(pos);
  row = pos - col * v.page_size;
  return v.table[b * v.table_sb + col];
}
__device__ __forceinline__ bool paged_checked(const PagedView& v, int page) {
  if ((unsigned)page < (unsigned)v.pages) return true;
  report_status(v.status, v.status_host, HA_DEV_BAD_INDEX);
  return false;
}
// Page and row within it of position `pos` (0 <= pos < capacity) of sequence b; page -1, and the failure reported, where the table names none.
__device__ __forceinline__ int paged_slot(const PagedView& v, int b, int pos, int& row) {
  const int page = paged_entry(v, b, pos, row);
  return paged_checked(v, page) ? page : -1;
}

}  // namespace ha
