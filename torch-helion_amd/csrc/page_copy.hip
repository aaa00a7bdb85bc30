// th_page_copy: pages of a KV cache copied to other pages in every layer, and
// page tables renamed after a move (forks and compaction of a paged cache; no
// counterpart in the reference, which has no cache).
//
// HBM bound: each byte is read once and written once. One workgroup moves one
// 32 KiB piece of one page of one tensor of one layer: eight 16-byte loads a
// lane, then the stores, both past the caches (nothing is used twice). 683 pages
// of 64 KiB in 8 layers of both caches, 1.43 GB: 266 us, 5.39 TB/s (282 us with
// 16 KiB pieces through the caches, 277 with the stores alone past them; a large
// device copy reaches 4.95 TB/s).
#include "common.h"

namespace th {

struct PageCopyK {
  char* kc; int64_t kl, kp;  // byte strides: layer, page
  char* vc; int64_t vl, vp;
  const int32_t* src;
  const int32_t* dst;
  int32_t* table; int64_t ldt;
  const int32_t* map;
  int64_t pages, bytes, table_entries;
  int n, layers, pieces, row_pages, copy_blocks;
};

constexpr int kPiece = 32768;

__global__ void __launch_bounds__(256) page_copy_kernel(PageCopyK p) {
  int64_t b = grid_index();
  if (b >= p.copy_blocks) {  // the workgroups past the copies rename the table
    const int64_t e = (b - p.copy_blocks) * 256 + threadIdx.x;
    if (e >= p.table_entries) return;
    int32_t* at = p.table + (e / p.row_pages) * p.ldt + e % p.row_pages;
    const int32_t page = *at;
    if (page >= 0 && page < p.pages) *at = p.map[page];
    return;
  }
  const int piece = b % p.pieces;
  b /= p.pieces;
  const int v = b & 1;
  b >>= 1;
  const int layer = b % p.layers, i = b / p.layers;
  const int64_t src = p.src[i], dst = p.dst[i];
  if (src < 0 || src >= p.pages || dst < 0 || dst >= p.pages || src == dst) return;
  char* base = (v ? p.vc + layer * p.vl : p.kc + layer * p.kl) + (int64_t)piece * kPiece;
  const int64_t stride = v ? p.vp : p.kp;
  const char* from = base + src * stride;
  char* to = base + dst * stride;
  const int n = (int)min((int64_t)kPiece, p.bytes - (int64_t)piece * kPiece);
  // buffer accesses: past n bytes a load is zero and a store is dropped
  typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
  constexpr int kNt = 2;  // cache policy: non-temporal
  const auto rf = __builtin_amdgcn_make_buffer_rsrc((void*)from, 0, n, 0x00020000);
  const auto rt = __builtin_amdgcn_make_buffer_rsrc((void*)to, 0, n, 0x00020000);
  u32x4 x[kPiece / 4096];
#pragma unroll
  for (int i = 0; i < kPiece / 4096; ++i)
    x[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rf, threadIdx.x * 16 + i * 4096, 0, kNt));
#pragma unroll
  for (int i = 0; i < kPiece / 4096; ++i)
    __builtin_amdgcn_raw_buffer_store_b128(x[i], rt, threadIdx.x * 16 + i * 4096, 0, kNt);
}

}  // namespace th

using namespace th;

extern "C" int th_page_copy(const th_page_copy_desc* d, void* stream) {
  TH_CHECK_ARG(d != nullptr, "th_page_copy: null descriptor");
  TH_CHECK_ARG(d->layers > 0 && d->n >= 0 && d->pages > 0 && d->page_bytes > 0, "th_page_copy: bad sizes");
  TH_CHECK_ARG(d->page_bytes % 16 == 0 && d->k_layer_bytes % 16 == 0 && d->v_layer_bytes % 16 == 0 &&
                   d->k_page_bytes % 16 == 0 && d->v_page_bytes % 16 == 0 &&
                   (((uintptr_t)d->k_cache | (uintptr_t)d->v_cache) & 15) == 0,
               "th_page_copy: pages must be 16-byte aligned and a multiple of 16 bytes");
  TH_CHECK_ARG(d->pages == 1 || (d->k_page_bytes >= d->page_bytes && d->v_page_bytes >= d->page_bytes),
               "th_page_copy: page stride < page_bytes");
  TH_CHECK_ARG(d->layers == 1 || (d->k_layer_bytes > 0 && d->v_layer_bytes > 0), "th_page_copy: bad layer stride");
  TH_CHECK_ARG(!d->page_table || (d->page_map && d->n_rows > 0 && d->row_pages > 0 && d->ld_page_table >= d->row_pages),
               "th_page_copy: a page table needs its sizes and page_map");
  if (d->n == 0 && !d->page_table) return TH_OK;
  TH_CHECK_ARG(d->n == 0 || (d->k_cache && d->v_cache && d->src && d->dst), "th_page_copy: null operand");
  const int64_t pieces = cdiv(d->page_bytes, kPiece);
  const int64_t copies = pieces * 2 * d->layers * d->n;
  const int64_t entries = d->page_table ? (int64_t)d->n_rows * d->row_pages : 0;
  const int64_t blocks = copies + cdiv(entries, 256);
  TH_CHECK_ARG(blocks < (int64_t)1 << 31, "th_page_copy: %lld workgroups exceed one launch", (long long)blocks);
  if (!device_ready()) {
    set_error("th_page_copy: th_init was not called for the current device");
    return TH_ERR_NOT_INIT;
  }
  PageCopyK k{};
  k.kc = (char*)d->k_cache; k.kl = d->k_layer_bytes; k.kp = d->k_page_bytes;
  k.vc = (char*)d->v_cache; k.vl = d->v_layer_bytes; k.vp = d->v_page_bytes;
  k.src = d->src; k.dst = d->dst; k.table = d->page_table; k.ldt = d->ld_page_table; k.map = d->page_map;
  k.pages = d->pages; k.bytes = d->page_bytes;
  k.n = d->n; k.layers = d->layers; k.row_pages = d->row_pages;
  k.pieces = (int)pieces;
  k.table_entries = entries;
  k.copy_blocks = (int)copies;
  hipLaunchKernelGGL(page_copy_kernel, grid_of(blocks), dim3(256), 0, (hipStream_t)stream, k);
  TH_CHECK_LAUNCH();
  return TH_OK;
}
