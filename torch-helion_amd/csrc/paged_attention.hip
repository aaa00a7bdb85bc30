// th_paged_attention: attention of one query per token over a paged KV cache.
#include "common.h"

#include <math.h>

namespace th {

struct PAttnK {
  const uint16_t* q; int64_t ldq;
  const void* k; int64_t kp, kt, kh;  // element strides: page, token, head
  const void* v; int64_t vp, vt, vh;
  uint16_t* o; int64_t ldo;
  const int32_t* positions;
  const int32_t* rows;
  const int32_t* table; int64_t ldt;
  int64_t pages;
  int n_rows, row_pages, pshift;
  int tokens, Hq, Hkv, G;
  int window;
  float scale, softcap;
  const float* slopes;
  const float* ks;
  const float* vs;
};

__device__ __forceinline__ float cache_elem(const void* c, int64_t i, bool e4m3) {
  if (e4m3) return __builtin_amdgcn_cvt_f32_fp8(((const uint8_t*)c)[i], 0);
  return bf16_to_f32(((const uint16_t*)c)[i]);
}

// The simple form: one workgroup per (token, query head), a key per wave step.
template <int D, bool E4>
__global__ void __launch_bounds__(256) paged_attn_simple_kernel(PAttnK p) {
  constexpr int R = D / 64;
  __shared__ float om[4][D], mm[4], lm[4];
  const int t = blockIdx.y, h = blockIdx.x, kvh = h / p.G;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t pos = p.positions[t];
  const int row = p.rows ? p.rows[t] : t;
  int64_t hi = min(pos + 1, (int64_t)p.row_pages << p.pshift), lo = 0;
  if (p.window) lo = max((int64_t)0, pos + 1 - p.window);
  if (row < 0 || row >= p.n_rows) hi = 0;
  float q[R], o[R], m = -INFINITY, l = 0.f;
  const float mul = p.scale * (p.ks ? p.ks[kvh] : 1.f);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    q[r] = bf16_to_f32(p.q[t * p.ldq + h * D + R * lane + r]) * mul;
    o[r] = 0.f;
  }
  for (int64_t j = lo + wave; j < hi; j += 4) {
    const int64_t page = p.table[row * p.ldt + (j >> p.pshift)], slot = j & ((1 << p.pshift) - 1);
    if (page < 0 || page >= p.pages) continue;
    float s = 0.f;
#pragma unroll
    for (int r = 0; r < R; ++r) s += q[r] * cache_elem(p.k, page * p.kp + slot * p.kt + kvh * p.kh + R * lane + r, E4);
#pragma unroll
    for (int x = 32; x; x >>= 1) s += __shfl_xor(s, x);
    if (p.softcap > 0.f) s = p.softcap * tanhf(s / p.softcap);
    if (p.slopes) s -= p.slopes[h] * (float)(pos - j);
    const float mn = fmaxf(m, s), mu = mn == -INFINITY ? 0.f : mn;
    const float a = expf(m - mu), e = expf(s - mu);
    m = mn;
    l = l * a + e;
#pragma unroll
    for (int r = 0; r < R; ++r)
      o[r] = o[r] * a + e * cache_elem(p.v, page * p.vp + slot * p.vt + kvh * p.vh + R * lane + r, E4);
  }
#pragma unroll
  for (int r = 0; r < R; ++r) om[wave][R * lane + r] = o[r];
  if (lane == 0) { mm[wave] = m; lm[wave] = l; }
  __syncthreads();
  for (int d = threadIdx.x; d < D; d += 256) {
    float mx = -INFINITY, ll = 0.f, oo = 0.f;
    for (int w = 0; w < 4; ++w) mx = fmaxf(mx, mm[w]);
    const float mu = mx == -INFINITY ? 0.f : mx;
    for (int w = 0; w < 4; ++w) {
      const float f = expf(mm[w] - mu);
      ll += lm[w] * f;
      oo += om[w][d] * f;
    }
    p.o[t * p.ldo + h * D + d] = f32_to_bf16(ll == 0.f ? 0.f : oo / ll * (p.vs ? p.vs[kvh] : 1.f));
  }
}

}  // namespace th

using namespace th;

extern "C" int64_t th_paged_attention_workspace_bytes(int32_t tokens, int32_t heads_q, int32_t heads_kv, int32_t head_dim) {
  if (tokens < 0 || heads_q <= 0 || heads_kv <= 0 || heads_q % heads_kv || (head_dim != 64 && head_dim != 128)) return -1;
  return 0;
}

extern "C" int th_paged_attention(const th_paged_attn_desc* d, void* stream) {
  TH_CHECK_ARG(d != nullptr, "th_paged_attention: null descriptor");
  TH_CHECK_ARG(d->tokens >= 0 && d->tokens <= 65535, "th_paged_attention: tokens %d out of range", d->tokens);
  TH_CHECK_ARG(d->heads_q > 0 && d->heads_kv > 0 && d->heads_q % d->heads_kv == 0,
               "th_paged_attention: heads_q=%d must be a multiple of heads_kv=%d", d->heads_q, d->heads_kv);
  TH_CHECK_ARG(d->head_dim == 64 || d->head_dim == 128, "th_paged_attention: head_dim %d unsupported", d->head_dim);
  TH_CHECK_ARG(d->cache_dtype == TH_BF16 || d->cache_dtype == TH_F8E4M3, "th_paged_attention: cache_dtype %d unsupported",
               d->cache_dtype);
  TH_CHECK_ARG(d->page_size >= 16 && (d->page_size & (d->page_size - 1)) == 0,
               "th_paged_attention: page_size %d must be a power of two of at least 16", d->page_size);
  TH_CHECK_ARG(d->n_rows > 0 && d->row_pages > 0 && d->pages > 0 && d->ld_page_table >= d->row_pages,
               "th_paged_attention: bad page table sizes");
  TH_CHECK_ARG((int64_t)d->row_pages * d->page_size < (int64_t)1 << 31, "th_paged_attention: row of 2^31 keys or more");
  TH_CHECK_ARG(d->window >= 0 && d->softcap >= 0.f, "th_paged_attention: window and softcap must not be negative");
  const int64_t row = (int64_t)d->heads_q * d->head_dim;
  TH_CHECK_ARG(d->ld_q >= row && d->ld_o >= row, "th_paged_attention: q/o row strides smaller than heads_q*head_dim");
  const int per = d->cache_dtype == TH_BF16 ? 8 : 16;  // elements in 16 bytes
  TH_CHECK_ARG(d->k_stride_h >= d->head_dim && d->v_stride_h >= d->head_dim && d->k_stride_t >= d->head_dim &&
                   d->v_stride_t >= d->head_dim && d->k_stride_page >= d->head_dim && d->v_stride_page >= d->head_dim,
               "th_paged_attention: cache stride < head_dim");
  TH_CHECK_ARG(d->ld_q % 8 == 0 && d->k_stride_h % per == 0 && d->v_stride_h % per == 0 && d->k_stride_t % per == 0 &&
                   d->v_stride_t % per == 0 && d->k_stride_page % per == 0 && d->v_stride_page % per == 0,
               "th_paged_attention: q and cache strides must be multiples of 16 bytes");
  TH_CHECK_ARG(d->k_stride_t < (1 << 22) && d->v_stride_t < (1 << 22) &&
                   d->k_stride_t * d->page_size < (int64_t)1 << 30 && d->v_stride_t * d->page_size < (int64_t)1 << 30,
               "th_paged_attention: token strides must be under 2^22 elements and 2^30 per page");
  TH_CHECK_ARG((((uintptr_t)d->q | (uintptr_t)d->k_cache | (uintptr_t)d->v_cache) & 15) == 0,
               "th_paged_attention: q and caches must be 16-byte aligned");
  TH_CHECK_ARG((!d->k_scale && !d->v_scale) || d->cache_dtype == TH_F8E4M3,
               "th_paged_attention: scales need an e4m3 cache");
  if (d->tokens == 0) return TH_OK;
  TH_CHECK_ARG(d->rows || d->tokens <= d->n_rows, "th_paged_attention: %d tokens without rows exceed the table's %d",
               d->tokens, d->n_rows);
  TH_CHECK_ARG(d->q && d->k_cache && d->v_cache && d->o && d->positions && d->page_table,
               "th_paged_attention: null tensor pointer");
  const int64_t need = th_paged_attention_workspace_bytes(d->tokens, d->heads_q, d->heads_kv, d->head_dim);
  TH_CHECK_ARG(need == 0 || (d->workspace && ((uintptr_t)d->workspace & 15) == 0 && d->workspace_bytes >= need),
               "th_paged_attention: workspace %lld < %lld bytes, or not 16-byte aligned", (long long)d->workspace_bytes,
               (long long)need);
  if (!device_ready()) {
    set_error("th_paged_attention: th_init was not called for the current device");
    return TH_ERR_NOT_INIT;
  }
  PAttnK k{};
  k.q = (const uint16_t*)d->q; k.ldq = d->ld_q;
  k.k = d->k_cache; k.kp = d->k_stride_page; k.kt = d->k_stride_t; k.kh = d->k_stride_h;
  k.v = d->v_cache; k.vp = d->v_stride_page; k.vt = d->v_stride_t; k.vh = d->v_stride_h;
  k.o = (uint16_t*)d->o; k.ldo = d->ld_o;
  k.positions = d->positions; k.rows = d->rows; k.table = d->page_table; k.ldt = d->ld_page_table; k.pages = d->pages;
  k.n_rows = d->n_rows; k.row_pages = d->row_pages; k.pshift = __builtin_ctz((unsigned)d->page_size);
  k.tokens = d->tokens; k.Hq = d->heads_q; k.Hkv = d->heads_kv; k.G = d->heads_q / d->heads_kv;
  k.window = d->window; k.scale = d->scale; k.softcap = d->softcap;
  k.slopes = d->slopes; k.ks = d->k_scale; k.vs = d->v_scale;
  const dim3 grid(d->heads_q, d->tokens);
  hipStream_t s = (hipStream_t)stream;
  const bool e4 = d->cache_dtype == TH_F8E4M3;
  if (d->head_dim == 128) {
    if (e4) hipLaunchKernelGGL((paged_attn_simple_kernel<128, true>), grid, dim3(256), 0, s, k);
    else hipLaunchKernelGGL((paged_attn_simple_kernel<128, false>), grid, dim3(256), 0, s, k);
  } else {
    if (e4) hipLaunchKernelGGL((paged_attn_simple_kernel<64, true>), grid, dim3(256), 0, s, k);
    else hipLaunchKernelGGL((paged_attn_simple_kernel<64, false>), grid, dim3(256), 0, s, k);
  }
  TH_CHECK_LAUNCH();
  return TH_OK;
}
