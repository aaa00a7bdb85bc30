// th_rope and th_paged_append: rotary positions token by token, into a tensor
// or into the pages of a KV cache (no counterpart in the reference, whose
// tables hold positions 0..S-1, optimizer/param_transforms.py:47-51).
//
// A pair (a, b) of a head at position p turns by phi = p f_i:
//   a' = s (a cos phi - b sin phi),  b' = s (b cos phi + a sin phi).
// Angles: p f_i / 2 pi is formed and reduced to a fraction of a turn in 64
// bits (a float loses a whole turn's worth of it past a million positions) and
// only the fraction goes through a single-precision sincospi. One token's
// angles serve all its heads, so a workgroup computes them once, into LDS.
// Both kernels are HBM bound (three products per element read and written).
#include "common.h"

#include <math.h>

namespace th {

struct RopeK {
  const void* q; int64_t ldq;      // heads rotated into qo
  void* qo; int64_t ldqo;
  const void* k; int64_t ldk;      // heads rotated into k_cache
  const void* v; int64_t ldv;      // heads stored into v_cache
  const void* positions;
  const int32_t* rows;
  const double* freqs;
  float scale, sign;               // sign -1: the inverse rotation
  int hq, hkv, hd, half, interleaved;
  const int32_t* table; int64_t ldt;
  int n_rows, row_pages, pshift;
  int64_t pages;
  void* kc; int64_t kp, kt, kh;    // element strides of the caches: page, token, head
  void* vc; int64_t vp, vt, vh;
  const float* ks;
  const float* vs;
  int32_t* n_invalid;
};

constexpr int kMaxHeadDim = 1024;

// fraction of a turn of pair i at position pos, in [-1/2, 1/2]
__device__ __forceinline__ float rope_turn(const RopeK& p, int64_t pos, int i) {
  const double t = (double)pos * p.freqs[i] * 0.15915494309189533577;  // 1 / (2 pi)
  return (float)(t - rint(t));
}

__device__ __forceinline__ uint8_t f32_to_e4m3(float x) {
  // saturated at the largest finite value; NaN stays NaN (fminf would drop it)
  const float c = x != x ? x : fminf(fmaxf(x, -448.f), 448.f);
  return (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, c, 0, false);
}

__device__ __forceinline__ float load_as_f32(const float* p) { return *p; }
__device__ __forceinline__ float load_as_f32(const uint16_t* p) { return bf16_to_f32(*p); }
__device__ __forceinline__ void store_f32(float* p, float x) { *p = x; }
__device__ __forceinline__ void store_f32(uint16_t* p, float x) { *p = f32_to_bf16(x); }
__device__ __forceinline__ void store_f32(uint8_t* p, float x) { *p = f32_to_e4m3(x); }

// Where token t's keys and values go: the element offsets of its slot in the
// two caches, or false (its row, position or page lies outside).
__device__ __forceinline__ bool cache_slot(const RopeK& p, int64_t t, int64_t pos, int64_t& ko, int64_t& vo) {
  const int64_t row = p.rows ? p.rows[t] : t;
  const int64_t pi = pos >> p.pshift;
  if (row < 0 || row >= p.n_rows || pi >= p.row_pages) return false;
  const int64_t page = p.table[row * p.ldt + pi];
  if (page < 0 || page >= p.pages) return false;
  const int64_t slot = pos & ((1 << p.pshift) - 1);
  ko = page * p.kp + slot * p.kt;
  vo = page * p.vp + slot * p.vt;
  return true;
}

// One workgroup per token; each thread takes a pair (or an unrotated element)
// of a head at a time, so any head_dim, rot_dim, stride and alignment goes.
// APPEND: positions are int32, negative ones are skipped, k and v are stored.
template <typename PosT, typename InT, typename OutT, typename CacheT, bool APPEND>
__global__ void __launch_bounds__(256) rope_elem_kernel(RopeK p) {
  __shared__ float cs[kMaxHeadDim / 2], sn[kMaxHeadDim / 2];
  const int64_t t = blockIdx.x;
  const int64_t pos = ((const PosT*)p.positions)[t];
  if (APPEND && pos < 0) return;
  for (int i = threadIdx.x; i < p.half; i += 256) {
    float s, c;
    sincospif(2.f * rope_turn(p, pos, i), &s, &c);
    cs[i] = c * p.scale;
    sn[i] = s * p.scale * p.sign;
  }
  __syncthreads();
  int64_t ko = 0, vo = 0;
  bool stored = false;
  if (APPEND) {
    stored = cache_slot(p, t, pos, ko, vo);
    if (!stored && threadIdx.x == 0 && p.n_invalid) atomicAdd(p.n_invalid, 1);
  }
  const int items = p.hd - p.half;  // pairs, then the elements past rot_dim
  auto rotate = [&](const InT* src, auto* dst, int i, float mul) {
    if (i < p.half) {
      const int a = p.interleaved ? 2 * i : i, b = p.interleaved ? 2 * i + 1 : i + p.half;
      const float x = load_as_f32(src + a), y = load_as_f32(src + b);
      store_f32(dst + a, (x * cs[i] - y * sn[i]) * mul);
      store_f32(dst + b, (y * cs[i] + x * sn[i]) * mul);
    } else {
      store_f32(dst + i + p.half, load_as_f32(src + i + p.half) * mul);
    }
  };
  for (int e = threadIdx.x; e < p.hq * items; e += 256) {
    const int h = e / items, i = e - h * items;
    rotate((const InT*)p.q + t * p.ldq + h * p.hd, (OutT*)p.qo + t * p.ldqo + h * p.hd, i, 1.f);
  }
  if (!APPEND || !stored) return;
  for (int e = threadIdx.x; e < p.hkv * items; e += 256) {
    const int h = e / items, i = e - h * items;
    rotate((const InT*)p.k + t * p.ldk + h * p.hd, (CacheT*)p.kc + ko + h * p.kh, i, p.ks ? 1.f / p.ks[h] : 1.f);
  }
  for (int e = threadIdx.x; e < p.hkv * p.hd; e += 256) {
    const int h = e / p.hd, i = e - h * p.hd;
    const float x = load_as_f32((const InT*)p.v + t * p.ldv + e);
    store_f32((CacheT*)p.vc + vo + h * p.vh + i, p.vs ? x * (1.f / p.vs[h]) : x);
  }
}

}  // namespace th

using namespace th;

extern "C" int th_rope(const th_rope_desc* d, void* stream) {
  TH_CHECK_ARG(d != nullptr, "th_rope: null descriptor");
  TH_CHECK_ARG(d->tokens >= 0 && d->tokens < (int64_t)1 << 31, "th_rope: tokens %lld out of range",
               (long long)d->tokens);
  TH_CHECK_ARG(d->heads > 0 && d->head_dim > 0 && d->head_dim <= kMaxHeadDim, "th_rope: heads %d / head_dim %d unsupported",
               d->heads, d->head_dim);
  TH_CHECK_ARG((int64_t)d->heads * d->head_dim < (int64_t)1 << 30, "th_rope: row of %d heads too wide", d->heads);
  TH_CHECK_ARG(d->rot_dim > 0 && d->rot_dim % 2 == 0 && d->rot_dim <= d->head_dim,
               "th_rope: rot_dim %d must be even and in 2..head_dim", d->rot_dim);
  TH_CHECK_ARG(d->dtype == TH_BF16 || d->dtype == TH_F32, "th_rope: dtype %d unsupported", d->dtype);
  TH_CHECK_ARG(d->positions_dtype == TH_I32 || d->positions_dtype == TH_I64, "th_rope: positions dtype %d unsupported",
               d->positions_dtype);
  const int64_t row = (int64_t)d->heads * d->head_dim;
  TH_CHECK_ARG(d->ld_x >= row && d->ld_out >= row, "th_rope: row stride < heads*head_dim");
  TH_CHECK_ARG(d->x != d->out || d->ld_x == d->ld_out, "th_rope: in place needs one row stride");
  if (d->tokens == 0) return TH_OK;
  TH_CHECK_ARG(d->x && d->positions && d->freqs && d->out, "th_rope: null operand");
  if (!device_ready()) {
    set_error("th_rope: th_init was not called for the current device");
    return TH_ERR_NOT_INIT;
  }
  RopeK k{};
  k.q = d->x; k.ldq = d->ld_x; k.qo = d->out; k.ldqo = d->ld_out;
  k.positions = d->positions; k.freqs = d->freqs;
  k.scale = d->scale; k.sign = d->inverse ? -1.f : 1.f;
  k.hq = d->heads; k.hd = d->head_dim; k.half = d->rot_dim / 2; k.interleaved = d->interleaved != 0;
  const dim3 grid((unsigned)d->tokens);
  hipStream_t s = (hipStream_t)stream;
  const bool i64 = d->positions_dtype == TH_I64;
  if (d->dtype == TH_BF16) {
    if (i64) hipLaunchKernelGGL((rope_elem_kernel<int64_t, uint16_t, uint16_t, uint16_t, false>), grid, dim3(256), 0, s, k);
    else hipLaunchKernelGGL((rope_elem_kernel<int32_t, uint16_t, uint16_t, uint16_t, false>), grid, dim3(256), 0, s, k);
  } else {
    if (i64) hipLaunchKernelGGL((rope_elem_kernel<int64_t, float, float, uint16_t, false>), grid, dim3(256), 0, s, k);
    else hipLaunchKernelGGL((rope_elem_kernel<int32_t, float, float, uint16_t, false>), grid, dim3(256), 0, s, k);
  }
  TH_CHECK_LAUNCH();
  return TH_OK;
}

extern "C" int th_paged_append(const th_paged_append_desc* d, void* stream) {
  TH_CHECK_ARG(d != nullptr, "th_paged_append: null descriptor");
  TH_CHECK_ARG(d->tokens >= 0 && d->tokens < (int64_t)1 << 31, "th_paged_append: tokens %lld out of range",
               (long long)d->tokens);
  TH_CHECK_ARG(d->heads_q >= 0 && d->heads_kv > 0 && d->head_dim > 0 && d->head_dim <= kMaxHeadDim,
               "th_paged_append: heads %d, %d / head_dim %d unsupported", d->heads_q, d->heads_kv, d->head_dim);
  TH_CHECK_ARG((int64_t)d->heads_q * d->head_dim < (int64_t)1 << 30 && (int64_t)d->heads_kv * d->head_dim < (int64_t)1 << 30,
               "th_paged_append: row of %d, %d heads too wide", d->heads_q, d->heads_kv);
  TH_CHECK_ARG(d->rot_dim >= 0 && d->rot_dim % 2 == 0 && d->rot_dim <= d->head_dim,
               "th_paged_append: rot_dim %d must be even and in 0..head_dim", d->rot_dim);
  TH_CHECK_ARG(d->in_dtype == TH_BF16 || d->in_dtype == TH_F32, "th_paged_append: in_dtype %d unsupported", d->in_dtype);
  TH_CHECK_ARG(d->cache_dtype == TH_BF16 || d->cache_dtype == TH_F8E4M3, "th_paged_append: cache_dtype %d unsupported",
               d->cache_dtype);
  TH_CHECK_ARG(d->page_size > 0 && (d->page_size & (d->page_size - 1)) == 0,
               "th_paged_append: page_size %d must be a power of two", d->page_size);
  TH_CHECK_ARG(d->n_rows > 0 && d->row_pages > 0 && d->pages > 0 && d->ld_page_table >= d->row_pages,
               "th_paged_append: bad page table sizes");
  const int64_t wq = (int64_t)d->heads_q * d->head_dim, wk = (int64_t)d->heads_kv * d->head_dim;
  TH_CHECK_ARG(d->ld_k >= wk && d->ld_v >= wk && (d->heads_q == 0 || (d->ld_q >= wq && d->ld_q_out >= wq)),
               "th_paged_append: row stride < heads*head_dim");
  TH_CHECK_ARG(d->heads_q == 0 || d->q != d->q_out || (d->in_dtype == TH_BF16 && d->ld_q == d->ld_q_out),
               "th_paged_append: queries in place need bf16 and one row stride");
  TH_CHECK_ARG(d->k_stride_h >= d->head_dim && d->v_stride_h >= d->head_dim && d->k_stride_t >= d->head_dim &&
                   d->v_stride_t >= d->head_dim && d->k_stride_page >= d->head_dim && d->v_stride_page >= d->head_dim,
               "th_paged_append: cache stride < head_dim");
  TH_CHECK_ARG((!d->k_scale && !d->v_scale) || d->cache_dtype == TH_F8E4M3, "th_paged_append: scales need an e4m3 cache");
  if (d->tokens == 0) return TH_OK;
  TH_CHECK_ARG(d->rows || d->tokens <= d->n_rows, "th_paged_append: %lld tokens without rows exceed the table's %d",
               (long long)d->tokens, d->n_rows);
  TH_CHECK_ARG(d->k && d->v && d->positions && d->page_table && d->k_cache && d->v_cache &&
                   (d->rot_dim == 0 || d->freqs) && (d->heads_q == 0 || (d->q && d->q_out)),
               "th_paged_append: null operand");
  if (!device_ready()) {
    set_error("th_paged_append: th_init was not called for the current device");
    return TH_ERR_NOT_INIT;
  }
  RopeK k{};
  k.q = d->q; k.ldq = d->ld_q; k.qo = d->q_out; k.ldqo = d->ld_q_out;
  k.k = d->k; k.ldk = d->ld_k; k.v = d->v; k.ldv = d->ld_v;
  k.positions = d->positions; k.rows = d->rows; k.freqs = d->freqs;
  k.scale = d->scale; k.sign = 1.f;
  k.hq = d->heads_q; k.hkv = d->heads_kv; k.hd = d->head_dim; k.half = d->rot_dim / 2; k.interleaved = d->interleaved != 0;
  k.table = d->page_table; k.ldt = d->ld_page_table;
  k.n_rows = d->n_rows; k.row_pages = d->row_pages; k.pshift = __builtin_ctz((unsigned)d->page_size); k.pages = d->pages;
  k.kc = d->k_cache; k.kp = d->k_stride_page; k.kt = d->k_stride_t; k.kh = d->k_stride_h;
  k.vc = d->v_cache; k.vp = d->v_stride_page; k.vt = d->v_stride_t; k.vh = d->v_stride_h;
  k.ks = d->k_scale; k.vs = d->v_scale; k.n_invalid = d->n_invalid;
  const dim3 grid((unsigned)d->tokens);
  hipStream_t s = (hipStream_t)stream;
  const bool f32 = d->in_dtype == TH_F32, e4 = d->cache_dtype == TH_F8E4M3;
  if (f32 && e4) hipLaunchKernelGGL((rope_elem_kernel<int32_t, float, uint16_t, uint8_t, true>), grid, dim3(256), 0, s, k);
  else if (f32) hipLaunchKernelGGL((rope_elem_kernel<int32_t, float, uint16_t, uint16_t, true>), grid, dim3(256), 0, s, k);
  else if (e4) hipLaunchKernelGGL((rope_elem_kernel<int32_t, uint16_t, uint16_t, uint8_t, true>), grid, dim3(256), 0, s, k);
  else hipLaunchKernelGGL((rope_elem_kernel<int32_t, uint16_t, uint16_t, uint16_t, true>), grid, dim3(256), 0, s, k);
  TH_CHECK_LAUNCH();
  return TH_OK;
}
