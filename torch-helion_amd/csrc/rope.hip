// th_rope and th_paged_append: rotary positions token by token, into a tensor
// or into the pages of a KV cache (no counterpart in the reference, whose
// tables hold positions 0..S-1, optimizer/param_transforms.py:47-51).
//
// A pair (a, b) of a head at position p turns by phi = p f_i:
//   a' = s (a cos phi - b sin phi),  b' = s (b cos phi + a sin phi).
// Angles: p f_i / 2 pi is formed and reduced to a fraction of a turn in 64
// bits (at a million radians a float's step is 1/16 of one) and only the
// fraction goes through a single-precision sincospi: 1e-7 radians from its
// rounding to a float, and two steps of 2^-24 of the sine. One token's
// angles serve all its heads, so a workgroup computes them once, into LDS.
// Both kernels are HBM bound (three products per element read and written).
#include "common.h"

#include <math.h>

#include <algorithm>

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

// Values by one scale, on their way to e4m3. A product with the reciprocal alone is a
// step of 2^-24 off at times, and a value that lies between two e4m3 ones then rounds
// to the wrong one; its remainder, one fused product, puts it right (Markstein 1990; no
// under- or overflow with scales of 2^-90 to 2^90 and quotients below 512, and from 448
// on all are stored as 448). 16004 tokens of two 8 x 128 heads: 70.5 us, with the
// reciprocal alone 68.9, with divisions 76.9-78.2.
struct Divide {
  float by, m;
  bool plain;
  __device__ __forceinline__ explicit Divide(float scale)
      : by(scale), m(1.f / scale), plain(fabsf(scale) >= 0x1p-90f && fabsf(scale) <= 0x1p90f) {}
  __device__ __forceinline__ float near(float x) const {  // where plain
    const float y = x * m, z = fmaf(fmaf(-y, by, x), m, y);
    return fabsf(y) < 512.f ? z : y;
  }
  __device__ __forceinline__ float operator()(float x) const { return plain ? near(x) : x / by; }
  __device__ __forceinline__ void eight(float* f) const {
    if (plain) {
#pragma unroll
      for (int r = 0; r < 8; ++r) f[r] = near(f[r]);
    } else {
#pragma unroll
      for (int r = 0; r < 8; ++r) f[r] /= by;
    }
  }
};

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
__global__ void __launch_bounds__(256) rope_elem_kernel(RopeK p, int64_t tokens) {
  __shared__ float cs[kMaxHeadDim / 2], sn[kMaxHeadDim / 2];
  const int64_t t = grid_index();
  if (t >= tokens) return;
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
  auto rotate = [&](const InT* src, auto* dst, int i, const float* scale) {
    constexpr bool kE4 = sizeof(*dst) == 1;  // no other has a scale
    const Divide by(kE4 && scale ? *scale : 1.f);
    const auto put = [&](int at, float y) { store_f32(dst + at, kE4 && scale ? by(y) : y); };
    if (i < p.half) {
      const int a = p.interleaved ? 2 * i : i, b = p.interleaved ? 2 * i + 1 : i + p.half;
      const float x = load_as_f32(src + a), y = load_as_f32(src + b);
      put(a, x * cs[i] - y * sn[i]);
      put(b, y * cs[i] + x * sn[i]);
    } else {
      put(i + p.half, load_as_f32(src + i + p.half));
    }
  };
  for (int e = threadIdx.x; e < p.hq * items; e += 256) {
    const int h = e / items, i = e - h * items;
    rotate((const InT*)p.q + t * p.ldq + h * p.hd, (OutT*)p.qo + t * p.ldqo + h * p.hd, i, nullptr);
  }
  if (!APPEND || !stored) return;
  for (int e = threadIdx.x; e < p.hkv * items; e += 256) {
    const int h = e / items, i = e - h * items;
    rotate((const InT*)p.k + t * p.ldk + h * p.hd, (CacheT*)p.kc + ko + h * p.kh, i, p.ks ? p.ks + h : nullptr);
  }
  for (int e = threadIdx.x; e < p.hkv * p.hd; e += 256) {
    const int h = e / p.hd, i = e - h * p.hd;
    const float x = load_as_f32((const InT*)p.v + t * p.ldv + e);
    store_f32((CacheT*)p.vc + vo + h * p.vh + i, p.vs ? Divide(p.vs[h])(x) : x);
  }
}

// Eight consecutive elements, one 16-byte access for 16-bit types (two for
// fp32, one of 8 bytes for e4m3).
template <typename T> struct Pack8;
template <> struct Pack8<uint16_t> { uint4 w; };
template <> struct Pack8<float> { float4 w[2]; };

typedef unsigned rope_u32x4 __attribute__((ext_vector_type(4)));

// NT: past the caches (non-temporal).
template <bool NT, typename T>
__device__ __forceinline__ Pack8<T> load8(const T* s) {
  if constexpr (NT) {
    Pack8<T> p;
    rope_u32x4* w = (rope_u32x4*)&p;
#pragma unroll
    for (int i = 0; i < (int)(sizeof(p) / 16); ++i) w[i] = __builtin_nontemporal_load((const rope_u32x4*)s + i);
    return p;
  }
  return *(const Pack8<T>*)s;
}
__device__ __forceinline__ void unpack8(const Pack8<uint16_t>& p, float* f) {
  const uint32_t w[4] = {p.w.x, p.w.y, p.w.z, p.w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void unpack8(const Pack8<float>& p, float* f) {
  *(float4*)f = p.w[0];
  *(float4*)(f + 4) = p.w[1];
}
template <bool NT>
__device__ __forceinline__ void store8(uint16_t* d, const float* f) {
  const rope_u32x4 w = {pk_bf16x2(f[0], f[1]), pk_bf16x2(f[2], f[3]), pk_bf16x2(f[4], f[5]), pk_bf16x2(f[6], f[7])};
  if constexpr (NT) __builtin_nontemporal_store(w, (rope_u32x4*)d);
  else *(rope_u32x4*)d = w;
}
template <bool NT>
__device__ __forceinline__ void store8(float* d, const float* f) {
  *(float4*)d = *(const float4*)f;
  *(float4*)(d + 4) = *(const float4*)(f + 4);
}
template <bool NT>
__device__ __forceinline__ void store8(uint8_t* d, const float* f) {
  int w[2];
  float c[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) c[i] = f[i] != f[i] ? f[i] : fminf(fmaxf(f[i], -448.f), 448.f);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    w[i] = __builtin_amdgcn_cvt_pk_fp8_f32(c[4 * i], c[4 * i + 1], 0, false);
    w[i] = __builtin_amdgcn_cvt_pk_fp8_f32(c[4 * i + 2], c[4 * i + 3], w[i], true);
  }
  *(uint2*)d = make_uint2((unsigned)w[0], (unsigned)w[1]);
}

constexpr int kMaxTokens = 16;       // tokens of one workgroup
constexpr int kMaxAngles = 1024;     // their angles

// The usual shapes: rotated halves, heads and strides in whole 16-byte pieces.
// A thread takes eight pairs at a time (two pieces), or a piece that is only
// copied, and has the next one's loads under way while it finishes one; the
// first are issued before the angles are known. tpb tokens share a workgroup,
// so that a token of few heads does not leave most of it idle.
//
// NT: the inputs, and an append's 16-bit outputs, go past the caches.
template <typename PosT, typename InT, typename OutT, typename CacheT, bool APPEND, bool NT>
__global__ void __launch_bounds__(256) rope_vec_kernel(RopeK p, int64_t tokens, int tpb) {
  __shared__ __attribute__((aligned(16))) float cs[kMaxAngles], sn[kMaxAngles];
  __shared__ int64_t slot_k[kMaxTokens], slot_v[kMaxTokens];  // -1: not stored
  __shared__ int live[kMaxTokens];
  const int64_t t0 = grid_index() * tpb;
  if (t0 >= tokens) return;
  const int nt = (int)min((int64_t)tpb, tokens - t0);
  const int turns = p.half >> 3, rest = (p.hd - 2 * p.half) >> 3, all = p.hd >> 3;
  const int heads = p.hq + p.hkv;  // hkv is 0 without APPEND
  const int n_turn = heads * turns, n_rest = heads * rest;
  const int units = n_turn + n_rest + p.hkv * all;

  struct Unit {
    Pack8<InT> a, b;
    int tok, h, i, kind;  // kind 0: pairs 8 i ..; 1: a copied piece i; 2: piece i of v; -1: none
  };
  auto load = [&](int e) {
    Unit x;
    x.kind = -1;
    if (e >= nt * units) return x;
    x.tok = e / units;
    e -= x.tok * units;
    const InT* src;
    if (e < n_turn) {
      x.kind = 0;
      x.h = e / turns;
      x.i = e - x.h * turns;
    } else if (e < n_turn + n_rest) {
      x.kind = 1;
      e -= n_turn;
      x.h = e / rest;
      x.i = e - x.h * rest;
    } else {
      x.kind = 2;
      e -= n_turn + n_rest;
      x.h = e / all;
      x.i = e - x.h * all;
    }
    const int64_t t = t0 + x.tok;
    if (x.kind == 2) src = (const InT*)p.v + t * p.ldv + x.h * p.hd;
    else if (x.h < p.hq) src = (const InT*)p.q + t * p.ldq + x.h * p.hd;
    else src = (const InT*)p.k + t * p.ldk + (x.h - p.hq) * p.hd;
    const int at = x.kind == 2 ? 8 * x.i : x.kind == 1 ? 2 * p.half + 8 * x.i : p.interleaved ? 16 * x.i : 8 * x.i;
    x.a = load8<NT>(src + at);
    if (x.kind == 0) x.b = load8<NT>(src + (p.interleaved ? at + 8 : at + p.half));
    return x;
  };
  Unit cur = load(threadIdx.x);

  for (int e = threadIdx.x; e < nt * p.half; e += 256) {
    const int tok = e / p.half, i = e - tok * p.half;
    float s, c;
    sincospif(2.f * rope_turn(p, ((const PosT*)p.positions)[t0 + tok], i), &s, &c);
    cs[e] = c * p.scale;
    sn[e] = s * p.scale * p.sign;
  }
  if (APPEND && threadIdx.x < nt) {
    const int64_t pos = ((const PosT*)p.positions)[t0 + threadIdx.x];
    int64_t ko = -1, vo = -1;
    live[threadIdx.x] = pos >= 0;
    if (pos >= 0 && !cache_slot(p, t0 + threadIdx.x, pos, ko, vo)) {
      ko = -1;
      if (p.n_invalid) atomicAdd(p.n_invalid, 1);
    }
    slot_k[threadIdx.x] = ko;
    slot_v[threadIdx.x] = vo;
  }
  __syncthreads();

  auto finish = [&](const Unit& x) {
    if (APPEND && !live[x.tok]) return;
    const bool query = x.kind != 2 && x.h < p.hq;
    if (!query && slot_k[x.tok] < 0) return;
    const int kh = x.kind == 2 ? x.h : x.h - p.hq;
    float a[8], b[8];
    unpack8(x.a, a);
    if (x.kind == 0) {
      unpack8(x.b, b);
      const float* c = cs + x.tok * p.half + 8 * x.i;
      const float* s = sn + x.tok * p.half + 8 * x.i;
      if (p.interleaved) {  // a: pairs 0..3, b: pairs 4..7
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float u = a[2 * r], v = a[2 * r + 1], w = b[2 * r], z = b[2 * r + 1];
          a[2 * r] = u * c[r] - v * s[r];
          a[2 * r + 1] = v * c[r] + u * s[r];
          b[2 * r] = w * c[4 + r] - z * s[4 + r];
          b[2 * r + 1] = z * c[4 + r] + w * s[4 + r];
        }
      } else {
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const float u = a[r], v = b[r];
          a[r] = u * c[r] - v * s[r];
          b[r] = v * c[r] + u * s[r];
        }
      }
    }
    const int at = x.kind == 2 ? 8 * x.i : x.kind == 1 ? 2 * p.half + 8 * x.i : p.interleaved ? 16 * x.i : 8 * x.i;
    const int bt = p.interleaved ? at + 8 : at + p.half;
    if (query) {
      OutT* d = (OutT*)p.qo + (t0 + x.tok) * p.ldqo + x.h * p.hd;
      store8<NT && APPEND>(d + at, a);
      if (x.kind == 0) store8<NT && APPEND>(d + bt, b);
      return;
    }
    if constexpr (APPEND) {
      const float* scales = x.kind == 2 ? p.vs : p.ks;
      if (scales) {
        const Divide by(scales[kh]);
        by.eight(a);
        if (x.kind == 0) by.eight(b);
      }
      CacheT* d = x.kind == 2 ? (CacheT*)p.vc + slot_v[x.tok] + kh * p.vh : (CacheT*)p.kc + slot_k[x.tok] + kh * p.kh;
      store8<NT && APPEND>(d + at, a);
      if (x.kind == 0) store8<NT && APPEND>(d + bt, b);
    }
  };
  for (int e = threadIdx.x; e < nt * units; e += 256) {
    const Unit next = load(e + 256);
    finish(cur);
    cur = next;
  }
}

static bool whole16(const void* p, int64_t ld, int size) { return ((uintptr_t)p & 15) == 0 && ld * size % 16 == 0; }

template <typename PosT, typename InT, typename OutT, typename CacheT, bool APPEND>
static void launch_rope(const RopeK& k, int64_t tokens, hipStream_t s) {
  bool vec = k.half % 8 == 0 && k.half <= kMaxAngles && k.hd % 8 == 0;
  if (k.hq) vec = vec && whole16(k.q, k.ldq, sizeof(InT)) && whole16(k.qo, k.ldqo, sizeof(OutT));
  if (APPEND) {
    // a cache piece is 8 elements: 16 bytes of bf16, 8 of e4m3
    const uintptr_t mask = 8 * sizeof(CacheT) - 1;
    vec = vec && whole16(k.k, k.ldk, sizeof(InT)) && whole16(k.v, k.ldv, sizeof(InT)) &&
          (((uintptr_t)k.kc | (uintptr_t)k.vc) & mask) == 0 && (k.kp | k.kt | k.kh | k.vp | k.vt | k.vh) % 8 == 0;
  }
  if (!vec) {
    hipLaunchKernelGGL((rope_elem_kernel<PosT, InT, OutT, CacheT, APPEND>), grid_of(tokens), dim3(256), 0, s, k, tokens);
    return;
  }
  const int units = (k.hq + k.hkv) * ((k.hd - k.half) >> 3) + k.hkv * (k.hd >> 3);
  int tpb = std::max(1, std::min(256 / units, kMaxTokens));
  if (k.half) tpb = std::min(tpb, kMaxAngles / k.half);
  // More than half of the 256 MB last-level cache would not be there for the next
  // kernel anyway. 16384 x 32 x 128 bf16 (268 MB) 47.8 -> 44.7 us, with its stores
  // past the caches too 47.3; 16004 prompt tokens into an e4m3 cache (361 MB) 71.3 ->
  // 67.5, with the loads alone 74.8 (1.4 us more each since the scale divides).
  const int64_t bytes = tokens * (((int64_t)k.hq + 2 * k.hkv) * k.hd * (int)sizeof(InT) + (int64_t)k.hq * k.hd * (int)sizeof(OutT) +
                                  2 * (int64_t)k.hkv * k.hd * (int)sizeof(CacheT));
  const dim3 grid = grid_of(cdiv(tokens, tpb));
  if (bytes > 128 << 20)
    hipLaunchKernelGGL((rope_vec_kernel<PosT, InT, OutT, CacheT, APPEND, true>), grid, dim3(256), 0, s, k, tokens, tpb);
  else
    hipLaunchKernelGGL((rope_vec_kernel<PosT, InT, OutT, CacheT, APPEND, false>), grid, dim3(256), 0, s, k, tokens, tpb);
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
  hipStream_t s = (hipStream_t)stream;
  const bool i64 = d->positions_dtype == TH_I64;
  if (d->dtype == TH_BF16) {
    if (i64) launch_rope<int64_t, uint16_t, uint16_t, uint16_t, false>(k, d->tokens, s);
    else launch_rope<int32_t, uint16_t, uint16_t, uint16_t, false>(k, d->tokens, s);
  } else {
    if (i64) launch_rope<int64_t, float, float, uint16_t, false>(k, d->tokens, s);
    else launch_rope<int32_t, float, float, uint16_t, false>(k, d->tokens, s);
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
  hipStream_t s = (hipStream_t)stream;
  const bool f32 = d->in_dtype == TH_F32, e4 = d->cache_dtype == TH_F8E4M3;
  if (f32 && e4) launch_rope<int32_t, float, uint16_t, uint8_t, true>(k, d->tokens, s);
  else if (f32) launch_rope<int32_t, float, uint16_t, uint16_t, true>(k, d->tokens, s);
  else if (e4) launch_rope<int32_t, uint16_t, uint16_t, uint8_t, true>(k, d->tokens, s);
  else launch_rope<int32_t, uint16_t, uint16_t, uint16_t, true>(k, d->tokens, s);
  TH_CHECK_LAUNCH();
  return TH_OK;
}
