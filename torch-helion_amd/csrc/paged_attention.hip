// th_paged_attention: attention of one query per token over a paged KV cache
// (no counterpart in the reference, which has no cache; the math is that of
// optimizer/evaluate.py:139-146 for one query row, with a window, capped scores
// and a bias by distance).
//
// HBM bound: 2 G operations per byte of a bf16 cache (G = query heads per kv
// head), so what counts is that every visible K and V byte is read once, that
// enough of them are in flight, and that all CUs have the same amount to read.
//
// Work: a tile is 8 KiB of K and 8 KiB of V (KT keys of one kv head), whatever
// the head size and type. The tiles of all (token, kv head) pairs form one
// line, and each of the 4 * grid waves takes an equal stretch of it, so ragged
// batches, one long sequence and many short ones are dealt out alike, with
// nothing about the lengths known on the host (a captured graph serves any
// lengths). A wave walks its stretch alone, with no workgroup barrier. The
// parts of a pair that was cut go through the workspace (m, l, o in fp32) to
// the join kernel; a pair inside one stretch is finished by its wave.
//
// One tile:
//   K        loaded straight in the operand layout of S^T = K Q^T
//            (v_mfma_f32_16x16x32_bf16: lane l holds row l % 16 and 8 dims from
//            8 (l / 16)): 16 bytes a lane, 64 contiguous bytes a row. The dims of
//            an e4m3 row are permuted (16 consecutive ones serve two k steps,
//            q alike), so that those loads are 16 bytes too.
//   V        loaded by rows, written to the wave's own LDS slice as bf16, and
//            read transposed (ds_read_b64_tr_b16) for O^T += V^T P^T; P^T is the
//            S^T accumulators as they are, rounded to bf16 (half a step is 2^-8 of
//            each p; sums and maxima stay fp32).
// The next tile's loads are issued as soon as S^T has used K, and land during
// the softmax and the second product. Buffer loads return zero past their
// range: unseen slots of a page and pages outside the cache cost no branch, and
// whatever they hold (NaN) never meets a zero probability.
#include "common.h"

#include <math.h>

#include <algorithm>

namespace th {

struct PAttnK {
  const uint16_t* q; int64_t ldq;
  const char* k; int64_t kp, kt, kh;  // byte strides: page, token, head
  const char* v; int64_t vp, vt, vh;
  uint16_t* o; int64_t ldo;
  const int32_t* positions;
  const int32_t* rows;
  const int32_t* table; int64_t ldt;
  int64_t pages;
  int n_rows, row_pages, pshift;
  int tokens, Hkv, G, nqb, gq;  // nqb blocks of gq <= 16 query heads per kv head
  int window;
  int o8;           // o in whole 8-byte pieces
  float scale, softcap;
  const float* slopes;
  const float* ks;
  const float* vs;
  int64_t* prefix;  // [tokens + 1]: tiles of one kv head of the tokens before
  float* ml;        // [2 waves][gq][2]
  float* part;      // [2 waves][gq][D], unnormalised
};

constexpr float kLog2e = 1.4426950408889634f;

typedef unsigned pa_u32x4 __attribute__((ext_vector_type(4)));
typedef short pa_s16x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ void pa_lds_order() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// A token's keys: [lo, hi) of its row; tiles start at lo rounded down to 16.
struct Span { int pos, row, lo, hi, base, tiles; };

template <int KT>
__device__ __forceinline__ Span span_from(const PAttnK& p, int pos, int row) {
  Span s;
  s.pos = pos;
  s.row = row;
  const bool in = row >= 0 && row < p.n_rows && pos >= 0;
  s.hi = in ? (int)min((int64_t)pos + 1, (int64_t)p.row_pages << p.pshift) : 0;
  s.lo = p.window ? (int)max((int64_t)0, (int64_t)pos + 1 - p.window) : 0;
  s.base = s.lo & ~15;
  s.tiles = s.hi > s.lo ? (s.hi - s.base + KT - 1) / KT : 0;
  return s;
}

template <int KT>
__device__ __forceinline__ Span span_of(const PAttnK& p, int t) {
  return span_from<KT>(p, p.positions[t], p.rows ? p.rows[t] : t);
}

// Equal stretches of n tiles over w waves: the first n % w get one more.
struct Share {
  int64_t each, more;
  __device__ __forceinline__ Share(int64_t n, int w) {
    if (n >> 31) {
      each = n / w;
      more = n - each * w;
    } else {
      each = (uint32_t)n / (uint32_t)w;
      more = (uint32_t)n - (uint32_t)each * (uint32_t)w;
    }
  }
  __device__ __forceinline__ int64_t begin(int i) const { return i * each + min((int64_t)i, more); }
  __device__ __forceinline__ int owner(int64_t u) const {
    const int64_t big = more * (each + 1);
    if ((u | big) >> 31) return (int)(u < big ? u / (each + 1) : more + (u - big) / each);
    return (int)((uint32_t)u < (uint32_t)big ? (uint32_t)u / (uint32_t)(each + 1)
                                             : (uint32_t)more + (uint32_t)(u - big) / (uint32_t)each);
  }
};

// 8 e4m3 values (two dwords) as 8 bf16: exact.
__device__ __forceinline__ bf16x8_t e4m3x8_to_bf16(unsigned lo, unsigned hi) {
  typedef __bf16 b2_t __attribute__((ext_vector_type(2)));
  union { b2_t h[4]; bf16x8_t v; } u;
  u.h[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false);
  u.h[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true);
  u.h[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false);
  u.h[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
  return u.v;
}

// LDS slot of 16-byte chunk c of V row r is c ^ sw(r): a transposing read (16
// rows, 32 bytes each) then hits every bank twice.
template <int D>
__device__ __forceinline__ int pa_sw(int r) { return D == 128 ? 2 * (r & 7) : 2 * ((r >> 1) & 3); }

template <int D, bool E4>
struct PaTile {
  static constexpr int RB = D * (E4 ? 1 : 2);   // bytes of a cached row
  static constexpr int KT = 8192 / RB;          // keys per tile
  static constexpr int NB = KT / 16;            // 16-key blocks
  static constexpr int CPR = RB / 16;           // 16-byte chunks per row
  static constexpr int RPI = 64 / CPR;          // V rows per load instruction
  static constexpr int LDS = KT * D * 2;        // one wave's V tile, bf16
};

template <int D, bool E4>
__global__ void __launch_bounds__(256, 2) paged_attn_kernel(PAttnK p) {
  using T = PaTile<D, E4>;
  constexpr int RB = T::RB, KT = T::KT, NB = T::NB, CPR = T::CPR, RPI = T::RPI;
  constexpr int NKS = D / 32, NDB = D / 16, JPR = RB / 64;  // JPR: K loads per 16-key block
  __shared__ __attribute__((aligned(16))) char smem[4 * T::LDS];
  __shared__ int64_t pre[257];
  __shared__ int64_t wsum[4];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int qc = lane & 15, g = lane >> 4;  // query column, lane group

  // ---- tiles before each of 256 runs of tokens
  const int per = (p.tokens + 255) >> 8;
  {
    int64_t n = 0;
    const int t0 = tid * per, t1 = min(p.tokens, t0 + per);
    for (int t = t0; t < t1; ++t) n += span_of<KT>(p, t).tiles;
    int64_t inc = n;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int64_t up = __shfl_up(inc, d);
      if (lane >= d) inc += up;
    }
    if (lane == 63) wsum[wave] = inc;
    __syncthreads();
    int64_t before = inc - n;
    for (int w = 0; w < wave; ++w) before += wsum[w];
    pre[tid] = before;
    if (tid == 255) pre[256] = before + n;
    if (blockIdx.x == 0) {  // for the join kernel
      int64_t at = before;
      for (int t = t0; t < t1; ++t) {
        p.prefix[t] = at;
        at += span_of<KT>(p, t).tiles;
      }
      if (tid == 255) p.prefix[p.tokens] = before + n;
    }
    __syncthreads();
  }
  const int HB = p.Hkv * p.nqb;
  const Share share(pre[256] * HB, gridDim.x * 4);
  const int me = wave * gridDim.x + blockIdx.x;  // few tiles: one wave per workgroup first
  const int64_t u0 = share.begin(me), u1 = share.begin(me + 1);
  if (u0 >= u1) return;

  // ---- the pair and tile that the stretch begins in
  int t = 0;
  for (int i = 0; i < 4; ++i) t += __popcll(__ballot(pre[64 * i + lane] * HB <= u0));
  t = (t - 1) * per;  // the last run that begins at or before u0
  int64_t at = pre[t / per];
  Span sp = span_of<KT>(p, t);
  while ((at + sp.tiles) * HB <= u0) {
    at += sp.tiles;
    sp = span_of<KT>(p, ++t);
  }
  int64_t u = u0;
  int hb, k;  // kv head block; tile of it
  {
    const int64_t rel = u0 - at * HB;
    if (rel >> 31) {
      hb = (int)(rel / sp.tiles);
    } else {
      hb = (int)((uint32_t)rel / (uint32_t)sp.tiles);
    }
    k = (int)(rel - (int64_t)hb * sp.tiles);
  }
  t = __builtin_amdgcn_readfirstlane(t);
  hb = __builtin_amdgcn_readfirstlane(hb);
  k = __builtin_amdgcn_readfirstlane(k);

  char* sv = smem + wave * T::LDS;
  // V: lane's row and chunk within one load instruction
  const int lr = lane / CPR, lc = lane % CPR;
  // V^T operand reads: this lane is source lane 4 e + j of group g, reading row
  // 4 g + e (and 16 + 4 g + e) of a 32-key block, columns 16 db + 4 j .. +3
  const int e4 = (lane & 15) >> 2, j4 = lane & 3;
  const int vr0 = 4 * g + e4;
  const int vxo = pa_sw<D>(vr0) >> 1;
  const char* rv = sv + vr0 * D * 2 + (j4 >> 1) * 16 + (j4 & 1) * 8;

  // ---- the load cursor (t, hb, k; sp): one tile ahead of the computation, also
  // over the ends of pairs and tokens
  // (the next token's position and row wait in vector registers: a scalar copy
  // would make the compiler wait for them where they are loaded)
  const int last_t = p.tokens - 1;
  int vzero = 0;
  asm volatile("" : "+v"(vzero));
  int npos, nrow = 0;
  auto load_next = [&]() {
    const int at_ = min(t + 1, last_t) + vzero;
    npos = p.positions[at_];
    if (p.rows) nrow = p.rows[at_];
  };
  load_next();
  // page numbers p0 .. p0 + 63 of the row, one a lane (-1: not in the cache)
  int p0 = 1 << 30, ids = -1;
  unsigned okbits = 0;  // bit b: block b of the loaded tile is in the cache
  pa_u32x4 kr[8], vr[8];
  auto load = [&]() {
    const int kvh = hb / p.nqb;
    const char* kb = p.k + (int64_t)kvh * p.kh;
    const char* vb = p.v + (int64_t)kvh * p.vh;
    const int j0 = sp.base + k * KT;
    const int first = j0 >> p.pshift, last = (min(j0 + KT, sp.hi) - 1) >> p.pshift;
    if (first < p0 || last - p0 >= 64) {
      p0 = first;
      const int at_ = p0 + lane;
      ids = at_ < p.row_pages ? p.table[(int64_t)sp.row * p.ldt + at_] : -1;
      if (ids >= p.pages) ids = -1;
    }
    okbits = 0;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const int jb = j0 + 16 * b;
      const int id = __builtin_amdgcn_readlane(ids, ((jb >> p.pshift) - p0) & 63);
      const int in = jb & ((1 << p.pshift) - 1);
      const int rows = min(16, sp.hi - jb);       // rows of this block below hi
      const bool ok = id >= 0 && rows > 0;
      okbits |= (ok ? 1u : 0u) << b;
      const char* kpage = kb + (int64_t)(ok ? id : 0) * p.kp + (int64_t)in * p.kt;
      const char* vpage = vb + (int64_t)(ok ? id : 0) * p.vp + (int64_t)in * p.vt;
      const auto kres = __builtin_amdgcn_make_buffer_rsrc((void*)kpage, 0, ok ? (int)((rows - 1) * p.kt) + RB : 0, 0x00020000);
      const auto vres = __builtin_amdgcn_make_buffer_rsrc((void*)vpage, 0, ok ? (int)((rows - 1) * p.vt) + RB : 0, 0x00020000);
#pragma unroll
      for (int j = 0; j < JPR; ++j)
        kr[b * JPR + j] = __builtin_bit_cast(
            pa_u32x4, __builtin_amdgcn_raw_buffer_load_b128(kres, qc * (int)p.kt + 64 * j + 16 * g, 0, 0));
#pragma unroll
      for (int i = 0; i < 16 / RPI; ++i) {
        const int r = i * RPI + lr;
        const int off = jb + r >= sp.lo ? r * (int)p.vt + 16 * lc : 0x7ffffff0;
        vr[b * (16 / RPI) + i] = __builtin_bit_cast(pa_u32x4, __builtin_amdgcn_raw_buffer_load_b128(vres, off, 0, 0));
      }
    }
  };
  // the pair's queries and scalars; a column past its heads repeats the last one
  // (no lane depends on another's column, and none of them is stored)
  bf16x8_t qn[NKS];
  float kscale_n = 1.f, slope_n = 0.f;
  auto load_pair = [&]() {
    const int kvh = hb / p.nqb, qb = hb - kvh * p.nqb;
    const int head = kvh * p.G + qb * 16 + min(qc, min(p.gq, p.G - qb * 16) - 1);
    const uint16_t* qrow = p.q + (int64_t)t * p.ldq + (int64_t)head * D;
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks)
      qn[ks] = *(const bf16x8_t*)(qrow + (E4 ? 64 * (ks >> 1) + 16 * g + 8 * (ks & 1) : 32 * ks + 8 * g));
    if (p.ks) kscale_n = p.ks[kvh];
    if (p.slopes) slope_n = p.slopes[head];
  };

  bf16x8_t qf[NKS];
  f32x4_t oacc[NDB];
  float m_run = 0.f, l_run = 0.f, mul = 0.f, slope = 0.f;
  // capped: softcap log2(e) tanh(mul s / (2 log2(e))), else mul s
  const bool cap = p.softcap > 0.f;
  const float mul0 = p.scale * (cap ? 2.f * kLog2e / p.softcap : kLog2e);
  const float capl = p.softcap * kLog2e;
  int k_begin = 0;
  int64_t u_begin = u0;
  bool fresh = true;
  load();
  load_pair();
  for (;;) {
    // ---- one tile of pair (ct, chb)
    const int ct = t, chb = hb, ck = k;
    const Span cs = sp;
    const unsigned ok = okbits;
    const int j0 = cs.base + ck * KT;
    if (fresh) {
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks) qf[ks] = qn[ks];
#pragma unroll
      for (int d = 0; d < NDB; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) oacc[d][r] = 0.f;
      m_run = -INFINITY;
      l_run = 0.f;
      mul = mul0 * kscale_n;
      slope = slope_n * kLog2e;
      k_begin = ck;
      u_begin = u;
    }
    pa_lds_order();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = i * RPI + lr;
      if constexpr (E4) {
        char* w = sv + r * D * 2 + (((2 * lc) ^ pa_sw<D>(r)) << 4);
        *(bf16x8_t*)w = e4m3x8_to_bf16(vr[i][0], vr[i][1]);
        *(bf16x8_t*)(w + 16) = e4m3x8_to_bf16(vr[i][2], vr[i][3]);
      } else {
        *(pa_u32x4*)(sv + r * D * 2 + ((lc ^ pa_sw<D>(r)) << 4)) = vr[i];
      }
    }
    f32x4_t s[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
#pragma unroll
      for (int r = 0; r < 4; ++r) s[b][r] = 0.f;
#pragma unroll
      for (int j = 0; j < JPR; ++j) {
        const pa_u32x4 x = kr[b * JPR + j];
        if constexpr (E4) {
          s[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(e4m3x8_to_bf16(x[0], x[1]), qf[2 * j], s[b], 0, 0, 0);
          s[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(e4m3x8_to_bf16(x[2], x[3]), qf[2 * j + 1], s[b], 0, 0, 0);
        } else {
          s[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, x), qf[j], s[b], 0, 0, 0);
        }
      }
    }
    ++u;
    const bool more = u < u1, ends = !more || ck + 1 == cs.tiles;
    if (more) {
      if (++k == sp.tiles) {
        k = 0;
        if (++hb == HB) {
          hb = 0;
          ++t;
          sp = span_from<KT>(p, __builtin_amdgcn_readfirstlane(npos), p.rows ? __builtin_amdgcn_readfirstlane(nrow) : t);
          while (sp.tiles == 0) sp = span_of<KT>(p, ++t);
          load_next();
          p0 = 1 << 30;
        }
      }
      load();
      if (ends) load_pair();
    }
    pa_lds_order();

    // scores in log2 units; this lane holds keys 16 b + 4 g + r of column qc
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float x = s[b][r] * mul;
        if (cap) x = capl - 2.f * capl * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x));
        s[b][r] = x;
      }
    if (p.slopes) {
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[b][r] -= slope * (float)(cs.pos - (j0 + 16 * b + 4 * g + r));
    }
    if (j0 < cs.lo || j0 + KT > cs.hi || ok != (1u << NB) - 1) {
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int j = j0 + 16 * b + 4 * g + r;
          if (j < cs.lo || j >= cs.hi || !(ok >> b & 1)) s[b][r] = -INFINITY;
        }
    }
    float mloc = -INFINITY;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) mloc = fmaxf(mloc, s[b][r]);
    mloc = fmaxf(mloc, __shfl_xor(mloc, 16));
    mloc = fmaxf(mloc, __shfl_xor(mloc, 32));
    const float m_new = fmaxf(m_run, mloc);
    const float m_use = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = __builtin_amdgcn_exp2f(m_run - m_use);
    m_run = m_new;
    float lsum = 0.f;
    bf16x8_t pf[NB / 2];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float e = __builtin_amdgcn_exp2f(s[b][r] - m_use);
        lsum += e;
        pf[b / 2][4 * (b & 1) + r] = (__bf16)e;
      }
    l_run = l_run * alpha + lsum;
#pragma unroll
    for (int d = 0; d < NDB; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) oacc[d][r] *= alpha;
#pragma unroll
    for (int b = 0; b < NB / 2; ++b)
#pragma unroll
      for (int db = 0; db < NDB; ++db) {
        const char* x = rv + b * 32 * D * 2 + ((db ^ vxo) << 5);
        const pa_s16x4 vlo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) pa_s16x4*)x);
        const pa_s16x4 vhi =
            __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) pa_s16x4*)(x + 16 * D * 2));
        const bf16x8_t vf = __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(vlo, vhi, 0, 1, 2, 3, 4, 5, 6, 7));
        oacc[db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[b], oacc[db], 0, 0, 0);
      }
    fresh = ends;
    if (!ends) continue;

    // ---- the pair's result here: the output, or a part for the join
    float l = l_run + __shfl_xor(l_run, 16);
    l += __shfl_xor(l, 32);
    const int kvh = chb / p.nqb, qb = chb - kvh * p.nqb;
    if (qc < min(p.gq, p.G - qb * 16)) {
      if (k_begin == 0 && ck + 1 == cs.tiles) {
        const float f = l == 0.f ? 0.f : (p.vs ? p.vs[kvh] : 1.f) / l;
        uint16_t* o = p.o + (int64_t)ct * p.ldo + (int64_t)(kvh * p.G + qb * 16 + qc) * D + 4 * g;
#pragma unroll
        for (int db = 0; db < NDB; ++db) {
          if (p.o8) {
            *(uint2*)(o + 16 * db) = make_uint2(pk_bf16x2(oacc[db][0] * f, oacc[db][1] * f),
                                                pk_bf16x2(oacc[db][2] * f, oacc[db][3] * f));
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r) o[16 * db + r] = f32_to_bf16(oacc[db][r] * f);
          }
        }
      } else {
        const int64_t slot = (int64_t)(2 * me + (u_begin != u0)) * p.gq + qc;
        if (g == 0) {
          p.ml[2 * slot] = m_run;
          p.ml[2 * slot + 1] = l;
        }
#pragma unroll
        for (int db = 0; db < NDB; ++db) *(f32x4_t*)(p.part + slot * D + 16 * db + 4 * g) = oacc[db];
      }
    }
    if (!more) break;
  }
}

// Joins the parts of one (token, query head): o = sum_i o_i 2^(m_i - m) / sum_i
// l_i 2^(m_i - m). Tokens without keys get zeros; pairs that one wave finished
// are left alone.
template <int D>
__global__ void __launch_bounds__(256) paged_attn_join_kernel(PAttnK p, int waves) {
  constexpr int LPR = D / 4, NG = 256 / LPR;  // lanes per row, rows at a time
  __shared__ float red[4];
  __shared__ float ls[NG];
  __shared__ f32x4_t os[NG][LPR];
  const int h = blockIdx.x, t = blockIdx.y, tid = threadIdx.x;
  const int kvh = h / p.G, in = h - kvh * p.G, qb = in >> 4, qc = in & 15;
  const int HB = p.Hkv * p.nqb, hb = kvh * p.nqb + qb;
  const int64_t a = p.prefix[t], tiles = p.prefix[t + 1] - a;
  uint16_t* o = p.o + (int64_t)t * p.ldo + (int64_t)h * D;
  if (tiles == 0) {
    if (tid < D) o[tid] = 0;
    return;
  }
  const Share share(p.prefix[p.tokens] * HB, waves);
  const int64_t b0 = a * HB + hb * tiles;
  const int w0 = share.owner(b0), n = share.owner(b0 + tiles - 1) - w0 + 1;
  if (n == 1) return;
  // part i is wave w0 + i's: its first segment's, or its last where that is another
  auto slot_of = [&](int i) {
    const int w = w0 + i;
    return (int64_t)(2 * w + (i == 0 && b0 != share.begin(w))) * p.gq + qc;
  };
  float mx = -INFINITY;
  for (int i = tid; i < n; i += 256) mx = fmaxf(mx, p.ml[2 * slot_of(i)]);
#pragma unroll
  for (int x = 32; x; x >>= 1) mx = fmaxf(mx, __shfl_xor(mx, x));
  if ((tid & 63) == 0) red[tid >> 6] = mx;
  __syncthreads();
  mx = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const float mu = mx == -INFINITY ? 0.f : mx;
  const int grp = tid / LPR, ln = tid - grp * LPR;
  float l = 0.f;
  f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int i = grp; i < n; i += NG) {
    const int64_t s = slot_of(i);
    const float f = __builtin_amdgcn_exp2f(p.ml[2 * s] - mu);
    l += p.ml[2 * s + 1] * f;
    const f32x4_t x = *(const f32x4_t*)(p.part + s * D + 4 * ln);
#pragma unroll
    for (int r = 0; r < 4; ++r) acc[r] += x[r] * f;
  }
  os[grp][ln] = acc;
  if (ln == 0) ls[grp] = l;
  __syncthreads();
  if (tid >= D) return;
  float ll = 0.f, oo = 0.f;
#pragma unroll
  for (int i = 0; i < NG; ++i) {
    ll += ls[i];
    oo += os[i][tid >> 2][tid & 3];
  }
  o[tid] = f32_to_bf16(ll == 0.f ? 0.f : oo / ll * (p.vs ? p.vs[kvh] : 1.f));
}

static int paged_grid() { return 2 * (device_cus() > 0 ? device_cus() : 256); }

}  // namespace th

using namespace th;

extern "C" int64_t th_paged_attention_workspace_bytes(int32_t tokens, int32_t heads_q, int32_t heads_kv, int32_t head_dim) {
  if (tokens < 0 || heads_q <= 0 || heads_kv <= 0 || heads_q % heads_kv || (head_dim != 64 && head_dim != 128)) return -1;
  const int64_t gq = std::min(heads_q / heads_kv, 16), slots = (int64_t)paged_grid() * 4 * 2;
  return cdiv((int64_t)(tokens + 1) * 8, 16) * 16 + cdiv(slots * gq * 2 * 4, 16) * 16 + slots * gq * head_dim * 4;
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
  TH_CHECK_ARG((int64_t)d->row_pages * d->page_size < (int64_t)1 << 30, "th_paged_attention: row of 2^30 keys or more");
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
  const int64_t es = d->cache_dtype == TH_BF16 ? 2 : 1;
  k.k = (const char*)d->k_cache; k.kp = d->k_stride_page * es; k.kt = d->k_stride_t * es; k.kh = d->k_stride_h * es;
  k.v = (const char*)d->v_cache; k.vp = d->v_stride_page * es; k.vt = d->v_stride_t * es; k.vh = d->v_stride_h * es;
  k.o = (uint16_t*)d->o; k.ldo = d->ld_o;
  k.positions = d->positions; k.rows = d->rows; k.table = d->page_table; k.ldt = d->ld_page_table; k.pages = d->pages;
  k.n_rows = d->n_rows; k.row_pages = d->row_pages; k.pshift = __builtin_ctz((unsigned)d->page_size);
  k.tokens = d->tokens; k.Hkv = d->heads_kv; k.G = d->heads_q / d->heads_kv;
  k.gq = std::min(k.G, 16); k.nqb = (int)cdiv(k.G, 16);
  k.o8 = d->ld_o % 4 == 0 && ((uintptr_t)d->o & 7) == 0;
  k.window = d->window; k.scale = d->scale; k.softcap = d->softcap;
  k.slopes = d->slopes; k.ks = d->k_scale; k.vs = d->v_scale;
  const int grid = paged_grid();
  char* ws = (char*)d->workspace;
  k.prefix = (int64_t*)ws;
  ws += cdiv((int64_t)(d->tokens + 1) * 8, 16) * 16;
  k.ml = (float*)ws;
  ws += cdiv((int64_t)grid * 8 * k.gq * 8, 16) * 16;
  k.part = (float*)ws;
  hipStream_t s = (hipStream_t)stream;
  const bool e4 = d->cache_dtype == TH_F8E4M3;
  if (d->head_dim == 128) {
    if (e4) hipLaunchKernelGGL((paged_attn_kernel<128, true>), dim3(grid), dim3(256), 0, s, k);
    else hipLaunchKernelGGL((paged_attn_kernel<128, false>), dim3(grid), dim3(256), 0, s, k);
  } else {
    if (e4) hipLaunchKernelGGL((paged_attn_kernel<64, true>), dim3(grid), dim3(256), 0, s, k);
    else hipLaunchKernelGGL((paged_attn_kernel<64, false>), dim3(grid), dim3(256), 0, s, k);
  }
  TH_CHECK_LAUNCH();
  const dim3 jgrid(d->heads_q, d->tokens);
  if (d->head_dim == 128) hipLaunchKernelGGL(paged_attn_join_kernel<128>, jgrid, dim3(256), 0, s, k, 4 * grid);
  else hipLaunchKernelGGL(paged_attn_join_kernel<64>, jgrid, dim3(256), 0, s, k, 4 * grid);
  TH_CHECK_LAUNCH();
  return TH_OK;
}
