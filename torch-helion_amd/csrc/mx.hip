// th_mx_quantize, th_mx_dequantize, th_mx_rmsnorm: tensors into the blocks of the
// OCP microscaling format and back (no counterpart in the reference).
//
// All three are HBM bound: every value is read once and written once, with a
// few instructions each. A lane holds 8 consecutive values (a chunk: 16 bytes
// of bf16) and a quad of lanes a block, whose largest magnitude they find with
// two lane exchanges; gfx950's scaled conversions do the division by the scale
// and the rounding. Where a copy of 1 GiB reaches 5.2 TB/s: 14336 x 4096 bf16
// to e2m1 29.5 us (5.0 TB/s) and back 28.0 (5.3), 16384 x 4096 fp32 to e4m3
// 59.8 (5.7), the norm of 16384 x 4096 bf16 with a residual 85 (5.5); 64 rows
// of 4096 take 2.2 and 3.0 us, a launch's time.
#include "mx.h"

#include <algorithm>

namespace th {

struct MxRowsK {
  int64_t rows;
  int cols, chunks;       // chunks of 8 columns, whole blocks: a multiple of 4
  int lanes_log2, segs;   // lanes of a row's stretch (4 .. 64), stretches a row
  const void* x; int64_t ldx;
  void* codes; int64_t ldc;
  uint8_t* scales; int64_t lds;
};

__device__ const float kMxNone[8] = {};

// 8 columns from col of a row; zeros instead for a chunk that the row ends in (see mx_tail8) or before. Without a
// branch, so that the loads of a wave are in flight together: with branches each waited for the one before, and the
// quantiser took 60 us instead of 30 for 14336 x 4096 of bf16.
template <typename T>
__device__ __forceinline__ void mx_load8(const T* row, int col, int cols, float (&v)[8]) {
  const T* at = col + 8 <= cols ? row + col : (const T*)kMxNone;
  if constexpr (sizeof(T) == 2) {
    const mx_u4 w = mx_load16(at);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  } else {
    const mx_u4 a = mx_load16(at), b = mx_load16(at + 4);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(i < 4 ? a[i] : b[i - 4]);
  }
}

// What mx_load8 left: the chunk that the row ends in.
template <typename T>
__device__ __forceinline__ void mx_tail8(const T* row, int col, int cols, float (&v)[8]) {
  if (col >= cols || col + 8 <= cols) return;
#pragma unroll
  for (int i = 0; i < 7; ++i) {
    if (col + i < cols) {
      if constexpr (sizeof(T) == 2) v[i] = bf16_to_f32(row[col + i]);
      else v[i] = row[col + i];
    }
  }
}

// v, of the precision of T already or rounded here, to 8 columns from col.
template <typename T>
__device__ __forceinline__ void mx_store8(T* row, int col, int cols, const float (&v)[8]) {
  if (col + 8 <= cols) {
    if constexpr (sizeof(T) == 2) {
      mx_store16(row + col, mx_u4{pk_bf16x2(v[0], v[1]), pk_bf16x2(v[2], v[3]), pk_bf16x2(v[4], v[5]), pk_bf16x2(v[6], v[7])});
    } else {
#pragma unroll
      for (int h = 0; h < 8; h += 4)
        mx_store16(row + col + h, mx_u4{__float_as_uint(v[h]), __float_as_uint(v[h + 1]), __float_as_uint(v[h + 2]), __float_as_uint(v[h + 3])});
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (col + i < cols) {
        if constexpr (sizeof(T) == 2) row[col + i] = f32_to_bf16(v[i]);
        else row[col + i] = v[i];
      }
  }
}

// Where a lane stands: unit u is a stretch of up to 64 lanes over one row, or of
// several short rows.
struct MxPlace {
  int64_t row;
  int c;
  bool live;
  __device__ __forceinline__ MxPlace(const MxRowsK& p, int64_t group, int seg, int lane) {
    row = (group << (6 - p.lanes_log2)) + (lane >> p.lanes_log2);
    c = (seg << p.lanes_log2) + (lane & ((1 << p.lanes_log2) - 1));
    live = row < p.rows && c < p.chunks;
  }
};

template <typename T, int U>
__global__ void __launch_bounds__(256) mx_quantize_kernel(MxRowsK p, bool e2m1) {
  const int lane = threadIdx.x & 63;
  const int64_t wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)) + grid_index() * 4;
  int64_t group = wave * U / p.segs;
  int seg = (int)(wave * U - group * p.segs);
  float v[U][8];
  int64_t groups[U];
  int segs[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const MxPlace at(p, group, seg, lane);
    mx_load8((const T*)p.x + min(at.row, p.rows - 1) * p.ldx, at.c * 8, p.cols, v[i]);
    groups[i] = group, segs[i] = seg;
    if (++seg == p.segs) seg = 0, ++group;
  }
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const MxPlace at(p, groups[i], segs[i], lane);  // (the lanes of a quad are live together)
    mx_tail8((const T*)p.x + min(at.row, p.rows - 1) * p.ldx, at.c * 8, p.cols, v[i]);
    mx_put8(v[i], e2m1, (uint8_t*)p.codes + at.row * p.ldc, p.scales + at.row * p.lds, at.c, at.live);
  }
}

template <typename T, bool E2M1, int U>
__global__ void __launch_bounds__(256) mx_dequantize_kernel(MxRowsK p, T* out, int64_t ldo) {
  const int lane = threadIdx.x & 63;
  const int64_t wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)) + grid_index() * 4;
  int64_t group = wave * U / p.segs;
  int seg = (int)(wave * U - group * p.segs);
  uint2 w[U];
  int s[U];
  int64_t groups[U];
  int segs[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const MxPlace at(p, group, seg, lane);
    const int64_t row = at.live ? at.row : 0;  // (a lane with nothing to do reads the first chunk)
    const int c = at.live ? at.c : 0;
    const uint8_t* codes = (const uint8_t*)p.codes + row * p.ldc;
    w[i] = make_uint2(0, 0);
    if constexpr (E2M1) w[i].x = *(const uint32_t*)(codes + 4 * (int64_t)c);
    else w[i] = *(const uint2*)(codes + 8 * (int64_t)c);
    s[i] = p.scales[row * p.lds + (c >> 2)];
    groups[i] = group, segs[i] = seg;
    if (++seg == p.segs) seg = 0, ++group;
  }
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const MxPlace at(p, groups[i], segs[i], lane);
    if (!at.live) continue;
    typedef float f2_t __attribute__((ext_vector_type(2)));
    const float scale = mx_scale_operand(s[i]);
    f2_t f[4];
    if constexpr (E2M1) {
      f[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i].x, scale, 0);
      f[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i].x, scale, 1);
      f[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i].x, scale, 2);
      f[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i].x, scale, 3);
    } else {
      f[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w[i].x, scale, false);
      f[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w[i].x, scale, true);
      f[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w[i].y, scale, false);
      f[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w[i].y, scale, true);
    }
    const float v[8] = {f[0][0], f[0][1], f[1][0], f[1][1], f[2][0], f[2][1], f[3][0], f[3][1]};
    mx_store8(out + at.row * ldo, at.c * 8, p.cols, v);
  }
}

struct MxNormK {
  int64_t rows;
  int cols, chunks;
  const void* x; int64_t ldx;
  const void* r; int64_t ldr;
  void* h; int64_t ldh;
  const float* gain;
  uint8_t* codes; int64_t ldc;
  uint8_t* scales; int64_t lds;
  float inv_n, eps;
  bool e2m1;
};

// A workgroup of NW waves for a row, which stays in registers from the sum of squares (fp32) to its codes: CH chunks a lane.
template <typename T, int NW, int CH>
__global__ void __launch_bounds__(64 * NW) mx_rmsnorm_kernel(MxNormK p) {
  __shared__ float part[NW];
  const int tid = threadIdx.x;
  const int64_t row = grid_index();
  if (row >= p.rows) return;
  const T* x = (const T*)p.x + row * p.ldx;
  float v[CH][8];
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int c = i * 64 * NW + tid;
    mx_load8(x, c * 8, p.cols, v[i]);
  }
  if (p.r) {
    const T* r = (const T*)p.r + row * p.ldr;
    float w[CH][8];
#pragma unroll
    for (int i = 0; i < CH; ++i) mx_load8(r, (i * 64 * NW + tid) * 8, p.cols, w[i]);
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int c = i * 64 * NW + tid;
      mx_tail8(x, c * 8, p.cols, v[i]);
      mx_tail8(r, c * 8, p.cols, w[i]);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[i][j] += w[i][j];
        if constexpr (sizeof(T) == 2) v[i][j] = bf16_to_f32(f32_to_bf16(v[i][j]));  // what the residual stream holds
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < CH; ++i) mx_tail8(x, (i * 64 * NW + tid) * 8, p.cols, v[i]);
  }
  if (p.h) {
    T* h = (T*)p.h + row * p.ldh;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int c = i * 64 * NW + tid;
      mx_store8(h, c * 8, p.cols, v[i]);
    }
  }
  // the sum of squares in units of 1 / by, the same bits in every thread
  auto sum_squares = [&](float by) __attribute__((always_inline)) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < CH; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float x = v[i][j] * by;
        ss = fmaf(x, x, ss);
      }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) ss += __shfl_xor(ss, d);
    if constexpr (NW > 1) {
      if ((tid & 63) == 0) part[tid >> 6] = ss;
      __syncthreads();
      ss = 0.f;
#pragma unroll
      for (int i = 0; i < NW; ++i) ss += part[i];
    }
    return ss;
  };
  const float mean = sum_squares(1.f) * p.inv_n + p.eps;
  float rs = rsqrtf(mean);
  // Squares past fp32's range (of values from 2^56 on), or so far below it that they lose bits (and eps with them): the sum
  // again in units of 2^80 or 2^-100, in which it is 2^112 or 2^96 at most. Half of the unit's power then goes to the
  // values and half to the root, so that neither leaves the range.
  if (mean == __uint_as_float(0x7f800000u) || mean < 0x1p-120f) {
    const float half = mean < 1.f ? 0x1p50f : 0x1p-40f;
    if constexpr (NW > 1) __syncthreads();  // every wave has read the parts
    rs = rsqrtf(sum_squares(half * half) * p.inv_n + p.eps * (half * half) * (half * half)) * half;
#pragma unroll
    for (int i = 0; i < CH; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] *= half;
  }
  uint8_t* codes = p.codes + row * p.ldc;
  uint8_t* scales = p.scales + row * p.lds;
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int c = i * 64 * NW + tid;
    if (i * 64 * NW >= p.chunks) break;
    float g[8];
    mx_load8(p.gain, c * 8, p.cols, g);
    mx_tail8(p.gain, c * 8, p.cols, g);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[i][j] = c * 8 + j < p.cols ? v[i][j] * rs * g[j] : 0.f;  // (a sum of squares of NaN makes 0 NaN)
    mx_put8(v[i], p.e2m1, codes, scales, c, c < p.chunks);
  }
}

template <typename T>
static void launch_norm(const MxNormK& k, hipStream_t s) {
  constexpr int64_t kMost = (int64_t)1 << 21;  // a launch dimension holds 2^32 threads, a workgroup up to 1024
  const dim3 g = k.rows <= kMost ? dim3((unsigned)k.rows) : dim3((unsigned)kMost, (unsigned)cdiv(k.rows, kMost));
#define TH_NORM(NW, CH) hipLaunchKernelGGL((mx_rmsnorm_kernel<T, NW, CH>), g, dim3(64 * NW), 0, s, k)
  // As many waves as a row has work for, 16 at most: 64 rows of 4096 take 3.0 us with eight waves of one chunk a lane,
  // 3.5 with four of two and 6.4 with one of eight, 16384 rows 85, 86 and 100; 4096 rows of 14336
  // 78 us with 16 of two, 81 with eight of four and 94 with four of eight. (Past 32768 columns the registers of 1024
  // threads do not hold a row, and 430 bytes a lane lie in memory: 1024 rows of 65536 216 us, 2.2 TB/s.)
  if (k.chunks <= 64) TH_NORM(1, 1);
  else if (k.chunks <= 256) TH_NORM(4, 1);
  else if (k.chunks <= 512) TH_NORM(8, 1);
  else if (k.chunks <= 1024) TH_NORM(8, 2);
  else if (k.chunks <= 2048) TH_NORM(16, 2);
  else if (k.chunks <= 4096) TH_NORM(16, 4);
  else TH_NORM(16, 8);
#undef TH_NORM
}

// Lays the rows out over waves; returns the units.
static int64_t place(MxRowsK& k) {
  k.chunks = (int)cdiv(k.cols, 32) * 4;
  k.lanes_log2 = 2;
  while (k.lanes_log2 < 6 && (1 << k.lanes_log2) < k.chunks) ++k.lanes_log2;
  k.segs = (int)cdiv(k.chunks, 1 << k.lanes_log2);
  return cdiv(k.rows, 64 >> k.lanes_log2) * k.segs;
}

// Units a wave takes: two, whose loads are in flight together, where eight waves a SIMD are left. Two against one:
// 14336 x 4096 bf16 to e2m1 29.5 and 31.7 us, back 28.0 and 31.9; 64 x 4096 to e4m3 2.4 and 2.2. (Four: 29.7 and
// 28.6, but 16384 x 4096 fp32 to e4m3 65 us instead of 60.)
static int per_wave(int64_t units) { return units >= 2 * 8 * 4 * 256 ? 2 : 1; }

static int64_t element_bytes(int dtype) { return dtype == TH_BF16 ? 2 : 4; }
template <typename D>
static MxSpan codes_of(const D* d, const void* codes) {
  return {codes, d->rows, d->ld_codes, cdiv(d->cols, 32) * (d->mx_dtype == TH_F4E2M1 ? 16 : 32)};
}
template <typename D>
static MxSpan scales_of(const D* d) {
  return {d->scales, d->rows, d->ld_scales, cdiv(d->cols, 32)};
}

}  // namespace th

using namespace th;

#define TH_CHECK_BLOCKS(name, d, codes_)                                                                                \
  do {                                                                                                                  \
    TH_CHECK_ARG((d)->rows >= 0 && (d)->cols > 0 && (d)->cols < (1 << 30), name ": rows=%lld cols=%d out of range",     \
                 (long long)(d)->rows, (d)->cols);                                                                      \
    TH_CHECK_ARG((d)->mx_dtype == TH_F8E4M3 || (d)->mx_dtype == TH_F4E2M1, name ": mx_dtype %d is neither e4m3 nor e2m1", \
                 (d)->mx_dtype);                                                                                        \
    const int64_t nb_ = cdiv((d)->cols, 32);                                                                            \
    TH_CHECK_ARG((d)->ld_codes >= nb_ * ((d)->mx_dtype == TH_F4E2M1 ? 16 : 32) && (d)->ld_codes % 16 == 0 &&           \
                     ((uintptr_t)(codes_) & 15) == 0,                                                                   \
                 name ": codes must be 16-byte aligned, their rows whole blocks in whole 16 bytes apart");              \
    TH_CHECK_ARG((d)->ld_scales >= nb_, name ": scale rows of fewer than %lld bytes", (long long)nb_);                 \
  } while (0)

#define TH_CHECK_READY(name)                                             \
  do {                                                                   \
    if (!device_ready()) {                                               \
      set_error(name ": th_init was not called for the current device"); \
      return TH_ERR_NOT_INIT;                                            \
    }                                                                    \
  } while (0)

extern "C" int th_mx_quantize(const th_mx_quantize_desc* d, void* stream) {
  TH_CHECK_ARG(d != nullptr, "th_mx_quantize: null descriptor");
  TH_CHECK_ARG(d->x_dtype == TH_BF16 || d->x_dtype == TH_F32, "th_mx_quantize: x_dtype %d unsupported", d->x_dtype);
  TH_CHECK_BLOCKS("th_mx_quantize", d, d->codes);
  TH_CHECK_ARG(d->ld_x >= d->cols, "th_mx_quantize: x row stride smaller than cols");
  if (d->rows == 0) return TH_OK;
  TH_CHECK_ARG(d->x && d->codes && d->scales, "th_mx_quantize: null tensor pointer");
  const MxSpan x{d->x, d->rows, d->ld_x * element_bytes(d->x_dtype), d->cols * element_bytes(d->x_dtype)};
  const MxSpan codes = codes_of(d, d->codes), scales = scales_of(d);
  TH_CHECK_ARG(!mx_meet(codes, x) && !mx_meet(scales, x) && !mx_meet(scales, codes),
               "th_mx_quantize: codes and scales need memory of their own");
  TH_CHECK_READY("th_mx_quantize");
  MxRowsK k{};
  k.rows = d->rows; k.cols = d->cols;
  k.x = d->x; k.ldx = d->ld_x; k.codes = d->codes; k.ldc = d->ld_codes; k.scales = d->scales; k.lds = d->ld_scales;
  const int64_t units = place(k);
  const int u = per_wave(units);
  TH_CHECK_ARG(cdiv(units, 4 * u) < (int64_t)1 << 38, "th_mx_quantize: too many rows");
  const dim3 g = grid_of(cdiv(units, 4 * u));
  const bool e2m1 = d->mx_dtype == TH_F4E2M1;
  hipStream_t s = (hipStream_t)stream;
  auto go = [&](auto one) {
    using T = decltype(one);
    if (u == 2) hipLaunchKernelGGL((mx_quantize_kernel<T, 2>), g, dim3(256), 0, s, k, e2m1);
    else hipLaunchKernelGGL((mx_quantize_kernel<T, 1>), g, dim3(256), 0, s, k, e2m1);
  };
  if (d->x_dtype == TH_BF16) go(uint16_t());
  else go(float());
  TH_CHECK_LAUNCH();
  return TH_OK;
}

extern "C" int th_mx_dequantize(const th_mx_dequantize_desc* d, void* stream) {
  TH_CHECK_ARG(d != nullptr, "th_mx_dequantize: null descriptor");
  TH_CHECK_ARG(d->out_dtype == TH_BF16 || d->out_dtype == TH_F32, "th_mx_dequantize: out_dtype %d unsupported", d->out_dtype);
  TH_CHECK_BLOCKS("th_mx_dequantize", d, d->codes);
  TH_CHECK_ARG(d->ld_out >= d->cols, "th_mx_dequantize: out row stride smaller than cols");
  if (d->rows == 0) return TH_OK;
  TH_CHECK_ARG(d->out && d->codes && d->scales, "th_mx_dequantize: null tensor pointer");
  const MxSpan out{d->out, d->rows, d->ld_out * element_bytes(d->out_dtype), d->cols * element_bytes(d->out_dtype)};
  TH_CHECK_ARG(!mx_meet(out, codes_of(d, d->codes)) && !mx_meet(out, scales_of(d)), "th_mx_dequantize: out needs memory of its own");
  TH_CHECK_READY("th_mx_dequantize");
  MxRowsK k{};
  k.rows = d->rows; k.cols = d->cols;
  k.codes = (void*)d->codes; k.ldc = d->ld_codes; k.scales = (uint8_t*)d->scales; k.lds = d->ld_scales;
  const int64_t units = place(k);
  const int u = per_wave(units);
  TH_CHECK_ARG(cdiv(units, 4 * u) < (int64_t)1 << 38, "th_mx_dequantize: too many rows");
  const dim3 g = grid_of(cdiv(units, 4 * u));
  hipStream_t s = (hipStream_t)stream;
  auto go = [&](auto one, auto four) {
    using T = decltype(one);
    constexpr bool F = decltype(four)::value;
    if (u == 2) hipLaunchKernelGGL((mx_dequantize_kernel<T, F, 2>), g, dim3(256), 0, s, k, (T*)d->out, d->ld_out);
    else hipLaunchKernelGGL((mx_dequantize_kernel<T, F, 1>), g, dim3(256), 0, s, k, (T*)d->out, d->ld_out);
  };
  auto typed = [&](auto one) {
    if (d->mx_dtype == TH_F4E2M1) go(one, std::true_type());
    else go(one, std::false_type());
  };
  if (d->out_dtype == TH_BF16) typed(uint16_t());
  else typed(float());
  TH_CHECK_LAUNCH();
  return TH_OK;
}

extern "C" int th_mx_rmsnorm(const th_mx_rmsnorm_desc* d, void* stream) {
  TH_CHECK_ARG(d != nullptr, "th_mx_rmsnorm: null descriptor");
  TH_CHECK_ARG(d->x_dtype == TH_BF16 || d->x_dtype == TH_F32, "th_mx_rmsnorm: x_dtype %d unsupported", d->x_dtype);
  TH_CHECK_BLOCKS("th_mx_rmsnorm", d, d->codes);
  TH_CHECK_ARG(d->cols <= 65536 && d->rows < (int64_t)1 << 31, "th_mx_rmsnorm: more than 65536 columns or 2^31 rows");
  TH_CHECK_ARG(d->ld_x >= d->cols && (!d->residual || d->ld_residual >= d->cols) && (!d->sum_out || d->ld_sum_out >= d->cols),
               "th_mx_rmsnorm: a row stride is smaller than cols");
  TH_CHECK_ARG((d->sum_out != d->x || d->ld_sum_out == d->ld_x || d->rows <= 1) &&
                   (!d->sum_out || d->sum_out != d->residual || d->ld_sum_out == d->ld_residual || d->rows <= 1),
               "th_mx_rmsnorm: in place needs one row stride");
  if (d->rows == 0) return TH_OK;
  TH_CHECK_ARG(d->x && d->gain && d->codes && d->scales, "th_mx_rmsnorm: null tensor pointer");
  const int64_t size = element_bytes(d->x_dtype), width = d->cols * size;
  const MxSpan x{d->x, d->rows, d->ld_x * size, width}, residual{d->residual, d->rows, d->ld_residual * size, width};
  const MxSpan sum{d->sum_out, d->rows, d->ld_sum_out * size, width}, gain{d->gain, 1, 0, (int64_t)d->cols * 4};
  const MxSpan codes = codes_of(d, d->codes), scales = scales_of(d);
  for (const MxSpan& own : {codes, scales})
    TH_CHECK_ARG(!mx_meet(own, x) && !mx_meet(own, residual) && !mx_meet(own, sum) && !mx_meet(own, gain),
                 "th_mx_rmsnorm: codes and scales need memory of their own");
  TH_CHECK_ARG(!mx_meet(scales, codes) && !mx_meet(sum, gain) && mx_same_or_apart(sum, x) && mx_same_or_apart(sum, residual),
               "th_mx_rmsnorm: codes, scales and sum_out need memory of their own; sum_out may be x or residual");
  TH_CHECK_READY("th_mx_rmsnorm");
  MxNormK k{};
  k.rows = d->rows; k.cols = d->cols; k.chunks = (int)cdiv(d->cols, 32) * 4;
  k.x = d->x; k.ldx = d->ld_x; k.r = d->residual; k.ldr = d->ld_residual; k.h = d->sum_out; k.ldh = d->ld_sum_out;
  k.gain = d->gain; k.codes = (uint8_t*)d->codes; k.ldc = d->ld_codes; k.scales = d->scales; k.lds = d->ld_scales;
  k.inv_n = 1.f / (float)d->cols; k.eps = d->eps;
  k.e2m1 = d->mx_dtype == TH_F4E2M1;
  hipStream_t s = (hipStream_t)stream;
  if (d->x_dtype == TH_BF16) launch_norm<uint16_t>(k, s);
  else launch_norm<float>(k, s);
  TH_CHECK_LAUNCH();
  return TH_OK;
}
