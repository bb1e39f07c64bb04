// Rows in 8 bits: the inputs of the 8-bit linear layers (fp8_linear.hip, gfx950).
//
//   rows       v = x, or x * gate
//   silu_mul   v = a c / (1 + e^-c)                          (SwiGLU's product)
//   rms_norm   t = x + r in x's type (r optional), v = t / sqrt(mean t^2 + eps) (1 + w)
//
// and of each row of v, for each block of 128 columns, the e4m3 codes of v / s
// with s = 2^e the smallest power of two that max|v| <= 448 s holds for (1 for a
// block of zeros).  A float's relative step does not depend on its exponent, so a
// power of two loses nothing against max|v| / 448 but a part of the subnormal
// codes, and the matrix cores take it as it is: one e8m0 byte, 2^(byte - 127).
// Infinities and NaN give NaN codes; the scale goes by what is finite.
//
// Outputs: codes (rows, 128 kb) with zeros behind dim, scales (rows, 4 ceil(kb / 4))
// with 127 (2^0) behind block kb - 1: the products read them a word at a time.
//
// Rounding: v is computed to within a few 2^-48 (rows, rms_norm; silu_mul 8 2^-24)
// and rounded to fp32 to odd, so that the one rounding that counts, to e4m3, is that
// of v itself: rounding to nearest twice would send values next to a tie the wrong way.
// A v beyond fp32's range counts as infinite, one below it (2^-150 at most) as 0.
//
// Streams of memory: 16 lanes a block, 8 columns a lane, so that a block's maximum is
// four rotations within a row of lanes and its codes leave as 128 bytes.  Large calls
// run at the rate of a copy (5.1 TB/s): silu_mul 32768 x 4096 120 to 126 us, 5.5 TB/s; norm
// with residual 32768 x 1024 45.8 us, 5.1; rows 8191 x 2056 9.9 us, 5.1.  Few rows are
// one latency after another: 4 rows 2.3 to 3.4 us, and the call's host time above that.
#include "fp8.h"
#include "prof.h"

#include <type_traits>

namespace sa {
namespace {

__device__ __forceinline__ float top_of(const float (&v)[8]) {
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(v[i]));   // (a NaN is passed over)
  return top;
}
// the block's scale and the lane's eight codes, of top_of(v); all 16 lanes of the block are here
__device__ __forceinline__ uint2 encode_block(float (&v)[8], float top, uint32_t& byte) {
  if (__any(top == __builtin_inff())) {
    top = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[i] = no_infinity(v[i]);
      top = fmaxf(top, fabsf(v[i]));
    }
  }
  byte = scale_byte(max16(top));
  const float scale = scale_value(byte);
  return uint2{encode4(v, scale), encode4(v + 4, scale)};
}

// where a lane's codes and, by the block's first lane, its scale go
struct RowsOut {
  uint8_t* codes;
  uint8_t* scales;
  int kb, words;   // blocks and words of scales a row
};
__device__ __forceinline__ void put_block(const RowsOut& o, long row, int b, int l16, const uint2& c, uint32_t byte) {
  *reinterpret_cast<uint2*>(o.codes + (row * o.kb + b) * kQBlock + 8 * l16) = c;
  uint8_t* s = o.scales + row * 4 * o.words;
  if (l16 == 0) s[b] = static_cast<uint8_t>(byte);
  else if (b == o.kb - 1 && l16 < 4 * o.words - b) s[b + l16] = 127;
}

// eight columns of a row from k on, those at or behind dim as 0: a whole piece by 16-byte
// accesses at any address (16-byte boundaries are no faster; one element at a time took
// 3 to 4 times as long), the row's last by elements
typedef uint32_t v4u_any __attribute__((ext_vector_type(4), aligned(2)));
typedef float v4f_any __attribute__((ext_vector_type(4), aligned(4)));
template <typename T>
__device__ __forceinline__ void load8(float (&v)[8], const T* row, int k, int dim) {
  if (k + 8 <= dim) {
    if constexpr (sizeof(T) == 2) {
      const v4u_any q = *reinterpret_cast<const v4u_any*>(row + k);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = bf16lo_to_f32(q[i]);
        v[2 * i + 1] = bf16hi_to_f32(q[i]);
      }
    } else {
      const v4f_any a = *reinterpret_cast<const v4f_any*>(row + k), b = *reinterpret_cast<const v4f_any*>(row + k + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = a[i];
        v[4 + i] = b[i];
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = k + i < dim ? to_f32(row[k + i]) : 0.0f;
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* row, int k, int dim, const float (&v)[8]) {
  if (k + 8 <= dim) {
    if constexpr (sizeof(T) == 2) {
      *reinterpret_cast<v4u_any*>(row + k) = v4u_any{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]),
                                                     pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])};
    } else {
      *reinterpret_cast<v4f_any*>(row + k) = v4f_any{v[0], v[1], v[2], v[3]};
      *reinterpret_cast<v4f_any*>(row + k + 4) = v4f_any{v[4], v[5], v[6], v[7]};
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (k + i < dim) row[k + i] = from_f32<T>(v[i]);
  }
}

// x - t ln 2, for t next to x log2 e, ln 2 in two words
__device__ __forceinline__ float left_of(float x, float t) {
  return fmaf(t, 1.9046542999e-9f, fmaf(t, -0.693147182464599609375f, x));
}
// a c / (1 + e^-c) in fp64 but for the exponential and the reciprocal, 5 2^-24 off at most:
// for gates so far that e^-c nears fp32's end, and where fp32 runs out below.  e is e^-|c|,
// times 2^164 where the unit would drop its digits; of e^-200 nothing is left whatever a is
__device__ __forceinline__ double silu64(float a, float c) {
  const float b = fminf(fabsf(c), 200.0f);
  const float t = -b * kLog2e;
  const bool far = t < -115.0f;
  float e = fast_exp2(far ? t + 164.0f : t);
  e = fmaf(e, left_of(-b, t), e);
  const float d = 1.0f + (far ? 0.0f : e);
  float r = __builtin_amdgcn_rcpf(d);
  r = fmaf(fmaf(-d, r, 1.0f), r, r);
  const double s = c >= 0.0f ? 1.0 : c < -200.0f ? 0.0 : static_cast<double>(e) * (far ? 0x1p-164 : 1.0);
  return static_cast<double>(a) * c * (r * s);
}

// v = x, x * gate, or x * silu(gate); 16 lanes a block, blocks in order
enum { kPlain = 0, kGated = 1, kSilu = 2 };
template <typename T, int MODE>
__global__ __launch_bounds__(256) void rows_kernel(const T* __restrict__ x, const T* __restrict__ gate, long ldx,
                                                   long ldg, int dim, uint32_t blocks, const RowsOut o) {
  const int l16 = threadIdx.x & 15;
  const uint32_t q = blockIdx.x * 16u + (threadIdx.x >> 4);
  if (q >= blocks) return;   // (16 lanes at a time)
  const uint32_t row = q / static_cast<uint32_t>(o.kb);
  const int b = static_cast<int>(q - row * o.kb), k = kQBlock * b + 8 * l16;
  float v[8], top;
  load8<T>(v, x + row * ldx, k, dim);
  if constexpr (MODE != kPlain) {
    float c[8];
    load8<T>(c, gate + row * ldg, k, dim);
    float y[8];
    if constexpr (MODE == kGated) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float p = v[i] * c[i];
        y[i] = to_odd(p, fmaf(v[i], c[i], -p));   // (exact for bf16)
      }
      top = top_of(y);
      if (top < 0x1p-100f && top != 0.0f) {   // (fp32 loses the remainder)
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = to_odd(static_cast<double>(v[i]) * c[i]);
        top = top_of(y);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        // e^-c by the transcendental unit (2^t, 1 ulp), with what t's rounding leaves
        const float t = -c[i] * kLog2e, e = fast_exp2(t), d = 1.0f + fmaf(e, left_of(-c[i], t), e);
        float r = __builtin_amdgcn_rcpf(d);
        r = fmaf(fmaf(-d, r, 1.0f), r, r);
        y[i] = v[i] * r * c[i];   // (a c may pass fp32's range where the result does not)
      }
      top = top_of(y);
      // by the lane's own numbers: a row's codes do not depend on those beside it
      bool ends = top_of(c) > 80.0f;
      if (top < 0x1p-100f) {   // (with a product that is not 0)
#pragma unroll
        for (int i = 0; i < 8; ++i) ends |= v[i] != 0.0f && c[i] != 0.0f;
      }
      if (ends) {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = to_odd(silu64(v[i], c[i]));
        top = top_of(y);
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = y[i];
  } else {
    top = top_of(v);
  }
  uint32_t byte;
  const uint2 c = encode_block(v, top, byte);
  put_block(o, row, b, l16, c, byte);
}

// 1 / sqrt(ss inv_dim + eps): the unit's estimate in fp64 (2^-23 off at most) and one Newton
// step; 0 for a row with an infinity
__device__ __forceinline__ double rstd_of(double ss, double inv_dim, double eps) {
  const double m = fma(ss, inv_dim, eps), e = __builtin_amdgcn_rsq(m);
  return m == static_cast<double>(__builtin_inff()) ? 0.0 : e * fma(-0.5 * m, e * e, 1.5);
}

// Four fp32 roundings leave a value within four of its last steps.  Its code is then the
// exact value's unless a border of the codes or of the scale lies that near.  All have the
// last 19 bits zero: ties have five significant bits, four or fewer below 2^-6 of the
// scale, and 448 has three.  So a wave takes them in fp64 (to_odd) only where one of its
// numbers lies within six steps of such bits, a piece of 512 in 80, or where fp32 runs out:
// for small values, and for rows whose factor is beyond 2^-64 or 2^64 (64 M numbers of dim
// 1024 without residual 48 us, all in fp64 63).
// A row stays in registers between its sum of squares and its codes: W waves a row
// and V pieces of 8 columns a lane (W = 1: four rows a workgroup).  The squares are
// summed in fp64, at fp32's rate but for the widening: in fp32 the row's factor is off
// by 2^-26, and one code in some 10^7 falls on the wrong side of its tie.
template <typename T, bool RES, int V, int W>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void rms_norm_fp8_kernel(
    const T* __restrict__ x, const T* __restrict__ res, const float* __restrict__ weight, long rows, long ldx,
    int dim, double inv_dim, double eps, T* __restrict__ sum, const RowsOut o) {
  const int tid = threadIdx.x, lane = tid & 63;
  const long row = W == 1 ? blockIdx.x * 4L + (tid >> 6) : static_cast<long>(blockIdx.x);
  const int t = W == 1 ? lane : tid, l16 = tid & 15;
  if (W == 1 && row >= rows) return;   // (whole waves; no barrier below for W = 1)
  float v[V][8], w[V][8];
  double ss = 0.0, s1 = 0.0;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int k = 8 * (t + 64 * W * j);
    load8<T>(v[j], x + row * ldx, k, dim);
    if constexpr (V <= 2) load8<float>(w[j], weight, k, dim);   // (with the row: one latency)
    if constexpr (RES) {
      float r[8];
      load8<T>(r, res + row * dim, k, dim);
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        if constexpr (sizeof(T) == 2) {
          const uint32_t p = pack_bf16x2(v[j][i] + r[i], v[j][i + 1] + r[i + 1]);
          v[j][i] = bf16lo_to_f32(p);
          v[j][i + 1] = bf16hi_to_f32(p);
        } else {
          v[j][i] += r[i];
          v[j][i + 1] += r[i + 1];
        }
      }
      store8<T>(sum + row * dim, k, dim, v[j]);
    }
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const double a = v[j][i], b = v[j][i + 1];
      ss = fma(a, a, ss);
      s1 = fma(b, b, s1);
    }
  }
  ss = wave_sum64(ss + s1);
  if constexpr (W > 1) {
    __shared__ double part[W];
    if (lane == 0) part[tid >> 6] = ss;
    __syncthreads();
    ss = 0.0;
#pragma unroll 4   // (16 at a time take the registers of a second workgroup on the CU)
    for (int i = 0; i < W; ++i) ss += part[i];
  }
  const double rstd = rstd_of(ss, inv_dim, eps);
  const float hi = static_cast<float>(rstd);
  const bool far = !(rstd >= 0x1p-64 && rstd <= 0x1p64);
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int p = t + 64 * W * j, k = 8 * p, b = p >> 4;
    if constexpr (V > 2) load8<float>(w[j], weight, k, dim);
    float y[8], top = 0.0f;
    bool near = far;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      y[i] = v[j][i] * hi * (1.0f + w[j][i]);
      near |= ((__float_as_uint(y[i]) + 6u) & 0x7ffffu) <= 12u && y[i] != 0.0f;
      top = fmaxf(top, fabsf(y[i]));
    }
    if (top < 0x1p-80f) {   // (with a number that is not 0)
#pragma unroll
      for (int i = 0; i < 8; ++i) near |= v[j][i] != 0.0f;
    }
    if (__any(near)) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float a = v[j][i];
        asm volatile("" : "+v"(a));   // (widened anew: the squares' fp64 copies would fill the registers)
        y[i] = to_odd(static_cast<double>(a) * rstd * (1.0 + static_cast<double>(w[j][i])));
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[j][i] = k + i < dim ? y[i] : 0.0f;
    if (b < o.kb) {   // (16 lanes at a time)
      uint32_t byte;
      const uint2 c = encode_block(v[j], top_of(v[j]), byte);
      put_block(o, row, b, l16, c, byte);
    }
  }
}

RowsOut rows_out(void* codes, void* scales, int dim) {
  const int kb = (dim + kQBlock - 1) / kQBlock;
  return RowsOut{static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales), kb, (kb + 3) / 4};
}

template <typename T>
void rows_go(int mode, const void* x, const void* gate, long ldx, long ldg, int dim, uint32_t blocks, const RowsOut& o,
             hipStream_t s) {
  auto go = [&](auto kern) {
    hipLaunchKernelGGL(kern, dim3((blocks + 15) / 16), dim3(256), 0, s, static_cast<const T*>(x),
                       static_cast<const T*>(gate), ldx, ldg, dim, blocks, o);
  };
  if (mode == kPlain) go(rows_kernel<T, kPlain>);
  else if (mode == kGated) go(rows_kernel<T, kGated>);
  else if constexpr (sizeof(T) == 2) go(rows_kernel<T, kSilu>);
}

constexpr long kFewRows = 512;
template <typename T, bool RES>
void norm_go(const void* x, const void* res, const float* w, long rows, long ldx, int dim, double eps, void* sum,
             const RowsOut& o, hipStream_t s) {
  auto go = [&](auto kern, int waves) {
    const long grid = waves == 1 ? (rows + 3) / 4 : rows;
    hipLaunchKernelGGL(kern, dim3(grid), dim3(waves == 1 ? 256 : 64 * waves), 0, s, static_cast<const T*>(x),
                       static_cast<const T*>(res), w, rows, ldx, dim, 1.0 / dim, eps, static_cast<T*>(sum), o);
  };
  // few rows are bound by one row's latency, and take more waves for it: with fewer 1 row
  // of 1024 takes 3.5 us, so 2.7, 1 of 8192 6.4 and 3.8, 512 of 1024 4.9 and 4.0, 512 of 4096
  // 6.3 and 6.5; more rows fill the card either way, and one wave a row needs no barrier
  if (rows <= kFewRows && dim > 512 && dim <= 8192) {
    if (dim <= 2048) go(rms_norm_fp8_kernel<T, RES, 1, 4>, 4);
    else go(rms_norm_fp8_kernel<T, RES, 1, 16>, 16);
    return;
  }
  // lanes without columns cost what the others do: a row takes the sizes that leave few of
  // them (64 M numbers with residual at dim 1280 95 us, by the sizes of 2048 116, at 5120 92
  // and 97, at 20000 121 and 220; at 1024 84)
  if (dim <= 512) go(rms_norm_fp8_kernel<T, RES, 1, 1>, 1);
  else if (dim <= 1024) go(rms_norm_fp8_kernel<T, RES, 2, 1>, 1);
  else if (dim <= 1536) go(rms_norm_fp8_kernel<T, RES, 3, 1>, 1);
  else if (dim <= 2048) go(rms_norm_fp8_kernel<T, RES, 1, 4>, 4);
  else if (dim <= 2560) go(rms_norm_fp8_kernel<T, RES, 5, 1>, 1);
  else if (dim <= 4096) go(rms_norm_fp8_kernel<T, RES, 2, 4>, 4);
  else if (dim <= 6144) go(rms_norm_fp8_kernel<T, RES, 3, 4>, 4);
  else if (dim <= 8192) go(rms_norm_fp8_kernel<T, RES, 4, 4>, 4);
  else if (dim <= 10240) go(rms_norm_fp8_kernel<T, RES, 5, 4>, 4);
  else if (dim <= 16384) go(rms_norm_fp8_kernel<T, RES, 2, 16>, 16);
  else if (dim <= 24576) go(rms_norm_fp8_kernel<T, RES, 3, 16>, 16);
  else if (dim <= 32768) go(rms_norm_fp8_kernel<T, RES, 4, 16>, 16);
  else go(rms_norm_fp8_kernel<T, RES, 8, 16>, 16);
}
constexpr int kMaxNormDim = 65536;
int norm_waves(int dim) { return dim <= 1536 ? 1 : dim <= 10240 ? 4 : 16; }   // at most (as norm_go)

constexpr long kMaxBlocks = ((1L << 24) - 1) * 16;   // 16 a workgroup of 256, a grid of less than 2^32 threads
int rows_check(const char* who, int dtype, long rows, int dim, const void* codes, const void* scales) {
  SA_CHECK_ARG(dtype == kF32 || dtype == kBF16, "%s: dtype code %d", who, dtype);
  SA_CHECK_ARG(rows >= 0 && dim > 0 && dim <= (1 << 26), "%s: bad sizes rows=%ld dim=%d", who, rows, dim);
  SA_CHECK_ARG(rows < (1L << 28) && rows * ((dim + kQBlock - 1L) / kQBlock) <= kMaxBlocks,
               "%s: %ld rows of %d columns are too many", who, rows, dim);
  SA_CHECK_ARG(rows == 0 || (codes && scales), "%s: null pointer", who);
  SA_CHECK_ARG(((reinterpret_cast<uintptr_t>(codes) & 15) | (reinterpret_cast<uintptr_t>(scales) & 3)) == 0,
               "%s: codes or scales are not aligned", who);
  return 0;
}

}  // namespace
}  // namespace sa

extern "C" int sa_rows_fp8(int dtype, const void* x, const void* gate, int silu, int64_t rows, int dim, int64_t ldx,
                           int64_t ldg, void* codes, void* scales, void* stream) {
  const char* who = silu ? "sa_rows_fp8 (silu)" : "sa_rows_fp8";
  if (const int rc = sa::rows_check(who, dtype, rows, dim, codes, scales)) return rc;
  if (rows == 0) return 0;
  SA_CHECK_ARG(x && (gate || !silu), "%s: null pointer", who);
  SA_CHECK_ARG(!silu || dtype == sa::kBF16, "%s: bfloat16 alone", who);
  SA_CHECK_ARG(ldx >= dim && (!gate || ldg >= dim), "%s: row strides %ld, %ld below dim %d", who,
               static_cast<long>(ldx), static_cast<long>(ldg), dim);
  const uintptr_t size = dtype == sa::kF32 ? 4 : 2;
  SA_CHECK_ARG(((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(gate)) & (size - 1)) == 0,
               "%s: inputs are not aligned to their type", who);
  hipStream_t s = static_cast<hipStream_t>(stream);
  sa::ProfScope prof_(silu ? "silu_mul_fp8" : "rows_fp8", s);
  const sa::RowsOut o = sa::rows_out(codes, scales, dim);
  const uint32_t blocks = static_cast<uint32_t>(rows * o.kb);
  const int mode = silu ? sa::kSilu : gate ? sa::kGated : sa::kPlain;
  if (dtype == sa::kF32) sa::rows_go<float>(mode, x, gate, ldx, ldg, dim, blocks, o, s);
  else sa::rows_go<sa::bf16>(mode, x, gate, ldx, ldg, dim, blocks, o, s);
  SA_CHECK_LAUNCH(who);
  return 0;
}

extern "C" int sa_rms_norm_fp8(int dtype, const void* x, const void* residual, const float* weight, int64_t rows,
                               int dim, int64_t ldx, double eps, void* sum, void* codes, void* scales, void* stream) {
  const char* who = "sa_rms_norm_fp8";
  if (const int rc = sa::rows_check(who, dtype, rows, dim, codes, scales)) return rc;
  if (rows == 0) return 0;
  SA_CHECK_ARG(dim <= sa::kMaxNormDim, "%s: dim %d above %d", who, dim, sa::kMaxNormDim);
  const int waves = sa::norm_waves(dim);   // (four rows a workgroup where that is one)
  SA_CHECK_ARG((waves == 1 ? (rows + 3) / 4 * 256 : rows * 64 * waves) < (1L << 32),
               "%s: %ld rows of %d columns are too many", who, static_cast<long>(rows), dim);
  SA_CHECK_ARG(x && weight && (!residual == !sum), "%s: null pointer, or one of residual and sum without the other", who);
  SA_CHECK_ARG(ldx >= dim, "%s: row stride %ld below dim %d", who, static_cast<long>(ldx), dim);
  const uintptr_t size = dtype == sa::kF32 ? 4 : 2;
  SA_CHECK_ARG(((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(residual) |
                 reinterpret_cast<uintptr_t>(sum)) & (size - 1)) == 0 && (reinterpret_cast<uintptr_t>(weight) & 3) == 0,
               "%s: inputs are not aligned to their type", who);
  hipStream_t s = static_cast<hipStream_t>(stream);
  sa::ProfScope prof_("rms_norm_fp8", s);
  const sa::RowsOut o = sa::rows_out(codes, scales, dim);
  auto go = [&](auto tag) {
    using T = decltype(tag);
    residual ? sa::norm_go<T, true>(x, residual, weight, rows, ldx, dim, eps, sum, o, s)
             : sa::norm_go<T, false>(x, residual, weight, rows, ldx, dim, eps, sum, o, s);
  };
  dtype == sa::kF32 ? go(float{}) : go(sa::bf16{});
  SA_CHECK_LAUNCH(who);
  return 0;
}
