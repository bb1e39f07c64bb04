// Linear layers in 8 bits with block scales (gfx950).
//
//   y[m, n] = sum_b 2^(ex[m, b] + ew[n / 128, b]) sum_{k in b} cx[m, k] cw[n, k] + bias[n]
//
// cx, cw e4m3 codes, b blocks of 128 columns, ex and ew the exponents of the
// rows' and the weight's scales (e8m0 bytes, fp8_rows.hip).  The matrix cores take
// both scales with the operands (one byte a lane for its 32 columns), so the sums
// over all blocks stay in one fp32 accumulator and the scales cost nothing.  They
// take the products of 8 columns together, aligned to the largest exponent and cut
// below 2^-13 of it (found by products of powers of two); those sums are added in
// fp32.  A result is so off by at most 7 2^-13 sum |x w| before its rounding to bf16,
// for random numbers by 2^-18 to 2^-20 of it, far below that rounding; the form
// without the cut, bf16 operands, has half the rate.
//
// Packed weights: tiles of 16 rows and 128 columns, (N / 16, K / 128, 8, 16, 16)
// bytes: in a tile, 16 columns of its 16 rows after each other, so that 16 lanes
// read 256 bytes in a row both from memory and from LDS.  N and K are padded with
// zeros to whole tiles.  Scales: (N / 128, 4 ceil(K / 512)) bytes.
#include "common.h"
#include "prof.h"

#include <algorithm>
#include <type_traits>

namespace sa {
namespace {

constexpr int kFp8Segs = 4;
struct Fp8Segs {
  const uint8_t* W[kFp8Segs];
  const uint8_t* scale[kFp8Segs];
  const bf16* bias[kFp8Segs];
  bf16* y[kFp8Segs];
  int N[kFp8Segs];
  int blk0[kFp8Segs + 1];
  int nseg;
};

typedef int v8i __attribute__((ext_vector_type(8)));
__device__ __forceinline__ v8i join16(const uint4& a, const uint4& b) {
  return v8i{static_cast<int>(a.x), static_cast<int>(a.y), static_cast<int>(a.z), static_cast<int>(a.w),
             static_cast<int>(b.x), static_cast<int>(b.y), static_cast<int>(b.z), static_cast<int>(b.w)};
}
// c += A B, both e4m3, 16 x 16 x 128; the scale is the low byte of sa, sb
__device__ __forceinline__ v4f mfma_fp8(const v8i& a, const v8i& b, const v4f& c, uint32_t sa, uint32_t sb) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, static_cast<int>(sa), 0,
                                                          static_cast<int>(sb));
}

// A workgroup of NW waves computes R tiles of 16 columns of y for 16 CT rows of x;
// the waves take the blocks of K in turn and their sums meet in LDS.  Lane 16 g + c
// holds columns 16 g .. + 15 and 64 + 16 g .. of a block, of row c.
template <int CT, int R, int NW>
__global__ __launch_bounds__(64 * NW) void fp8_few_kernel(const uint8_t* __restrict__ x,
                                                          const uint8_t* __restrict__ xs, const Fp8Segs sg, int M,
                                                          int kb_n) {
  __shared__ float part[NW * R * CT * 256];
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, c = lane & 15, g = lane >> 4;
  const int across = sg.blk0[kFp8Segs];   // workgroups a row of tiles
  const int bid = blockIdx.x % across, m0 = blockIdx.x / across * 16 * CT;
  int seg = 0;
#pragma unroll
  for (int i = 1; i < kFp8Segs; ++i) seg += (i < sg.nseg && bid >= sg.blk0[i]) ? 1 : 0;
  const int N = sg.N[seg], tiles = (N + 15) >> 4, words = (kb_n + 3) >> 2;
  const int t0 = (bid - sg.blk0[seg]) * R;
  const uint8_t* W = sg.W[seg];
  const uint8_t* S = sg.scale[seg];

  v4f acc[R][CT];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int t = 0; t < CT; ++t) acc[r][t] = v4f{0.f, 0.f, 0.f, 0.f};
  for (int kb = wid; kb < kb_n; kb += NW) {
    v8i w[R], xf[CT];
    uint32_t sw[R], sx[CT];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int t = min(t0 + r, tiles - 1);   // (behind the last: not stored)
      const uint4* p = reinterpret_cast<const uint4*>(W + (static_cast<long>(t) * kb_n + kb) * 2048) + lane;
      w[r] = join16(p[0], p[64]);
      sw[r] = S[static_cast<long>(t >> 3) * 4 * words + kb];
    }
#pragma unroll
    for (int t = 0; t < CT; ++t) {
      const long row = min(m0 + 16 * t + c, M - 1);
      const uint4* p = reinterpret_cast<const uint4*>(x + (row * kb_n + kb) * 128) + g;
      xf[t] = join16(p[0], p[4]);
      sx[t] = xs[row * 4 * words + kb];
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int t = 0; t < CT; ++t) acc[r][t] = mfma_fp8(w[r], xf[t], acc[r][t], sw[r], sx[t]);
  }
  // lane (c, g) holds columns 4 g + e of the tile for row 16 t + c of x
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int t = 0; t < CT; ++t)
      *reinterpret_cast<float4*>(part + ((wid * CT + t) * 16 + c) * 16 * R + 16 * r + 4 * g) =
          make_float4(acc[r][t][0], acc[r][t][1], acc[r][t][2], acc[r][t][3]);
  __syncthreads();
  const bf16* bias = sg.bias[seg];
  bf16* y = sg.y[seg];
  for (int e = tid; e < R * CT * 256; e += 64 * NW) {
    const int row = m0 + e / (16 * R), n = 16 * t0 + e % (16 * R);
    float v = 0.0f;
#pragma unroll
    for (int i = 0; i < NW; ++i) v += part[i * R * CT * 256 + e];
    if (row < M && n < N) y[static_cast<long>(row) * N + n] = from_f32<bf16>(v + (bias ? to_f32(bias[n]) : 0.0f));
  }
}

// the weights in bf16, (N, K) row-major; a code times its scale is a bf16 number
// (but for scales below 2^-117).  One workgroup a tile and block.
__global__ __launch_bounds__(128) void fp8_dequant_kernel(const uint8_t* __restrict__ W,
                                                          const uint8_t* __restrict__ scale, bf16* __restrict__ out,
                                                          int N, int K, int kb_n) {
  const int kb = blockIdx.x % kb_n, tile = blockIdx.x / kb_n;
  const int j = threadIdx.x >> 4, l = threadIdx.x & 15, half = l & 1;   // piece of 16 columns, its half
  const uint32_t byte = scale[static_cast<long>(tile >> 3) * 4 * ((kb_n + 3) >> 2) + kb];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = (l >> 1) + 8 * i, n = 16 * tile + r, k = 128 * kb + 16 * j + 8 * half;
    const uint2 q = *reinterpret_cast<const uint2*>(W + static_cast<long>(blockIdx.x) * 2048 + j * 256 + r * 16 + 8 * half);
    if (n >= N) continue;
    const uint32_t u[2] = {q.x, q.y};
    bf16* o = out + static_cast<long>(n) * K + k;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float v = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(u[e >> 2] >> (8 * (e & 3))), 0);
      if (k + e < K) o[e] = from_f32<bf16>(ldexpf(v, static_cast<int>(byte) - 127));
    }
  }
}

template <int CT, int R, int NW>
void fp8_few(const void* x, const void* xs, Fp8Segs& sg, int M, int kb, hipStream_t s) {
  sg.blk0[0] = 0;
  for (int i = 0; i < kFp8Segs; ++i)
    sg.blk0[i + 1] = sg.blk0[i] + (i < sg.nseg ? ((sg.N[i] + 15) / 16 + R - 1) / R : 0);
  hipLaunchKernelGGL((fp8_few_kernel<CT, R, NW>), dim3(sg.blk0[kFp8Segs] * ((M + 16 * CT - 1) / (16 * CT))),
                     dim3(64 * NW), 0, s, static_cast<const uint8_t*>(x), static_cast<const uint8_t*>(xs), sg, M, kb);
}

}  // namespace
}  // namespace sa

extern "C" int sa_fp8_linear(const void* codes, const void* scales, int64_t M, int K, int nseg,
                             const int64_t* matrices, void* stream) {
  const char* who = "sa_fp8_linear";
  SA_CHECK_ARG(M >= 1 && M <= (1 << 24) && K > 0 && K <= (1 << 22), "%s: M %ld must be 1..2^24 and K %d 1..2^22", who,
               static_cast<long>(M), K);
  SA_CHECK_ARG(nseg >= 1 && nseg <= sa::kFp8Segs, "%s: %d weight matrices, 1..%d allowed", who, nseg, sa::kFp8Segs);
  SA_CHECK_ARG(codes && scales && matrices, "%s: null pointer", who);
  SA_CHECK_ARG(((reinterpret_cast<uintptr_t>(codes) & 15) | (reinterpret_cast<uintptr_t>(scales) & 3)) == 0,
               "%s: codes or scales of x are not aligned", who);
  sa::Fp8Segs sg{};
  sg.nseg = nseg;
  long tiles = 0;
  for (int i = 0; i < nseg; ++i) {
    const int64_t* m = matrices + 5 * i;   // packed, scales, bias, y, N
    SA_CHECK_ARG(m[0] && m[1] && m[3] && m[4] > 0 && m[4] <= (1L << 24), "%s: weight matrix %d: null pointer or N %ld",
                 who, i, static_cast<long>(m[4]));
    SA_CHECK_ARG((m[0] & 15) == 0 && (m[1] & 3) == 0 && ((m[2] | m[3]) & 1) == 0, "%s: weight matrix %d is not aligned",
                 who, i);
    tiles += (m[4] + 15) / 16;
    sg.W[i] = reinterpret_cast<const uint8_t*>(m[0]);
    sg.scale[i] = reinterpret_cast<const uint8_t*>(m[1]);
    sg.bias[i] = reinterpret_cast<const sa::bf16*>(m[2]);
    sg.y[i] = reinterpret_cast<sa::bf16*>(m[3]);
    sg.N[i] = static_cast<int>(m[4]);
  }
  SA_CHECK_ARG(tiles * ((M + 63) / 64) < (1L << 23), "%s: %ld rows and %ld columns are too many", who,
               static_cast<long>(M), 16 * tiles);   // (2^32 threads a grid)
  hipStream_t s = static_cast<hipStream_t>(stream);
  sa::ProfScope prof_("fp8_linear", s);
  const int kb = (K + 127) / 128, m = static_cast<int>(M);
  if (m <= 16) sa::fp8_few<1, 1, 8>(codes, scales, sg, m, kb, s);
  else if (m <= 32) sa::fp8_few<2, 1, 8>(codes, scales, sg, m, kb, s);
  else sa::fp8_few<4, 2, 8>(codes, scales, sg, m, kb, s);
  SA_CHECK_LAUNCH(who);
  return 0;
}

extern "C" int sa_fp8_dequant_bf16(const void* packed, const void* scales, int N, int K, void* out, void* stream) {
  const char* who = "sa_fp8_dequant_bf16";
  SA_CHECK_ARG(N > 0 && K > 0, "%s: bad sizes N=%d K=%d", who, N, K);
  SA_CHECK_ARG(packed && scales && out, "%s: null pointer", who);
  SA_CHECK_ARG((reinterpret_cast<uintptr_t>(packed) & 7) == 0, "%s: packed weights are not aligned", who);
  const long kb = (K + 127L) / 128, blocks = ((N + 15L) / 16) * kb;
  SA_CHECK_ARG(blocks < (1L << 25), "%s: weights too large", who);   // (2^32 threads a grid)
  hipStream_t s = static_cast<hipStream_t>(stream);
  sa::ProfScope prof_("fp8_dequant", s);
  hipLaunchKernelGGL(sa::fp8_dequant_kernel, dim3(blocks), dim3(128), 0, s, static_cast<const uint8_t*>(packed),
                     static_cast<const uint8_t*>(scales), static_cast<sa::bf16*>(out), N, K, static_cast<int>(kb));
  SA_CHECK_LAUNCH(who);
  return 0;
}
