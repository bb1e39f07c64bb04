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

typedef float v16f __attribute__((ext_vector_type(16)));
// c += A B, both e4m3, 32 x 32 x 64
__device__ __forceinline__ v16f mfma_fp8(const v8i& a, const v8i& b, const v16f& c, uint32_t sa, uint32_t sb) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 0, 0, 0, static_cast<int>(sa), 0,
                                                         static_cast<int>(sb));
}
__device__ __forceinline__ v8i lds_frag(const uint8_t* p, const uint8_t* q) {
  return join16(*reinterpret_cast<const uint4*>(p), *reinterpret_cast<const uint4*>(q));
}
__device__ __forceinline__ void lds_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// A workgroup of four waves (2 by 2) computes 64 SN columns of y for 64 SM rows of x;
// a wave SN by SM squares of 32 (W as the first operand, so that a lane holds four
// neighbouring columns of one row).  A step is one block of 128 columns of K, in LDS in
// two stages that DMA fills: W as it is packed, x as rows of 128 bytes whose pieces of
// 16 are permuted by row (piece p of row r at p ^ (r & 7)), so that eight lanes read
// all banks.  Operands are held for half a step (64 columns): while the matrix cores
// take one half, the next is read, also over the steps' border, so that a step needs
// one barrier, in its middle: there this step's stage has been read by all and the
// next one has landed.
template <int SN, int SM>
__global__ __launch_bounds__(256, SN * SM > 4 ? 1 : 2) void fp8_tile_kernel(const uint8_t* __restrict__ x,
                                                                          const uint8_t* __restrict__ xs,
                                                                          const Fp8Segs sg, int M, int kb_n,
                                                                          int mtiles) {
  constexpr int BN = 64 * SN, BM = 64 * SM, kW = BN * 128, kStage = (BN + BM) * 128;
  constexpr int kPitch = 64 * SN + 16;                    // bytes of a row of y in LDS
  static_assert(4 * 32 * kPitch <= 2 * kStage, "y fits the stages");
  __shared__ __align__(16) uint8_t smem[2 * kStage + 4 * BN];
  float* bias_lds = reinterpret_cast<float*>(smem + 2 * kStage);
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 31, h = lane >> 5;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6), wn = wid & 1, wm = wid >> 1;

  // tiles in order of the XCDs, a part of the list each; in it, four rows of tiles at a time
  const int ntiles = sg.blk0[kFp8Segs], total = ntiles * mtiles;
  int id = blockIdx.x;
  {
    const int per = total >> 3, more = total & 7, xcd = id & 7;
    id = xcd * per + min(xcd, more) + (id >> 3);
  }
  const int band = id / (4 * ntiles), left = id - band * 4 * ntiles, high = min(4, mtiles - 4 * band);
  const int mt = 4 * band + left % high, nt = left / high;
  int seg = 0;
#pragma unroll
  for (int i = 1; i < kFp8Segs; ++i) seg += (i < sg.nseg && nt >= sg.blk0[i]) ? 1 : 0;
  const int N = sg.N[seg], tiles = (N + 15) >> 4, words = (kb_n + 3) >> 2;
  const int n0 = (nt - sg.blk0[seg]) * BN, m0 = mt * BM;
  const bf16* bias = sg.bias[seg];
  if (tid < BN) bias_lds[tid] = bias && n0 + tid < N ? to_f32(bias[n0 + tid]) : 0.0f;

  // DMA: 1 KB an instruction; a wave takes SN * 2 of W and SM * 2 of x
  const uint32_t ls = lds_addr(smem);
  const uint8_t* wbase = sg.W[seg] + static_cast<long>(n0 >> 4) * kb_n * 2048;
  const uint8_t* xbase = x + static_cast<long>(m0) * kb_n * 128;
  uint32_t woff[2 * SN], xoff[2 * SM];
#pragma unroll
  for (int i = 0; i < 2 * SN; ++i) {
    const int q = wid * 2 * SN + i, t = min(q >> 1, tiles - 1 - (n0 >> 4));   // (behind the last: not stored)
    woff[i] = static_cast<uint32_t>(t) * kb_n * 2048 + (q & 1) * 1024 + lane * 16;
  }
#pragma unroll
  for (int i = 0; i < 2 * SM; ++i) {
    const int r = min((wid * 2 * SM + i) * 8 + (lane >> 3), M - 1 - m0);
    xoff[i] = static_cast<uint32_t>(r) * kb_n * 128 + ((lane & 7) ^ (lane >> 3)) * 16;
  }
  auto dma_w = [&](int i, int t, uint32_t stage) __attribute__((always_inline)) {
    dma_lds16(wbase + static_cast<long>(t) * 2048, woff[i], stage + ((wid * 2 * SN + i) << 10));
  };
  auto dma_x = [&](int i, int t, uint32_t stage) __attribute__((always_inline)) {
    dma_lds16(xbase + static_cast<long>(t) * 128, xoff[i], stage + kW + ((wid * 2 * SM + i) << 10));
  };
  // scales, a word for four blocks: the rows' a lane each, the weight's one for the wave
  const uint8_t* wsp = sg.scale[seg] + static_cast<long>(min((n0 + wn * 32 * SN) >> 7, (N - 1) >> 7)) * 4 * words;
  uint32_t sx[SM], nsx[SM], sw, nsw;
  const uint8_t* xsp[SM];
#pragma unroll
  for (int j = 0; j < SM; ++j) xsp[j] = xs + static_cast<long>(min(m0 + (wm * SM + j) * 32 + c, M - 1)) * 4 * words;
  auto load_scales = [&](int g) __attribute__((always_inline)) {
    nsw = *reinterpret_cast<const uint32_t*>(wsp + 4 * g);
#pragma unroll
    for (int j = 0; j < SM; ++j) nsx[j] = *reinterpret_cast<const uint32_t*>(xsp[j] + 4 * g);
  };
  auto take_scales = [&]() __attribute__((always_inline)) {
    sw = nsw;
#pragma unroll
    for (int j = 0; j < SM; ++j) sx[j] = nsx[j];
  };

  // operands' places in a stage: piece 4 half + 2 h + i of a row
  const int wa = wn * SN * 4096 + (c >> 4) * 2048 + h * 512 + (c & 15) * 16;
  int xa[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) xa[i] = kW + wm * SM * 4096 + c * 128 + ((((i >> 1) * 4 + 2 * h + (i & 1)) ^ (c & 7)) * 16);
  v8i fw[2][SN], fx[2][SM];
  auto read_w = [&](int half, int s, int stage) __attribute__((always_inline)) {
    const uint8_t* p = smem + stage + wa + s * 4096 + half * 1024;
    fw[half][s] = lds_frag(p, p + 256);
  };
  auto read_x = [&](int half, int s, int stage) __attribute__((always_inline)) {
    const uint8_t* p = smem + stage + s * 4096;
    fx[half][s] = lds_frag(p + xa[2 * half], p + xa[2 * half + 1]);
  };
  // operand r in the order in which the products need them: one of W, those of x, the rest of W
  auto read_frag = [&](int half, int r, int stage) __attribute__((always_inline)) {
    if (r == 0) read_w(half, 0, stage);
    else if (r <= SM) read_x(half, r - 1, stage);
    else if (r < SN + SM) read_w(half, r - SM, stage);
  };
  constexpr int kReads = SN * SM >= 8 ? 1 : 2, kDma = (2 * (SN + SM) + SN * SM - 1) / (SN * SM);
  static_assert(kReads * SN * SM >= SN + SM, "all operands are read");
  v16f acc[SN][SM];
#pragma unroll
  for (int i = 0; i < SN; ++i)
#pragma unroll
    for (int j = 0; j < SM; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;

#pragma unroll
  for (int i = 0; i < 2 * SN; ++i) dma_w(i, 0, ls);
#pragma unroll
  for (int i = 0; i < 2 * SM; ++i) dma_x(i, 0, ls);
  load_scales(0);
  __builtin_amdgcn_s_waitcnt(vm_lgkm_wait<0>());
  lds_barrier();
  take_scales();
  if (kb_n > 1) {
#pragma unroll
    for (int i = 0; i < 2 * SN; ++i) dma_w(i, 1, ls + kStage);
#pragma unroll
    for (int i = 0; i < 2 * SM; ++i) dma_x(i, 1, ls + kStage);
  }
#pragma unroll
  for (int r = 0; r < SN + SM; ++r) read_frag(0, r, 0);

  // step t: MORE: a step t + 2 follows, NEXT: a step t + 1
  auto step = [&](int t, auto next, auto more) __attribute__((always_inline)) {
    constexpr bool NEXT = decltype(next)::value, MORE = decltype(more)::value;
    const int cur = (t & 1) * kStage, oth = kStage - cur;
    if (NEXT && (t & 3) == 1) load_scales(min((t >> 2) + 1, words - 1));
    // (the order is kept as written: reads and DMA go out between the products)
#pragma unroll
    for (int k = 0; k < SN * SM; ++k) {
      const int i = k / SM, j = k % SM;
      acc[i][j] = mfma_fp8(fw[0][i], fx[0][j], acc[i][j], sw, sx[j]);
#pragma unroll
      for (int r = k * kReads; r < (k + 1) * kReads; ++r) read_frag(1, r, cur);
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (NEXT) {
      __builtin_amdgcn_s_waitcnt(vm_lgkm_wait<0>());
      lds_barrier();   // this stage is read by all, the next one has landed
    }
#pragma unroll
    for (int k = 0; k < SN * SM; ++k) {
      const int i = k / SM, j = k % SM;
      acc[i][j] = mfma_fp8(fw[1][i], fx[1][j], acc[i][j], sw, sx[j]);
      if constexpr (NEXT) {
#pragma unroll
        for (int r = k * kReads; r < (k + 1) * kReads; ++r) read_frag(0, r, oth);
      }
      if constexpr (MORE) {
#pragma unroll
        for (int d = k * kDma; d < (k + 1) * kDma; ++d) {
          if (d < 2 * SN) dma_w(d, t + 2, ls + cur);
          else if (d < 2 * (SN + SM)) dma_x(d - 2 * SN, t + 2, ls + cur);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (NEXT) {
      if ((t & 3) == 3) {
        take_scales();
      } else {
        sw >>= 8;
#pragma unroll
        for (int j = 0; j < SM; ++j) sx[j] >>= 8;
      }
    }
  };
  using yes = std::integral_constant<bool, true>;
  using no = std::integral_constant<bool, false>;
  int t = 0;
  for (; t + 2 < kb_n; ++t) step(t, yes{}, yes{});
  if (t + 1 < kb_n) step(t++, yes{}, no{});
  step(t, no{}, no{});

  // rows of y through LDS, 32 at a time, the wave's own: whole pieces of 64 SN columns
  __builtin_amdgcn_s_waitcnt(kLgkmWait0);
  lds_barrier();
  uint8_t* ys = smem + wid * 32 * kPitch;
  bf16* y = sg.y[seg];
  const int nw = n0 + wn * 32 * SN;
  const bool whole = (N & 7) == 0 && (reinterpret_cast<uintptr_t>(y) & 15) == 0;
#pragma unroll
  for (int j = 0; j < SM; ++j) {
    // lane (c, h) holds columns 8 q + 4 h + e of square i for row c
#pragma unroll
    for (int i = 0; i < SN; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float4 b = *reinterpret_cast<const float4*>(bias_lds + wn * 32 * SN + 32 * i + 8 * q + 4 * h);
        *reinterpret_cast<uint2*>(ys + c * kPitch + (32 * i + 8 * q + 4 * h) * 2) =
            uint2{pack_bf16x2(acc[i][j][4 * q] + b.x, acc[i][j][4 * q + 1] + b.y),
                  pack_bf16x2(acc[i][j][4 * q + 2] + b.z, acc[i][j][4 * q + 3] + b.w)};
      }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const int mw = m0 + (wm * SM + j) * 32;
    if (whole) {
      constexpr int kLanes = 4 * SN;
#pragma unroll
      for (int r = 0; r < 32; r += 64 / kLanes) {
        const int row = r + lane / kLanes, n = nw + 8 * (lane % kLanes);
        const uint4 v = *reinterpret_cast<const uint4*>(ys + row * kPitch + 16 * (lane % kLanes));
        if (mw + row < M && n < N) *reinterpret_cast<uint4*>(y + static_cast<long>(mw + row) * N + n) = v;
      }
    } else {
      for (int e = lane; e < 32 * 32 * SN; e += 64) {
        const int row = e / (32 * SN), k = e % (32 * SN);
        if (mw + row < M && nw + k < N)
          y[static_cast<long>(mw + row) * N + nw + k] = *reinterpret_cast<const bf16*>(ys + row * kPitch + 2 * k);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
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

template <int SN, int SM>
void fp8_tile(const void* x, const void* xs, Fp8Segs& sg, int M, int kb, hipStream_t s) {
  sg.blk0[0] = 0;
  for (int i = 0; i < kFp8Segs; ++i)
    sg.blk0[i + 1] = sg.blk0[i] + (i < sg.nseg ? (sg.N[i] + 64 * SN - 1) / (64 * SN) : 0);
  const int mtiles = (M + 64 * SM - 1) / (64 * SM);
  hipLaunchKernelGGL((fp8_tile_kernel<SN, SM>), dim3(sg.blk0[kFp8Segs] * mtiles), dim3(256), 0, s,
                     static_cast<const uint8_t*>(x), static_cast<const uint8_t*>(xs), sg, M, kb, mtiles);
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
  else if (m <= 64) sa::fp8_few<4, 2, 8>(codes, scales, sg, m, kb, s);
  else {
    long big = 0;   // tiles of 256 by 256
    for (int i = 0; i < nseg; ++i) big += (sg.N[i] + 255) / 256;
    big *= (m + 255) / 256;
    if (big >= 200) sa::fp8_tile<4, 4>(codes, scales, sg, m, kb, s);
    else if (big >= 60) sa::fp8_tile<2, 2>(codes, scales, sg, m, kb, s);
    else sa::fp8_tile<1, 1>(codes, scales, sg, m, kb, s);
  }
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
