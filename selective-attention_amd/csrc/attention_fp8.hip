// Paged GQA decode attention over a cache held in 8 bits (gfx950).
//
// A block is one page of tokens of one kv head.  A full block's keys are e4m3
// codes k_pages (num_pages, Hkv, ps, D) with one scale k_scale (num_pages,
// Hkv), its values codes v_pages (num_pages, Hkv, D, ps), transposed, with
// v_scale; a code stands for code * scale, and the scales are powers of two.
// A row's open block, the seq_len % ps tokens behind its last full page, is in
// bfloat16: k_tail (batch, Hkv, ps, D), v_tail (batch, Hkv, D, ps).
//
//   o = sum_j p_j v_j / sum_j p_j,   p_j = 2^(log2(e) (scale q.k_j +
//   [j not the newest] bias_j) - m),  m the running maximum
//
// The split is stream-K over 64-key tiles, as in the bf16 decode (attention.hip):
// one resident round of W one-wave workgroups, each the same number of tiles
// of the (row, kv head, tile) list, partial sums joined by the merge kernel.
// Short tables take one workgroup a (row, kv head) instead and need no merge.
// What differs from the bf16 cache is the tile: 64 D codes are a quarter to a half of the
// registers of the bf16 tile, widened to bf16 MFMA operands right before
// their product (v_cvt_scalef32_pk_bf16_fp8, two codes an instruction, which
// multiplies by the block's power of two on the way: exact, every e4m3 number
// times 2^e is a bf16 number).
//
// Operand order.  Lane (c, g) = (lane & 15, lane >> 4) loads 16 codes at once.
// K: dims 64 s + 16 g .. + 15 of key 16 (c >> 2) + 4 kt + (c & 3), the k-steps
// 2 s and 2 s + 1 of the contraction over dims (q is loaded in the same
// order).  The score tile kt then leaves lane (c, g) the keys 16 g + 4 kt + i,
// i = 0..3, of query column c, so the four tiles give it keys 16 g .. + 15:
// what its V^T load of 16 codes (dim 16 t + c, keys 16 g .. + 15) contracts.
#include "common.h"
#include "decode.h"
#include "prof.h"

#include <type_traits>

namespace sa {
namespace {

// 8 e4m3 codes (two words) times the power of two `scale` as a bf16 fragment
__device__ __forceinline__ v8bf widen8(uint32_t lo, uint32_t hi, float scale) {
  const uint4 r = {
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true))};
  return __builtin_bit_cast(v8bf, r);
}

// 16 bytes of a buffer at a lane's and a constant offset.  NT: non-temporal, the
// line is not kept.  The codes are read once a step, and without it the caches'
// own traffic costs a tenth: 64 rows of 1 to 32 thousand keys, 8 heads of 128,
// 435 us; 386 with it, 6.3 TB/s.  Only where a tile takes whole lines: at 128 keys a
// page the two tiles of a V^T row share its line (5.3 TB/s without, 4.3 with).
template <bool NT>
__device__ __forceinline__ uint4 buf_load16(__amdgpu_buffer_rsrc_t r, unsigned off) {
  return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, NT ? 2 : 0));
}

// Eight weights as two bf16 operands, p = hi + lo to 2^-16 of p.  One operand
// alone would round each weight by up to 2^-8, as much as the output's own rounding
// and more where values cancel.  The matrix cores stand idle for most of the time
// that the codes' bytes take: 64 rows of 1 to 32 thousand keys, 8 heads of 128, 386 us,
// 380 with the one operand; 4 rows of 5000 to 8193, 16 gated heads of 64, which
// latency bounds, 21.1 and 19.7.
struct SplitP {
  v8bf hi, lo;
};
__device__ __forceinline__ SplitP split_p(const v4f& a, const v4f& b) {
  SplitP r;
  r.hi = pack_p(a, b);
  const uint4 u = __builtin_bit_cast(uint4, r.hi);
  r.lo = pack_p(v4f{a[0] - bf16lo_to_f32(u.x), a[1] - bf16hi_to_f32(u.x), a[2] - bf16lo_to_f32(u.y), a[3] - bf16hi_to_f32(u.y)},
                v4f{b[0] - bf16lo_to_f32(u.z), b[1] - bf16hi_to_f32(u.z), b[2] - bf16lo_to_f32(u.w), b[3] - bf16hi_to_f32(u.w)});
  return r;
}
// two bf16 with infinities and NaN as 0: an open block's infinite value meets a
// weight's low part, 0 or of either sign, as 0
__device__ __forceinline__ uint32_t finite_pair(uint32_t w) {
  w = (w & 0x7f80u) == 0x7f80u ? w & 0xffff0000u : w;
  return (w & 0x7f800000u) == 0x7f800000u ? w & 0xffffu : w;
}

struct Slot8 {
  long blk;          // (page, kv head) of the tile in the pool
  int k0;            // the tile's first key inside its page
  bool ok;           // a valid page id: else the tile has no keys
  float ks, vs;      // the block's scales
};

struct Fp8Cache {
  const uint8_t *k, *v;
  const float *k_scale, *v_scale;
  const bf16 *k_tail, *v_tail;
  const int32_t* page_table;
  const float* bias;
  int Hkv, max_pages, num_pages;
};

// One wave over the tiles t_begin, t_begin + S, ... < t_end of the n keys of (row
// bi, kv head kvh): its sums O^T (acc), their reference m and weight l, for the
// query heads in qf, those of columns c < grp.
template <int D, bool BIAS, int PS, int S>
__device__ __forceinline__ void row_tiles(const Fp8Cache& kv, int bi, int kvh, int n, int t_begin, int t_end,
                                          int grp, float scale_log2, const v8bf (&qf)[D / 32],
                                          v4f (&acc)[D / 16], float& m, float& l) {
  constexpr int DT = D / 16, KS = D / 32, K2 = D / 64;
  constexpr int ps = PS, tshift = PS == 128 ? 1 : 0;   // log2(64-key tiles per page)
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const int Hkv = kv.Hkv, num_pages = kv.num_pages;
  const float* key_bias = kv.bias;
  // the lane's place in a tile of codes, K (key, dim) and V^T (dim, key)
  const unsigned koff = static_cast<unsigned>((16 * (c >> 2) + (c & 3)) * D + 16 * g);
  const unsigned voff = static_cast<unsigned>(c * ps + 16 * g);
  const int t_open = (n / ps) << tshift;   // first tile of the open block
  const int t_close = min(t_end, t_open);
  const int32_t* prow = kv.page_table + static_cast<long>(bi) * kv.max_pages;

  // scale, bias (not on the newest key) and mask of the score tiles; entry
  // (kt, i) is key 16 g + 4 kt + i of the tile at sequence position pos0.
  // keep[kt] gets the byte mask of the keys that take part.
  auto finish = [&](v4f (&sc)[4], const float* brow, int nk, int pos0, uint32_t (&keep)[4])
                    __attribute__((always_inline)) {
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
      float4 bv = make_float4(0.f, 0.f, 0.f, 0.f);
      if constexpr (BIAS) bv = *reinterpret_cast<const float4*>(brow + 16 * g + 4 * kt);
      const float bs[4] = {bv.x, bv.y, bv.z, bv.w};
      keep[kt] = 0u;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = 16 * g + 4 * kt + i;
        bool on = key < nk;
        float val = sc[kt][i] * scale_log2;
        if constexpr (BIAS) {
          const bool newest = key == n - 1 - pos0;
          val = newest ? val : val + bs[i] * kLog2e;
          on = on && (newest || bs[i] != kNegInf);   // a dropped key counts for nothing, whatever it holds
        }
        sc[kt][i] = on && c < grp ? val : kNegInf;
        keep[kt] |= on ? 0xffu << (8 * i) : 0u;
      }
    }
  };

  // full blocks, in runs of at most 64 pages: lane j holds the id and the
  // scales of the run's page p0 + j
  int r0 = t_begin;
  while (r0 < t_close) {
    const int p0 = r0 >> tshift;
    const int r1 = min(t_close, (p0 + 64) << tshift);
    const int my_page = lane <= ((r1 - 1) >> tshift) - p0 ? prow[p0 + lane] : -1;
    const bool my_ok = my_page >= 0 && my_page < num_pages;
    // invalid ids read page 0, which exists, and contribute no keys
    const long my_blk = static_cast<long>(my_ok ? my_page : 0) * Hkv + kvh;
    const float my_ks = kv.k_scale[my_blk], my_vs = kv.v_scale[my_blk];
    auto slot_of = [&](int t) {
      const int j = (t >> tshift) - p0;
      const int page = __builtin_amdgcn_readlane(my_page, j);
      Slot8 sl;
      sl.ok = page >= 0 && page < num_pages;
      sl.blk = static_cast<long>(sl.ok ? page : 0) * Hkv + kvh;
      sl.k0 = (t & tshift) * 64;
      sl.ks = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(my_ks), j));
      sl.vs = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(my_vs), j));
      return sl;
    };
    uint4 kf[4][K2], vf[DT];
    auto load_k = [&](const Slot8& sl) __attribute__((always_inline)) {
      const __amdgpu_buffer_rsrc_t r = make_rsrc(kv.k + (sl.blk * ps + sl.k0) * D);
#pragma unroll
      for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int s = 0; s < K2; ++s) kf[kt][s] = buf_load16<true>(r, koff + (4 * kt * D + 64 * s));
    };
    auto load_v = [&](const Slot8& sl) __attribute__((always_inline)) {
      const __amdgpu_buffer_rsrc_t r = make_rsrc(kv.v + sl.blk * ps * D + sl.k0);
#pragma unroll
      for (int t = 0; t < DT; ++t) vf[t] = buf_load16<PS == 64>(r, voff + 16 * t * ps);
    };
    Slot8 cur = slot_of(r0);
    load_k(cur);
    load_v(cur);
    auto tile = [&](auto more_c, int t, const Slot8& nxt) __attribute__((always_inline)) {
      constexpr bool kMore = decltype(more_c)::value;
      v4f sc[4];
#pragma unroll
      for (int kt = 0; kt < 4; ++kt) {
        sc[kt] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < K2; ++s) {
          const uint4 x = kf[kt][s];
          sc[kt] = mfma_bf16(widen8(x.x, x.y, cur.ks), qf[2 * s], sc[kt]);
          sc[kt] = mfma_bf16(widen8(x.z, x.w, cur.ks), qf[2 * s + 1], sc[kt]);
        }
      }
      if constexpr (kMore) load_k(nxt);
      uint32_t keep[4];
      finish(sc, key_bias + cur.blk * ps + cur.k0, cur.ok ? 64 : 0, 64 * t, keep);
      softmax_block<4, DT>(sc, acc, m, l);
      const SplitP pa = split_p(sc[0], sc[1]), pb = split_p(sc[2], sc[3]);
      if (cur.ok) {
#pragma unroll
        for (int tt = 0; tt < DT; ++tt) {
          uint4 x = vf[tt];
          if constexpr (BIAS) x = uint4{x.x & keep[0], x.y & keep[1], x.z & keep[2], x.w & keep[3]};
          const v8bf va = widen8(x.x, x.y, cur.vs), vb = widen8(x.z, x.w, cur.vs);
          acc[tt] = mfma_bf16(va, pa.hi, acc[tt]);
          acc[tt] = mfma_bf16(vb, pb.hi, acc[tt]);
          acc[tt] = mfma_bf16(va, pa.lo, acc[tt]);
          acc[tt] = mfma_bf16(vb, pb.lo, acc[tt]);
        }
      }
      if constexpr (kMore) load_v(nxt);
    };
    int t = r0;
    for (; t + S < r1; t += S) {
      const Slot8 nxt = slot_of(t + S);
      tile(BoolC<true>{}, t, nxt);
      cur = nxt;
    }
    tile(BoolC<false>{}, t, cur);
    r0 = t + S;
  }

  // the open block, in bf16
  int t_first = t_begin;
  if (t_open > t_begin) t_first += (t_open - t_begin + S - 1) / S * S;
  for (int t = t_first; t < t_end; t += S) {
    const int page = prow[t >> tshift];
    if (page < 0 || page >= num_pages) continue;   // wave-uniform
    const int k0 = (t & tshift) * 64, nk = min(64, n - 64 * t);
    const long tail = (static_cast<long>(bi) * Hkv + kvh) * ps * D;
    const __amdgpu_buffer_rsrc_t kb = make_rsrc(kv.k_tail + tail + k0 * D), vb = make_rsrc(kv.v_tail + tail + k0);
    v4f sc[4];
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
      sc[kt] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        sc[kt] = mfma_bf16(buf_load_v8bf(kb, 2 * koff + 2 * (4 * kt * D + 64 * (ks >> 1) + 8 * (ks & 1)), 0),
                           qf[ks], sc[kt]);
    }
    uint32_t keep[4];
    finish(sc, key_bias + (static_cast<long>(page) * Hkv + kvh) * ps + k0, nk, 64 * t, keep);
    softmax_block<4, DT>(sc, acc, m, l);
    // two keys a word: byte masks to 16-bit masks (slots past nk hold what
    // the buffer held, NaN perhaps)
    uint32_t km[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      km[i] = __builtin_amdgcn_perm(0u, keep[i >> 1], (i & 1) ? 0x03030202u : 0x01010000u);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const SplitP p = split_p(sc[2 * h], sc[2 * h + 1]);
#pragma unroll
      for (int tt = 0; tt < DT; ++tt) {
        uint4 x = buf_load16<false>(vb, 2 * voff + 16 * h + 32 * tt * ps);
        x = uint4{x.x & km[4 * h], x.y & km[4 * h + 1], x.z & km[4 * h + 2], x.w & km[4 * h + 3]};
        acc[tt] = mfma_bf16(__builtin_bit_cast(v8bf, x), p.hi, acc[tt]);
        x = uint4{finite_pair(x.x), finite_pair(x.y), finite_pair(x.z), finite_pair(x.w)};
        acc[tt] = mfma_bf16(__builtin_bit_cast(v8bf, x), p.lo, acc[tt]);
      }
    }
  }
}

// the group's query heads, column c = lane & 15, dims in the order of the K operand
template <int D>
__device__ __forceinline__ void load_q(v8bf (&qf)[D / 32], const bf16* q, int grp) {
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const bf16* row = q + min(c, grp - 1) * D;
#pragma unroll
  for (int ks = 0; ks < D / 32; ++ks)
    qf[ks] = c < grp ? load_v8bf(row + 64 * (ks >> 1) + 16 * g + 8 * (ks & 1)) : zero_v8bf();
}

template <int D, bool BIAS, int PS>
__global__ __launch_bounds__(64, 2) void paged_decode_fp8_kernel(
    const bf16* __restrict__ q, const Fp8Cache kv, const int32_t* __restrict__ seq_lens,
    int32_t* __restrict__ cum_row, float* __restrict__ part_o, float* __restrict__ part_ml, int b,
    int Hq, int W, float scale_log2) {
  constexpr int DT = D / 16, ps = PS;
  const int Hkv = kv.Hkv, max_pages = kv.max_pages;
  const int w = blockIdx.x;
  const int lane = threadIdx.x, c = lane & 15, g = lane >> 4;
  // row plan: up to 64 rows each wave forms it in its lanes (lane r holds row
  // r's 64-key tiles and the tiles before it), wave 0 stores it for the merge
  const bool lane_plan = b <= 64;
  int ex_l = 0, tot = 0;
  if (lane_plan) {
    const int nb = lane < b ? (decode_row_len(seq_lens, lane, max_pages, ps) + 63) >> 6 : 0;
    int incl = nb;
#pragma unroll
    for (int o2 = 1; o2 < 64; o2 <<= 1) {
      const int t = __shfl_up(incl, o2, 64);
      if (lane >= o2) incl += t;
    }
    ex_l = incl - nb;
    tot = __builtin_amdgcn_readlane(incl, 63);
    if (w == 0 && lane < b) {
      cum_row[lane + 1] = incl;
      if (lane == 0) cum_row[0] = 0;
    }
  }
  auto crow = [&](int r) -> int {   // tiles of the rows before r, r in [0, b]
    return lane_plan ? (r < 64 ? __builtin_amdgcn_readlane(ex_l, r) : tot) : cum_row[r];
  };
  const long T = static_cast<long>(Hkv) * crow(b);
  W = static_cast<int>(min(static_cast<long>(W), T));   // every wave gets a tile
  if (w >= W) return;
  long gt = decode_wave_begin(w, T, W);
  const long gt_end = decode_wave_begin(w + 1, T, W);
  const int grp = Hq / Hkv;

  // row of the first tile: the largest r with Hkv * cum_row[r] <= gt
  int bi = 0;
  if (lane_plan) {
    bi = __popcll(__ballot(lane < b && static_cast<long>(Hkv) * ex_l <= gt)) - 1;
  } else {
    int lo = 0, span = b;   // 64-ary search, answer in [lo, lo + span)
    while (span > 1) {
      const int step = (span + 63) >> 6;
      const int r = lo + lane * step;
      const bool le = r < lo + span && static_cast<long>(Hkv) * cum_row[r] <= gt;
      const int k = __popcll(__ballot(le));   // >= 1: lane 0 reads cum_row[lo]
      const int nlo = lo + (k - 1) * step;
      span = min(step, lo + span - nlo);
      lo = nlo;
    }
    bi = lo;
  }

  while (gt < gt_end) {
    long rb = static_cast<long>(Hkv) * crow(bi);
    int tb = crow(bi + 1) - crow(bi);
    while (gt >= rb + static_cast<long>(Hkv) * tb) {   // rows with no tiles
      ++bi;
      rb = static_cast<long>(Hkv) * crow(bi);
      tb = crow(bi + 1) - crow(bi);
    }
    const int off = static_cast<int>(gt - rb);
    const int kvh = off / tb;
    const int t_begin = off - kvh * tb;
    const int t_end = t_begin + static_cast<int>(min(gt_end - gt, static_cast<long>(tb - t_begin)));
    const int n = decode_row_len(seq_lens, bi, max_pages, ps);
    v8bf qf[D / 32];
    load_q<D>(qf, q + (static_cast<long>(bi) * Hq + kvh * grp) * D, grp);
    float m = kNegInf, l = 0.0f;
    v4f acc[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t) acc[t] = v4f{0.f, 0.f, 0.f, 0.f};
    row_tiles<D, BIAS, PS, 1>(kv, bi, kvh, n, t_begin, t_end, grp, scale_log2, qf, acc, m, l);

    // partial of this segment: O^T[d][q] unnormalised, with m (log2 domain) and l
    const long seg = static_cast<long>(bi) * Hkv + kvh + w;
    if (c < grp) {
      float* po = part_o + (seg * grp + c) * D;
#pragma unroll
      for (int t = 0; t < DT; ++t)
        *reinterpret_cast<float4*>(po + 16 * t + 4 * g) = make_float4(acc[t][0], acc[t][1], acc[t][2], acc[t][3]);
      if (g == 0) {
        part_ml[(seg * grp + c) * 2] = m;
        part_ml[(seg * grp + c) * 2 + 1] = l;
      }
    }
    gt += t_end - t_begin;
  }
}

// Short tables: one workgroup a (row, kv head), its waves taking the row's tiles in
// turn and joining in LDS (32 KB of sums O^T), so that no second launch and no workspace follow.  The
// rows' own lengths stand on the device; the table's width, which bounds them, is
// what the host can go by.
template <int D>
constexpr int kShortWaves = 512 / D;   // (half or twice as many: 16 rows of 1024 keys, D 64, 11.8 or 15.7 us; 10.2 so)
template <int D, bool BIAS, int PS>
__global__ __launch_bounds__(64 * kShortWaves<D>) void paged_decode_fp8_short_kernel(
    const bf16* __restrict__ q, const Fp8Cache kv, const int32_t* __restrict__ seq_lens,
    bf16* __restrict__ o, int Hq, float scale_log2) {
  constexpr int DT = D / 16, NW = kShortWaves<D>;
  __shared__ float so[NW][16][D];
  __shared__ float sm[NW][16], sl[NW][16];
  const int kvh = blockIdx.x % kv.Hkv, bi = blockIdx.x / kv.Hkv, grp = Hq / kv.Hkv;
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = decode_row_len(seq_lens, bi, kv.max_pages, PS);
  const bf16* qg = q + (static_cast<long>(bi) * Hq + kvh * grp) * D;
  v8bf qf[D / 32];
  load_q<D>(qf, qg, grp);
  float m = kNegInf, l = 0.0f;
  v4f acc[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) acc[t] = v4f{0.f, 0.f, 0.f, 0.f};
  row_tiles<D, BIAS, PS, NW>(kv, bi, kvh, n, wid, (n + 63) >> 6, grp, scale_log2, qf, acc, m, l);
  if (c < grp) {
#pragma unroll
    for (int t = 0; t < DT; ++t)
      *reinterpret_cast<float4*>(&so[wid][c][16 * t + 4 * g]) = make_float4(acc[t][0], acc[t][1], acc[t][2], acc[t][3]);
    if (g == 0) {
      sm[wid][c] = m;
      sl[wid][c] = l;
    }
  }
  __syncthreads();
  bf16* og = o + (static_cast<long>(bi) * Hq + kvh * grp) * D;
  for (int e = tid; e < grp * D / 2; e += 64 * NW) {
    const int col = 2 * e / D, d = 2 * e % D;
    float M = kNegInf;
#pragma unroll
    for (int i = 0; i < NW; ++i) M = fmaxf(M, sm[i][col]);
    float L = 0.0f, a0 = 0.0f, a1 = 0.0f;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      const float w = sm[i][col] == kNegInf ? 0.0f : fast_exp2(sm[i][col] - M);
      const float2 v = *reinterpret_cast<const float2*>(&so[i][col][d]);
      L = fmaf(w, sl[i][col], L);
      a0 = fmaf(w, v.x, a0);
      a1 = fmaf(w, v.y, a1);
    }
    const float inv = L > 0.0f ? 1.0f / L : 0.0f;
    *reinterpret_cast<uint32_t*>(og + 2 * e) = pack_bf16x2(a0 * inv, a1 * inv);
  }
}

// Joins the segments of one (batch row, query head): sum_s w_s o_s / sum_s w_s l_s,
// w_s = 2^(m_s - max m), in the order of the segments whatever the launch.  A step
// behind the stream-K launch with little data, so latency is what counts: four
// waves, each a quarter of the segments with eight loads in flight (attention of 1
// row of 32000 keys, 8 heads of 128, 256 segments a head: 42 us with one wave a
// head, as the bf16 cache's merge has it, 24 so; 4 rows of 6600, 16 heads of 64:
// 3 us less, 21.3).
template <int D>
__global__ __launch_bounds__(256) void paged_decode_fp8_merge_kernel(
    const float* __restrict__ part_o, const float* __restrict__ part_ml,
    const int32_t* __restrict__ cum_row, bf16* __restrict__ o, int b, int Hq, int Hkv, int W) {
  constexpr int SPW = 128 / D;   // segments a wave takes at once, two dims a lane
  constexpr int kMergeSegs = 512;   // segments whose weights stand in LDS at once
  __shared__ float wsh[kMergeSegs];
  __shared__ float red[4][128];
  __shared__ float lred[4];
  const int qh = blockIdx.x % Hq, bi = blockIdx.x / Hq;
  const int grp = Hq / Hkv, kvh = qh / grp, qi = qh % grp;
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  bf16* orow = o + (static_cast<long>(bi) * Hq + qh) * D;
  const int c0 = cum_row[bi], tb = cum_row[bi + 1] - c0;
  if (tb <= 0) {   // no keys
    if (2 * tid < D) *reinterpret_cast<uint32_t*>(orow + 2 * tid) = 0u;
    return;
  }
  const long T = static_cast<long>(Hkv) * cum_row[b];
  W = static_cast<int>(min(static_cast<long>(W), T));   // as in the decode kernel
  const long g0 = static_cast<long>(Hkv) * c0 + static_cast<long>(kvh) * tb;
  const int w0 = decode_wave_of(g0, T, W), nseg = decode_wave_of(g0 + tb - 1, T, W) - w0 + 1;
  const long slot0 = static_cast<long>(bi) * Hkv + kvh + w0;
  auto ml_of = [&](int s) { return *reinterpret_cast<const float2*>(part_ml + ((slot0 + s) * grp + qi) * 2); };
  float M = kNegInf;
  for (int s = lane; s < nseg; s += 64) M = fmaxf(M, ml_of(s).x);
  M = wave_max(M);   // every wave for itself
  float L = 0.0f, a0 = 0.0f, a1 = 0.0f;
  const int half = lane / (D / 2), d = 2 * (lane % (D / 2));
  for (int s0 = 0; s0 < nseg; s0 += kMergeSegs) {
    const int ns = min(kMergeSegs, nseg - s0);
    if (s0 > 0) __syncthreads();
    for (int s = tid; s < ns; s += 256) {
      const float2 ml = ml_of(s0 + s);
      const float w = ml.x == kNegInf ? 0.0f : fast_exp2(ml.x - M);
      wsh[s] = w;
      L += w * ml.y;
    }
    __syncthreads();
#pragma unroll 8
    for (int s = SPW * wid + half; s < ns; s += 4 * SPW) {
      const float2 v = *reinterpret_cast<const float2*>(part_o + ((slot0 + s0 + s) * grp + qi) * D + d);
      a0 = fmaf(wsh[s], v.x, a0);
      a1 = fmaf(wsh[s], v.y, a1);
    }
  }
  L = wave_sum(L);
  if (lane == 0) lred[wid] = L;
  if constexpr (SPW == 2) {
    a0 += __shfl_xor(a0, 32, 64);
    a1 += __shfl_xor(a1, 32, 64);
  }
  if (half == 0) *reinterpret_cast<float2*>(&red[wid][d]) = make_float2(a0, a1);
  __syncthreads();
  if (2 * tid < D) {
    const float l = (lred[0] + lred[1]) + (lred[2] + lred[3]);
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    const float2 r0 = *reinterpret_cast<const float2*>(&red[0][2 * tid]), r1 = *reinterpret_cast<const float2*>(&red[1][2 * tid]);
    const float2 r2 = *reinterpret_cast<const float2*>(&red[2][2 * tid]), r3 = *reinterpret_cast<const float2*>(&red[3][2 * tid]);
    *reinterpret_cast<uint32_t*>(orow + 2 * tid) =
        pack_bf16x2(((r0.x + r1.x) + (r2.x + r3.x)) * inv, ((r0.y + r1.y) + (r2.y + r3.y)) * inv);
  }
}

// f(D, bias, page size, their number among the eight), the first three as constants
template <typename F>
auto with_sizes(int head_dim, int page_size, bool bias, F f) {
  using std::integral_constant;
  auto page = [&](auto d, auto bi, int i) {
    return page_size == 64 ? f(d, bi, integral_constant<int, 64>{}, i)
                           : f(d, bi, integral_constant<int, 128>{}, i + 1);
  };
  auto gate = [&](auto d, int i) {
    return bias ? page(d, integral_constant<bool, true>{}, i) : page(d, integral_constant<bool, false>{}, i + 2);
  };
  return head_dim == 128 ? gate(integral_constant<int, 128>{}, 0) : gate(integral_constant<int, 64>{}, 4);
}

// Whether the one-launch kernel takes a call, by the table's width in keys and the
// number of (row, kv head) pairs.  Measured, GPU time of one and of two launches in
// us (rows of half to all of the width, gated heads of 64 / ungated of 128): one
// row, 16 / 8 heads, 256 keys 4.2, 8.5 / 4.5, 8.1; 1024 keys 7.5, 8.9 / 8.4, 9.1
// (a launch costs the host some 4 us besides); 2048 keys 13.5, 10.1 / 17.0, 9.2.
// 16 rows, 2048 keys 15.7, 21.6 / 19.5, 23.2; 4096 keys 26.3, 30.5 / 34.2, 32.7.
inline bool short_table(long keys, long pairs) { return keys <= 1024 || (keys <= 2048 && pairs >= 128); }

}  // namespace
}  // namespace sa

extern "C" size_t sa_paged_decode_fp8_workspace_size(int batch, int num_q_heads, int num_kv_heads,
                                                     int head_dim, int page_size, int max_pages) {
  if (batch < 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads || max_pages < 0 ||
      sa::short_table(static_cast<long>(max_pages) * page_size, static_cast<long>(batch) * num_kv_heads))
    return 0;
  return sa::decode_ws_layout(batch, num_q_heads, num_kv_heads, head_dim, sa::kDecodeMaxWaves, nullptr, nullptr);
}

extern "C" int sa_paged_decode_fp8_fwd(
    const void* q, const void* k_pages, const void* v_pages, const float* k_scale,
    const float* v_scale, const void* k_tail, const void* v_tail, const int32_t* page_table,
    const int32_t* seq_lens, const float* key_bias, int batch, int num_q_heads, int num_kv_heads,
    int head_dim, int page_size, int max_pages, int num_pages, float softmax_scale, void* o,
    void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "sa_paged_decode_fp8_fwd";
  if (const int rc = sa::decode_check(sa::kBF16, q, k_pages, v_pages, page_table, seq_lens,
                                      key_bias, batch, num_q_heads, num_kv_heads, head_dim,
                                      page_size, max_pages, num_pages, o, who))
    return rc;
  SA_CHECK_ARG(k_scale && v_scale && k_tail && v_tail, "%s: null pointer", who);
  SA_CHECK_ARG(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_pages) |
                 reinterpret_cast<uintptr_t>(v_pages) | reinterpret_cast<uintptr_t>(k_tail) |
                 reinterpret_cast<uintptr_t>(v_tail)) & 15) == 0,
               "%s: q, the pages and the tails must be 16-byte aligned", who);
  SA_CHECK_ARG(static_cast<long>(batch) * num_q_heads < (1L << 23), "%s: batch %d too large", who, batch);
  const size_t need = sa_paged_decode_fp8_workspace_size(batch, num_q_heads, num_kv_heads, head_dim,
                                                         page_size, max_pages);
  SA_CHECK_ARG(workspace_bytes >= need && (workspace || need == 0), "%s: workspace %zu B < %zu B", who,
               workspace_bytes, need);
  if (batch == 0) return 0;
  const float scale = softmax_scale > 0.f ? softmax_scale : 1.0f / sqrtf(static_cast<float>(head_dim));
  const float sl2 = scale * sa::kLog2e;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const sa::Fp8Cache kv{static_cast<const uint8_t*>(k_pages), static_cast<const uint8_t*>(v_pages),
                        k_scale, v_scale, static_cast<const sa::bf16*>(k_tail),
                        static_cast<const sa::bf16*>(v_tail), page_table, key_bias,
                        num_kv_heads, max_pages, num_pages};
  const auto* qp = static_cast<const sa::bf16*>(q);
  const bool bias = key_bias != nullptr;
  if (sa::short_table(static_cast<long>(max_pages) * page_size, static_cast<long>(batch) * num_kv_heads)) {
    sa::ProfScope prof_("paged_decode_fp8_short", s);
    sa::with_sizes(head_dim, page_size, bias, [&](auto d, auto bi, auto ps, int) {
      constexpr int D = decltype(d)::value;
      hipLaunchKernelGGL((sa::paged_decode_fp8_short_kernel<D, decltype(bi)::value, decltype(ps)::value>),
                         dim3(batch * num_kv_heads), dim3(64 * sa::kShortWaves<D>), 0, s, qp, kv, seq_lens,
                         static_cast<sa::bf16*>(o), num_q_heads, sl2);
      return 0;
    });
    SA_CHECK_LAUNCH("paged_decode_fp8_short");
    return 0;
  }
  sa::DecodeWs ws;
  sa::decode_ws_layout(batch, num_q_heads, num_kv_heads, head_dim, sa::kDecodeMaxWaves, workspace, &ws);
  const int W = sa::with_sizes(head_dim, page_size, bias, [](auto d, auto bi, auto ps, int i) {
    return sa::decode_waves(
        sa::paged_decode_fp8_kernel<decltype(d)::value, decltype(bi)::value, decltype(ps)::value>, i);
  });
  if (const int rc = sa::decode_plan_launch(seq_lens, batch, page_size, max_pages, ws, s)) return rc;
  {
    sa::ProfScope prof_("paged_decode_fp8", s);
    sa::with_sizes(head_dim, page_size, bias, [&](auto d, auto bi, auto ps, int) {
      hipLaunchKernelGGL(
          (sa::paged_decode_fp8_kernel<decltype(d)::value, decltype(bi)::value, decltype(ps)::value>),
          dim3(W), dim3(64), 0, s, qp, kv, seq_lens, ws.cum_row, ws.part_o, ws.part_ml, batch,
          num_q_heads, W, sl2);
      return 0;
    });
    SA_CHECK_LAUNCH("paged_decode_fp8");
  }
  sa::ProfScope prof_("paged_decode_fp8_merge", s);
  auto merge = [&](auto kern) {
    hipLaunchKernelGGL(kern, dim3(batch * num_q_heads), dim3(256), 0, s, ws.part_o, ws.part_ml,
                       ws.cum_row, static_cast<sa::bf16*>(o), batch, num_q_heads, num_kv_heads, W);
  };
  head_dim == 128 ? merge(sa::paged_decode_fp8_merge_kernel<128>) : merge(sa::paged_decode_fp8_merge_kernel<64>);
  SA_CHECK_LAUNCH("paged_decode_fp8_merge");
  return 0;
}
