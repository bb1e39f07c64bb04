// Paged decode attention: workspace layout, the launches and the device pieces
// shared by the decode entry points (attention.hip, attention_fp8.hip,
// decode_noalloc.hip).
#pragma once

#include "attn_tile.h"
#include "common.h"

namespace sa {

// most waves a stream-K decode launch uses on any device
constexpr int kDecodeMaxWaves = 8192;

// workspace: segment partials for b * Hkv + W segment ids (segment id =
// row * Hkv + kv head + wave, wave < W), then cum_row (b + 1 ints)
struct DecodeWs {
  float* part_o;
  float* part_ml;
  int32_t* cum_row;
};
inline size_t decode_ws_layout(int b, int Hq, int Hkv, int D, int W, void* base, DecodeWs* out) {
  const size_t segs = static_cast<size_t>(b) * Hkv + W;
  const size_t grp = static_cast<size_t>(Hq / Hkv);
  const size_t o_bytes = (segs * grp * D * sizeof(float) + 255) & ~size_t(255);
  const size_t ml_bytes = (segs * grp * 2 * sizeof(float) + 255) & ~size_t(255);
  const size_t cum_bytes = ((static_cast<size_t>(b) + 1) * sizeof(int32_t) + 255) & ~size_t(255);
  if (out) {
    char* p = static_cast<char*>(base);
    out->part_o = reinterpret_cast<float*>(p);
    out->part_ml = reinterpret_cast<float*>(p + o_bytes);
    out->cum_row = reinterpret_cast<int32_t*>(p + o_bytes + ml_bytes);
  }
  return o_bytes + ml_bytes + cum_bytes + 256;
}

// Online-softmax update for one block of keys.  s[kt][i]: log2-domain scores
// of keys 16kt + 4g + i for query column (lane & 15); masked entries are
// -inf.  Converts s to probabilities in place, rescales o, updates m and l.
template <int KT, int DT>
__device__ __forceinline__ void softmax_block(v4f (&s)[KT], v4f (&o)[DT], float& m, float& l) {
  float mx = kNegInf;
#pragma unroll
  for (int kt = 0; kt < KT; ++kt)
#pragma unroll
    for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[kt][i]);
  mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
  mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
  const float m_new = fmaxf(m, mx);
  const float alpha = (m == kNegInf) ? 0.0f : fast_exp2(m - m_new);
  float sum = 0.0f;
#pragma unroll
  for (int kt = 0; kt < KT; ++kt)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float p = (s[kt][i] == kNegInf) ? 0.0f : fast_exp2(s[kt][i] - m_new);
      s[kt][i] = p;
      sum += p;
    }
  sum += __shfl_xor(sum, 16, 64);
  sum += __shfl_xor(sum, 32, 64);
  l = l * alpha + sum;
  m = m_new;
#pragma unroll
  for (int t = 0; t < DT; ++t) o[t] *= alpha;
}

template <bool B>
struct BoolC {
  static constexpr bool value = B;
};

// tiles of row r: ceil(clamp(seq_lens[r], 0, max_pages * ps) / 64)
__device__ __forceinline__ int decode_row_len(const int32_t* seq_lens, int r, int max_pages, int ps) {
  return min(max(seq_lens[r], 0), max_pages * ps);
}

// first tile of wave w and the wave that holds tile g (W waves, T tiles)
__device__ __forceinline__ long decode_wave_begin(int w, long T, int W) {
  return static_cast<long>(w) * T / W;
}
__device__ __forceinline__ int decode_wave_of(long g, long T, int W) {
  return static_cast<int>(((g + 1) * W + T - 1) / T - 1);
}

// waves of one resident round: CUs x resident 64-thread blocks per CU
template <typename K>
inline int decode_waves(K kern, int variant) {
  static int cache[64][8] = {};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 1024;
  if (cache[dev][variant] == 0) {
    int cus = 0, per_cu = 0;
    if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess ||
        hipOccupancyMaxActiveBlocksPerMultiprocessor(&per_cu, kern, 64, 0) != hipSuccess ||
        cus <= 0 || per_cu <= 0)
      return 1024;
    cache[dev][variant] = min(cus * per_cu, kDecodeMaxWaves);
  }
  return cache[dev][variant];
}

int decode_plan_launch(const int32_t* seq_lens, int batch, int page_size, int max_pages,
                       const DecodeWs& ws, hipStream_t s);
int decode_check(int dtype, const void* q, const void* k_pages, const void* v_pages,
                 const int32_t* page_table, const int32_t* seq_lens, const float* key_bias,
                 int batch, int num_q_heads, int num_kv_heads, int head_dim, int page_size,
                 int max_pages, int num_pages, const void* o, const char* who);
int decode_wave_count(int head_dim, bool bias);
int decode_launch(const void* q, const void* k_pages, const void* v_pages,
                  const int32_t* page_table, const int32_t* seq_lens, const float* key_bias,
                  int batch, int num_q_heads, int num_kv_heads, int head_dim, int page_size,
                  int max_pages, int num_pages, float softmax_scale, void* o, const DecodeWs& ws,
                  int W, hipStream_t s);

}  // namespace sa
