// Microscaled 4-bit operands (mx4) shared by the quantisation and product kernels.
//
// A row of K values (K a multiple of 32) is K/2 bytes of codes, the value of
// even index in the low half of a byte, and mx4_pitch(K) bytes of scales: byte
// j < K/32 is the biased exponent s of the 32 values 32 j .., each standing
// for code * 2^(s - 127) (s = 255: NaN); the rest pads the row to 8 bytes per
// 256 values and is never used.  A code is a sign bit and the index of 0,
// 0.5, 1, 1.5, 2, 3, 4, 6.
#pragma once

#include "common.h"
#include "gemm.h"

namespace moe {

inline __host__ __device__ int64_t mx4_pitch(int64_t K) { return (K + 255) / 256 * 8; }

// The scale byte of a block whose largest size has the fp32 bits `top`: the
// largest exponent that leaves it below 8 (values over 6 then round to 6),
// at least 2^-127; 255 for an infinity or NaN in the block.
__device__ __forceinline__ uint32_t mx4_scale(uint32_t top) {
  const int e = static_cast<int>(top >> 23);
  return e == 255 ? 255u : static_cast<uint32_t>(max(e - 2, 0));
}
// The float of a scale byte for the conversion instructions, which use its
// exponent alone (also 0, for 2^-127).
__device__ __forceinline__ float mx4_scale_f(uint32_t s) { return __uint_as_float(s << 23); }

// silu(g) u with the hardware's exponential and reciprocal (1 ulp each).
__device__ __forceinline__ float mx4_act(float g, float u) {
  const float e = __builtin_amdgcn_exp2f(-1.44269504f * g);  // past the float range: 0 or infinity
  return g * u * __builtin_amdgcn_rcpf(1.0f + e);
}

// The largest of the four lane quarters' values, in every quarter (register swaps of 16- and 32-lane rows).
__device__ __forceinline__ uint32_t quarters_max(uint32_t v) {
  const auto a = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  v = max(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  return max(b[0], b[1]);
}

// One product launch.
struct Mx4Gemm {
  const uint8_t *a, *a_scales;  // [a_rows, K]
  const int32_t* row_index;     // row r of the product reads row row_index[r] / row_div of A (null: row r)
  const int64_t* ids;           // slots, instead of offs and row_index: row r's group, reading row r / row_div
  const void* x;                // slots: A's rows as they are, bf16 or f32
  int row_div, a_rows;
  uint32_t div_magic, div_shift;  // x / row_div = x * div_magic >> div_shift for 0 <= x < 2^31
  const uint8_t *w, *w_scales;  // [G][N, K], or with swiglu [G][2 N, K]: gate rows, then up rows
  const int32_t* offs;
  int G, rows, N, K;
  bf16_t* c;                    // [rows, N] bf16, or
  float* c32;                   // (without swiglu) f32, or
  uint8_t *c_codes, *c_scales;  // (with swiglu) mx4
};
enum { MX4_PLAIN = 0, MX4_SWIGLU = 1, MX4_SWIGLU_MX4 = 2, MX4_PLAIN_F32 = 3 };
constexpr bool mx4_glu(int epi) { return epi == MX4_SWIGLU || epi == MX4_SWIGLU_MX4; }

// Rows of group g, clamped so that malformed offsets never address outside [0, rows).
__device__ __forceinline__ int mx4_group_rows(const Mx4Gemm& p, int g, int& lo) {
  int hi = 0;
  lo = 0;
  if (g < p.G) {
    hi = min(max(p.offs[g], 0), p.rows);
    lo = g ? min(max(p.offs[g - 1], 0), hi) : 0;
  }
  return hi - lo;
}

// The row of A behind entry i of row_index (negative entries stay out of range).
__device__ __forceinline__ int mx4_source_row(const Mx4Gemm& p, int i) {
  const uint64_t q = static_cast<uint64_t>(static_cast<uint32_t>(i)) * p.div_magic >> p.div_shift;
  return i < 0 ? -1 : static_cast<int>(q);
}

struct Mx4Tile {
  int g, r0, rows, n;  // group, first row, rows, column tile
};

// Block `block` of the grid's tile: tiles of up to BM rows in group-major
// order, then column tile, then rows (whose blocks read the same weights), an
// XCD's blocks taking neighbouring tiles.  A group's rows are split evenly
// over its tiles in steps of 16.  False where the grid has a block to spare.
template <int BM>
__device__ __forceinline__ bool mx4_find_tile(const Mx4Gemm& p, int n_tiles, int block, Mx4Tile& t) {
  constexpr int kXcd = 8;
  const int lane = threadIdx.x & (kWave - 1);
  int total = 0;
  for (int c0 = 0; c0 < p.G; c0 += kWave) {
    int lo;
    const int cnt = mx4_group_rows(p, c0 + lane, lo);
    total += __builtin_amdgcn_readlane(wave_inclusive_scan((cnt + BM - 1) / BM), kWave - 1);
  }
  total = __builtin_amdgcn_readfirstlane(total) * n_tiles;
  const int share = (total + kXcd - 1) / kXcd;
  const int idx = block / kXcd, tile = (block % kXcd) * share + idx;
  if (idx >= share || tile >= total) return false;
  for (int c0 = 0, base = 0; c0 < p.G; c0 += kWave) {
    int lo;
    const int cnt = mx4_group_rows(p, c0 + lane, lo);
    const int n = n_tiles * ((cnt + BM - 1) / BM);
    const int incl = wave_inclusive_scan(n);
    const int tot = __builtin_amdgcn_readlane(incl, kWave - 1);
    if (tile < base + tot) {
      const int w = __builtin_amdgcn_readfirstlane(__builtin_ctzll(__ballot(base + incl > tile)));
      const int local = tile - base - __builtin_amdgcn_readlane(incl - n, w);
      const int rows = __builtin_amdgcn_readlane(cnt, w), parts = (rows + BM - 1) / BM;
      const int per = ((rows + parts - 1) / parts + 15) & ~15;  // (parts - 1) * per < rows: parts - 1 whole BMs are
      t.n = local / parts;
      const int part = local - t.n * parts;
      t.g = c0 + w;
      t.r0 = __builtin_amdgcn_readlane(lo, w) + part * per;
      t.rows = min(per, rows - part * per);
      return t.rows > 0;
    }
    base += tot;
  }
  return false;
}

// Most tiles that groups of `rows` rows in all can need: one per nonempty
// group and one per BM further rows.
inline int64_t mx4_most_tiles(int64_t rows, int64_t G, int64_t BM) {
  const int64_t groups = G < rows ? G : rows;
  return groups + (rows - groups) / BM;
}

typedef int mx4_frag_t __attribute__((ext_vector_type(8)));
// D[n, m] += sum over 128 k of W[n, k] A[m, k]: lane l holds row l % 16 of
// either operand, values of one 32-block per lane quarter l / 16, and of the
// result column m = l % 16, rows n = 4 (l / 16) .. + 3.  STEP picks the byte of
// the lanes' scale words.
template <int STEP>
__device__ __forceinline__ f32x4_t mx4_mfma(const uint4& w, const uint4& a, const f32x4_t& c, uint32_t sw,
                                            uint32_t sa) {
  const mx4_frag_t wf = {static_cast<int>(w.x), static_cast<int>(w.y), static_cast<int>(w.z), static_cast<int>(w.w),
                         0, 0, 0, 0};
  const mx4_frag_t af = {static_cast<int>(a.x), static_cast<int>(a.y), static_cast<int>(a.z), static_cast<int>(a.w),
                         0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf, af, c, 4, 4, STEP, sw, STEP, sa);
}

// Blocks of the few-row kernel side by side over N output columns.
inline int64_t mx4_few_columns(int64_t N, int epi) { return mx4_glu(epi) ? (N + 31) / 32 : (N + 63) / 64; }
inline int64_t mx4_tile_columns(int64_t N, int epi) { return mx4_glu(epi) ? (N + 127) / 128 : (N + 255) / 256; }

// Products of few tiles in all (mx4_few.hip).
int mx4_few(const Mx4Gemm& p, int epi, hipStream_t stream, const char* name);
// The experts of a few slots: gate and up (p: rows = T k slots, ids, x, row_div = k, the act rows' mx4 output) and
// down with the weighted sum (mx4_few.hip).
int mx4_slots(const Mx4Gemm& up, bool is_f32, const uint8_t* down, const uint8_t* down_scales, const float* weights,
              int64_t T, int64_t H, int64_t k, void* out, hipStream_t stream);
// Products of many rows per group in tiles of up to bm (64, 128 or 256) rows (mx4_tile.hip).
int mx4_tile(const Mx4Gemm& p, int epi, int bm, hipStream_t stream, const char* name);

}  // namespace moe
