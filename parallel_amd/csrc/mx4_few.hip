// Grouped products of mx4 operands where there are few tiles: a decoding
// token's experts, a handful of rows.  Each weight byte is used by up to 16
// rows, and what counts is how many loads are in flight at once.
//
// A block takes up to 16 rows of one group and four 16-row weight tiles (with
// swiglu gate and up tiles in turn, so that a lane holds both of an act value);
// its four waves split K: wave w multiplies the 256-deep steps w, w + 4, ...,
// and the waves' sums are added through LDS in wave order.  Operands go from
// memory to registers: lane l reads, of row l % 16, the two neighbouring
// 32-blocks 2 (l / 16) and + 1 of a 256-deep step, 32 bytes of a row's 128-byte
// line, and their two scales, one 16-bit load; each block is one of the step's
// two MFMAs' (products may take k in any order, so no operand is laid out anew).
//
// Against 64-row LDS tiles (mx4_tile.hip), of which few leave most CUs idle:
// gate and up of 8 rows of 8 groups, 2048 x 768, 6.7 against 11.2 us (6.7 MB of
// weights: launch and latency), of 32 rows of 28 groups 13.7 against 13.4; one
// group's 32 rows x 2048 x 2048 6.8 against 10.5, its 256 rows 21.6 against 11.5.
// With `ids` every row is a tile of its own in the order the rows come, and no
// sort or search for it: the experts of a few tokens share none to speak of.
#include "mx4.h"

namespace moe {
namespace {

constexpr int kFewWaves = 4, kFewTiles = 4;

template <int EPI>
__global__ __launch_bounds__(kFewWaves * kWave) void mx4_few_kernel(const Mx4Gemm p, int n_tiles) {
  constexpr bool GLU = mx4_glu(EPI);
  constexpr int NT = kFewTiles, kCols = (GLU ? NT / 2 : NT) * 16;  // output columns per block
  const int lane = threadIdx.x & (kWave - 1), i16 = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Mx4Tile t;
  if (p.ids) {
    t.r0 = blockIdx.x / n_tiles;
    t.n = blockIdx.x - t.r0 * n_tiles;
    t.rows = 1;
    const int64_t g = p.ids[t.r0];
    if (g < 0 || g >= p.G) return;  // the whole block
    t.g = static_cast<int>(g);
  } else if (!mx4_find_tile<16>(p, n_tiles, blockIdx.x, t)) {
    return;
  }
  const int n0 = t.n * kCols;
  const int64_t wide = GLU ? 2 * static_cast<int64_t>(p.N) : p.N;
  const uint32_t half_k = static_cast<uint32_t>(p.K) / 2, pitch = static_cast<uint32_t>(mx4_pitch(p.K));
  const auto rs_a = make_rsrc(p.a, static_cast<uint32_t>(p.a_rows) * half_k);
  const auto rs_as = make_rsrc(p.a_scales, static_cast<uint32_t>(p.a_rows) * pitch);
  const auto rs_w = make_rsrc(p.w + t.g * wide * half_k, static_cast<uint32_t>(wide) * half_k);
  const auto rs_ws = make_rsrc(p.w_scales + t.g * wide * pitch, static_cast<uint32_t>(wide) * pitch);

  // The lane's rows of the operands (row 0, and nothing read, where there is none).
  bool a_in = i16 < t.rows, w_in[NT];
  int src = t.r0 + (a_in ? i16 : 0);
  if (p.ids || p.row_index) src = mx4_source_row(p, p.ids ? src : p.row_index[src]);
  a_in = a_in && src >= 0 && src < p.a_rows;
  const uint32_t a_row = a_in ? src : 0;
  uint32_t w_row[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int n = n0 + 16 * (GLU ? j / 2 : j) + i16;
    w_in[j] = n < p.N;
    w_row[j] = w_in[j] ? (GLU && j % 2 ? p.N + n : n) : 0;
  }

  f32x4_t acc[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) acc[j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};

  struct Step {
    uint4 a[2], w[NT][2];
    uint32_t sa, sw[NT];
  };
  const int steps = (p.K + 255) / 256;
  auto load = [&](Step& s, int k) __attribute__((always_inline)) {
    const uint32_t at = 128u * k + 32u * q, sat = 8u * k + 2u * q;
    const int left = p.K / 32 - (8 * k + 2 * q);       // the lane's blocks inside K: 2, 1, or fewer
    const uint32_t keep = left > 1 ? 0xffffu : 0xffu;  // (scale padding may hold anything)
    auto get = [](__amdgpu_buffer_rsrc_t rs, uint32_t off, bool in) __attribute__((always_inline)) {
      const auto v = __builtin_amdgcn_raw_buffer_load_b128(rs, in ? off : kOOB, 0, 0);
      return make_uint4(v[0], v[1], v[2], v[3]);
    };
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const uint32_t off = w_row[j] * half_k + at;
      s.w[j][0] = get(rs_w, off, w_in[j] && left > 0);
      s.w[j][1] = get(rs_w, off + 16, w_in[j] && left > 1);
      s.sw[j] = __builtin_amdgcn_raw_buffer_load_b16(rs_ws, w_in[j] && left > 0 ? w_row[j] * pitch + sat : kOOB, 0, 0) & keep;
    }
    const uint32_t off = a_row * half_k + at;
    s.a[0] = get(rs_a, off, a_in && left > 0);
    s.a[1] = get(rs_a, off + 16, a_in && left > 1);
    s.sa = __builtin_amdgcn_raw_buffer_load_b16(rs_as, a_in && left > 0 ? a_row * pitch + sat : kOOB, 0, 0) & keep;
  };
  auto multiply = [&](const Step& s) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      acc[j] = mx4_mfma<0>(s.w[j][0], s.a[0], acc[j], s.sw[j], s.sa);
      acc[j] = mx4_mfma<1>(s.w[j][1], s.a[1], acc[j], s.sw[j], s.sa);
    }
  };
  Step s0, s1;
  int k = wave;
  if (k < steps) load(s0, k);
  for (; k < steps; k += 2 * kFewWaves) {  // past K: zeros
    load(s1, k + kFewWaves);
    multiply(s0);
    load(s0, k + 2 * kFewWaves);
    multiply(s1);
  }

  __shared__ f32x4_t sums[kFewWaves][NT][kWave];
#pragma unroll
  for (int j = 0; j < NT; ++j) sums[wave][j][lane] = acc[j];
  __syncthreads();
  if (wave) return;
  f32x4_t v[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    v[j] = sums[0][j][lane];
#pragma unroll
    for (int w = 1; w < kFewWaves; ++w) v[j] += sums[w][j][lane];
  }

  // Lane l holds row l % 16 and columns 16 j + 4 q .. + 3 of the block's in v[j].
  const bool in = i16 < t.rows;
  const int64_t row = t.r0 + i16;
  if constexpr (!GLU) {
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int n = n0 + 16 * j + 4 * q;
      if (!in || n >= p.N) continue;
      if constexpr (EPI == MX4_PLAIN_F32)
        *reinterpret_cast<float4*>(p.c32 + row * p.N + n) = make_float4(v[j][0], v[j][1], v[j][2], v[j][3]);
      else
        *reinterpret_cast<uint2*>(p.c + row * p.N + n) =
            make_uint2(pack_bf16x2(v[j][0], v[j][1]), pack_bf16x2(v[j][2], v[j][3]));
    }
  } else {
    float act[2][4];
#pragma unroll
    for (int e = 0; e < 8; ++e) act[e / 4][e % 4] = mx4_act(v[2 * (e / 4)][e % 4], v[2 * (e / 4) + 1][e % 4]);
    if constexpr (EPI == MX4_SWIGLU) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int n = n0 + 16 * h + 4 * q;
        if (in && n < p.N)
          *reinterpret_cast<uint2*>(p.c + row * p.N + n) =
              make_uint2(pack_bf16x2(act[h][0], act[h][1]), pack_bf16x2(act[h][2], act[h][3]));
      }
    } else {  // quantised from fp32: one rounding, to 4 bits; the block's 32 values are in the four lane quarters
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(act[e / 4][e % 4]) & 0x7fffffffu);
      top = quarters_max(top);
      const uint32_t s = mx4_scale(top);
      const float f = mx4_scale_f(s);
      if (in && n0 < p.N) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t c = 0;
          c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, act[h][0], act[h][1], f, 0);
          c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, act[h][2], act[h][3], f, 1);
          *reinterpret_cast<uint16_t*>(p.c_codes + row * (p.N / 2) + (n0 + 16 * h + 4 * q) / 2) =
              static_cast<uint16_t>(s == 255u ? 0u : c);
        }
        if (q == 0) p.c_scales[row * mx4_pitch(p.N) + n0 / 32] = static_cast<uint8_t>(s);
      }
    }
  }
}

}  // namespace

int mx4_few(const Mx4Gemm& p, int epi, hipStream_t stream, const char* name) {
  const int64_t n_tiles = mx4_few_columns(p.N, epi);
  const int64_t most = (p.ids ? p.rows : mx4_most_tiles(p.rows, p.G, 16)) * n_tiles;
  MOE_REQUIRE(most < (1ll << 30), MOE_ERR_UNSUPPORTED, "%s: too many tiles", name);
  const dim3 grid(static_cast<unsigned>(p.ids ? most : (most + 7) / 8 * 8)), block(kFewWaves * kWave);
  const int n = static_cast<int>(n_tiles);
  if (epi == MX4_PLAIN)
    hipLaunchKernelGGL((mx4_few_kernel<MX4_PLAIN>), grid, block, 0, stream, p, n);
  else if (epi == MX4_PLAIN_F32)
    hipLaunchKernelGGL((mx4_few_kernel<MX4_PLAIN_F32>), grid, block, 0, stream, p, n);
  else if (epi == MX4_SWIGLU)
    hipLaunchKernelGGL((mx4_few_kernel<MX4_SWIGLU>), grid, block, 0, stream, p, n);
  else
    hipLaunchKernelGGL((mx4_few_kernel<MX4_SWIGLU_MX4>), grid, block, 0, stream, p, n);
  return launch_status(name);
}

}  // namespace moe
