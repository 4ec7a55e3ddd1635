// Grouped products of mx4 operands for groups of few rows: each weight byte is
// used by 16 MT rows at most, so HBM's stream of weights is the bound.
//
// A block takes up to 16 MT rows of one group and NT 16-row weight tiles (with
// swiglu gate and up tiles in turn, so that a lane holds both of an act value);
// its waves split K: wave w multiplies the 256-deep steps w, w + WK, ..., and
// the waves' sums are added through LDS in wave order.  Operands go from
// memory to registers with no LDS: lane l reads, of row l % 16, the two
// neighbouring 32-blocks 2 (l / 16) and + 1 of a 256-deep step, 32 bytes of a
// row's 128-byte line, and their two scales, one 16-bit load; each block is one
// of the step's two MFMAs' (products may take k in any order, so no operand is
// laid out anew).
#include "mx4.h"

namespace moe {
namespace {

template <int MT, int NT, int WK, int EPI>
__global__ __launch_bounds__(WK * kWave) void mx4_few_kernel(const Mx4Gemm p, int n_tiles) {
  constexpr bool GLU = EPI != MX4_PLAIN;
  constexpr int kCols = (GLU ? NT / 2 : NT) * 16;  // output columns per block
  const int lane = threadIdx.x & (kWave - 1), i16 = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Mx4Tile t;
  if (!mx4_find_tile<16 * MT>(p, n_tiles, blockIdx.x, t)) return;  // the whole block
  const int n0 = t.n * kCols;
  const int64_t wide = GLU ? 2 * static_cast<int64_t>(p.N) : p.N;
  const uint32_t half_k = static_cast<uint32_t>(p.K) / 2, pitch = static_cast<uint32_t>(mx4_pitch(p.K));
  const auto rs_a = make_rsrc(p.a, static_cast<uint32_t>(p.a_rows) * half_k);
  const auto rs_as = make_rsrc(p.a_scales, static_cast<uint32_t>(p.a_rows) * pitch);
  const auto rs_w = make_rsrc(p.w + t.g * wide * half_k, static_cast<uint32_t>(wide) * half_k);
  const auto rs_ws = make_rsrc(p.w_scales + t.g * wide * pitch, static_cast<uint32_t>(wide) * pitch);

  uint32_t a_row[MT], w_row[NT];  // the lane's rows; past the end: a row whose offset is out of range
  bool a_in[MT], w_in[NT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int m = 16 * i + i16;
    a_in[i] = m < t.rows;
    int r = t.r0 + (a_in[i] ? m : 0);
    if (p.row_index) r = mx4_source_row(p, p.row_index[r]);
    a_in[i] = a_in[i] && r >= 0 && r < p.a_rows;
    a_row[i] = a_in[i] ? r : 0;
  }
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int n = n0 + 16 * (GLU ? j / 2 : j) + i16;
    w_in[j] = n < p.N;
    w_row[j] = w_in[j] ? (GLU && j % 2 ? p.N + n : n) : 0;
  }

  f32x4_t acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};

  struct Step {
    uint4 a[MT][2], w[NT][2];
    uint32_t sa[MT], sw[NT];
  };
  const int steps = (p.K + 255) / 256;
  auto load = [&](Step& s, int k) __attribute__((always_inline)) {
    const uint32_t at = 128u * k + 32u * q, sat = 8u * k + 2u * q;
    const int left = p.K / 32 - (8 * k + 2 * q);  // the lane's blocks inside K: 0, 1 or 2
    const uint32_t keep = left > 1 ? 0xffffu : 0xffu;
    auto get = [&](__amdgpu_buffer_rsrc_t rs, uint32_t off, bool in) __attribute__((always_inline)) {
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
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const uint32_t off = a_row[i] * half_k + at;
      s.a[i][0] = get(rs_a, off, a_in[i] && left > 0);
      s.a[i][1] = get(rs_a, off + 16, a_in[i] && left > 1);
      s.sa[i] = __builtin_amdgcn_raw_buffer_load_b16(rs_as, a_in[i] && left > 0 ? a_row[i] * pitch + sat : kOOB, 0, 0) & keep;
    }
  };
  auto multiply = [&](const Step& s) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        acc[i][j] = mx4_mfma<0>(s.w[j][0], s.a[i][0], acc[i][j], s.sw[j], s.sa[i]);
        acc[i][j] = mx4_mfma<1>(s.w[j][1], s.a[i][1], acc[i][j], s.sw[j], s.sa[i]);
      }
  };
  Step s0, s1;
  int k = wave;
  if (k < steps) load(s0, k);
  for (; k < steps; k += 2 * WK) {  // past K: zeros
    load(s1, k + WK);
    multiply(s0);
    load(s0, k + 2 * WK);
    multiply(s1);
  }

  if constexpr (WK > 1) {
    __shared__ f32x4_t sums[WK][MT][NT][kWave];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) sums[wave][i][j][lane] = acc[i][j];
    __syncthreads();
    for (int i = wave; i < MT; i += WK) {
      f32x4_t v[NT];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        v[j] = sums[0][i][j][lane];
#pragma unroll
        for (int w = 1; w < WK; ++w) v[j] += sums[w][i][j][lane];
      }
      mx4_store_rows<EPI, NT>(p, v, t.r0 + 16 * i + i16, 16 * i + i16 < t.rows, n0, q);
    }
  } else {
#pragma unroll
    for (int i = 0; i < MT; ++i)
      mx4_store_rows<EPI, NT>(p, acc[i], t.r0 + 16 * i + i16, 16 * i + i16 < t.rows, n0, q);
  }
}

template <int MT, int NT, int WK>
int launch(const Mx4Gemm& p, int epi, hipStream_t stream, const char* name) {
  const int cols = (epi == MX4_PLAIN ? NT : NT / 2) * 16;
  const int n_tiles = (p.N + cols - 1) / cols;
  const int64_t most = mx4_most_tiles(p.rows, p.G, 16 * MT) * n_tiles;
  MOE_REQUIRE(most < (1ll << 30), MOE_ERR_UNSUPPORTED, "%s: too many tiles", name);
  const dim3 grid(static_cast<unsigned>((most + 7) / 8 * 8)), block(WK * kWave);
  if (epi == MX4_PLAIN)
    hipLaunchKernelGGL((mx4_few_kernel<MT, NT, WK, MX4_PLAIN>), grid, block, 0, stream, p, n_tiles);
  else if (epi == MX4_SWIGLU)
    hipLaunchKernelGGL((mx4_few_kernel<MT, NT, WK, MX4_SWIGLU>), grid, block, 0, stream, p, n_tiles);
  else
    hipLaunchKernelGGL((mx4_few_kernel<MT, NT, WK, MX4_SWIGLU_MX4>), grid, block, 0, stream, p, n_tiles);
  return launch_status(name);
}

}  // namespace

int mx4_few(const Mx4Gemm& p, int epi, hipStream_t stream, const char* name) {
  const int64_t mean = (static_cast<int64_t>(p.rows) + p.G - 1) / p.G;
  return mean <= 16 ? launch<1, 4, 4>(p, epi, stream, name) : launch<4, 4, 4>(p, epi, stream, name);
}

}  // namespace moe
