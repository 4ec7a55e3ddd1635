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
// Loads in flight, not bytes, bound it: 8 rows of 8 groups' gate and up, 2048 x
// 768 (6.7 MB of weights) take 6.9 us, of which a launch is 2 and each of the
// waves' two steps a memory latency; 64-row LDS tiles (mx4_tile.hip), of which
// few leave most CUs idle, take 10.6.

// The experts of a few tokens (Mx4Slots) need no sort: they share none to speak
// of, so every slot (token and choice) is a tile of its own, read by its id.
// Gate and up quantise the token's row on the way (a wave its own 256 values a
// step, through 144 bytes of LDS); down takes a token and 16 columns a block, a
// wave per slot, and adds the weighted slots in fp32.  One token's experts are
// 2 launches, 6.8 + 4.8 us at 2048 x 768, 8 of 128 experts.
#include <type_traits>

#include "mx4.h"

namespace moe {
namespace {

constexpr int kFewWaves = 4, kFewTiles = 4;

// X: uint8_t for mx4 activations, else the type of the rows (p.x) that slots quantise for themselves.
template <int EPI, class X>
__global__ __launch_bounds__(kFewWaves * kWave) void mx4_few_kernel(const Mx4Gemm p, int n_tiles) {
  constexpr bool SLOTS = !std::is_same<X, uint8_t>::value;
  constexpr bool GLU = mx4_glu(EPI);
  constexpr int NT = kFewTiles, kCols = (GLU ? NT / 2 : NT) * 16;  // output columns per block
  const int lane = threadIdx.x & (kWave - 1), i16 = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Mx4Tile t;
  if constexpr (SLOTS) {
    t.r0 = blockIdx.x / n_tiles;
    t.n = blockIdx.x - t.r0 * n_tiles;
    t.rows = 1;
    const int64_t g = p.ids[t.r0];
    if (g < 0 || g >= p.G) return;  // the whole block
    t.g = static_cast<int>(g);
  } else {
    if (!mx4_find_tile<16>(p, n_tiles, blockIdx.x, t)) return;
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
  if (SLOTS || p.row_index) src = mx4_source_row(p, SLOTS ? src : p.row_index[src]);
  a_in = a_in && src >= 0 && src < p.a_rows;
  const uint32_t a_row = a_in || SLOTS ? src : 0;  // (a slot's whole wave reads its row)
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
    uint4 a[2], w[NT][2];  // (a slot's row: four values a lane in a[0])
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
    if constexpr (SLOTS) {
      const int c = 256 * k + 4 * lane;
      const X* x = static_cast<const X*>(p.x) + static_cast<int64_t>(a_row) * p.K + c;
      s.a[0] = make_uint4(0, 0, 0, 0);
      if (c < p.K) {
        if constexpr (std::is_same<X, float>::value) {
          s.a[0] = *reinterpret_cast<const uint4*>(x);
        } else {
          const uint2 v = *reinterpret_cast<const uint2*>(x);
          s.a[0] = make_uint4(v.x << 16, v.x & 0xffff0000u, v.y << 16, v.y & 0xffff0000u);
        }
      }
      return;
    }
    const uint32_t off = a_row * half_k + at;
    s.a[0] = get(rs_a, off, a_in && left > 0);
    s.a[1] = get(rs_a, off + 16, a_in && left > 1);
    s.sa = __builtin_amdgcn_raw_buffer_load_b16(rs_as, a_in && left > 0 ? a_row * pitch + sat : kOOB, 0, 0) & keep;
  };
  __shared__ __attribute__((aligned(16))) char rows[SLOTS ? kFewWaves : 1][144];
  // A slot's four values a lane to the fragments of the whole wave (every row of the operand the same): blocks of 32
  // are eight neighbouring lanes, their codes 16 bits a lane.
  auto quantise = [&](Step& s) __attribute__((always_inline)) {
    const uint32_t v[4] = {s.a[0].x, s.a[0].y, s.a[0].z, s.a[0].w};
    uint32_t top = max(max(v[0] & 0x7fffffffu, v[1] & 0x7fffffffu), max(v[2] & 0x7fffffffu, v[3] & 0x7fffffffu));
    top = max(top, static_cast<uint32_t>(dpp_move_i<dpp::kQuadXor1>(0, static_cast<int>(top))));
    top = max(top, static_cast<uint32_t>(dpp_move_i<dpp::kQuadXor2>(0, static_cast<int>(top))));
    top = max(top, static_cast<uint32_t>(dpp_move_i<dpp::kHalfMirror>(0, static_cast<int>(top))));
    const uint32_t scale = mx4_scale(top);
    const float by = mx4_scale_f(scale);
    uint32_t c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, __uint_as_float(v[0]), __uint_as_float(v[1]), by, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, __uint_as_float(v[2]), __uint_as_float(v[3]), by, 1);
    char* mine = rows[wave];
    // (A wave's LDS operations keep their order; the fences keep the compiler's.)
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    reinterpret_cast<uint16_t*>(mine)[lane] = static_cast<uint16_t>(scale == 255u ? 0u : c);
    if (lane % 8 == 0) mine[128 + lane / 8] = static_cast<char>(scale);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    s.a[0] = *reinterpret_cast<const uint4*>(mine + 32 * q);
    s.a[1] = *reinterpret_cast<const uint4*>(mine + 32 * q + 16);
    s.sa = *reinterpret_cast<const uint16_t*>(mine + 128 + 2 * q);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  };
  auto multiply = [&](Step& s) __attribute__((always_inline)) {
    if constexpr (SLOTS) quantise(s);
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

// out[t, 16 columns] = sum over the token's slots of weight * (act row of the slot) W[id]^T, H rows of I values.
constexpr int kSlotWaves = 8;
template <class X>
__global__ __launch_bounds__(kSlotWaves * kWave) void mx4_slot_down_kernel(
    const uint8_t* __restrict__ act, const uint8_t* __restrict__ act_scales, const uint8_t* __restrict__ w,
    const uint8_t* __restrict__ w_scales, const int64_t* __restrict__ ids, const float* __restrict__ weights, int E,
    int H, int I, int k, int n_tiles, X* __restrict__ out) {
  const int lane = threadIdx.x & (kWave - 1), i16 = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t t = blockIdx.x / n_tiles;
  const int n = (blockIdx.x % n_tiles) * 16 + i16;
  const bool in = n < H;
  const uint32_t half = static_cast<uint32_t>(I) / 2, pitch = static_cast<uint32_t>(mx4_pitch(I));
  const int steps = (I + 255) / 256;
  f32x4_t sum = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int j = wave; j < k; j += kSlotWaves) {
    const int64_t slot = t * k + j, g = ids[slot];
    if (g < 0 || g >= E) continue;  // wave-uniform
    const auto rw = make_rsrc(w + g * H * half, static_cast<uint32_t>(H) * half);
    const auto rws = make_rsrc(w_scales + g * H * pitch, static_cast<uint32_t>(H) * pitch);
    const auto ra = make_rsrc(act + slot * half, half);
    const auto ras = make_rsrc(act_scales + slot * pitch, pitch);
    f32x4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s0 = 0; s0 < steps; s0 += 4) {  // four steps' loads at a time (past I: zeros)
      uint4 wf[4][2], af[4][2];
      uint32_t sw[4], sa[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int s = s0 + u;
        const uint32_t at = 128u * s + 32u * q, sat = 8u * s + 2u * q;
        const int left = I / 32 - (8 * s + 2 * q);
        const uint32_t keep = left > 1 ? 0xffffu : 0xffu;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const auto a = __builtin_amdgcn_raw_buffer_load_b128(rw, in && left > h ? n * half + at + 16 * h : kOOB, 0, 0);
          const auto b = __builtin_amdgcn_raw_buffer_load_b128(ra, left > h ? at + 16 * h : kOOB, 0, 0);
          wf[u][h] = make_uint4(a[0], a[1], a[2], a[3]);
          af[u][h] = make_uint4(b[0], b[1], b[2], b[3]);
        }
        sw[u] = __builtin_amdgcn_raw_buffer_load_b16(rws, in && left > 0 ? n * pitch + sat : kOOB, 0, 0) & keep;
        sa[u] = __builtin_amdgcn_raw_buffer_load_b16(ras, left > 0 ? sat : kOOB, 0, 0) & keep;
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        acc = mx4_mfma<0>(wf[u][0], af[u][0], acc, sw[u], sa[u]);
        acc = mx4_mfma<1>(wf[u][1], af[u][1], acc, sw[u], sa[u]);
      }
    }
    const float by = weights[slot];
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[e] += by * acc[e];
  }
  // Every row of the activation operand was the slot's: lane 16 q holds columns 4 q .. + 3.
  __shared__ float sums[kSlotWaves][16];
  if (i16 == 0)
#pragma unroll
    for (int e = 0; e < 4; ++e) sums[wave][4 * q + e] = sum[e];
  __syncthreads();
  if (threadIdx.x < 16 && n < H) {
    float o = 0.0f;
#pragma unroll
    for (int v = 0; v < kSlotWaves; ++v) o += sums[v][threadIdx.x];
    if constexpr (std::is_same<X, float>::value) out[t * H + n] = o;
    else out[t * H + n] = f32_to_bf16(o);
  }
}

}  // namespace

int mx4_few(const Mx4Gemm& p, int epi, hipStream_t stream, const char* name) {
  const int64_t n_tiles = mx4_few_columns(p.N, epi);
  const int64_t most = mx4_most_tiles(p.rows, p.G, 16) * n_tiles;
  MOE_REQUIRE(most < (1ll << 30), MOE_ERR_UNSUPPORTED, "%s: too many tiles", name);
  const dim3 grid(static_cast<unsigned>((most + 7) / 8 * 8)), block(kFewWaves * kWave);
  const int n = static_cast<int>(n_tiles);
  if (epi == MX4_PLAIN)
    hipLaunchKernelGGL((mx4_few_kernel<MX4_PLAIN, uint8_t>), grid, block, 0, stream, p, n);
  else if (epi == MX4_PLAIN_F32)
    hipLaunchKernelGGL((mx4_few_kernel<MX4_PLAIN_F32, uint8_t>), grid, block, 0, stream, p, n);
  else if (epi == MX4_SWIGLU)
    hipLaunchKernelGGL((mx4_few_kernel<MX4_SWIGLU, uint8_t>), grid, block, 0, stream, p, n);
  else
    hipLaunchKernelGGL((mx4_few_kernel<MX4_SWIGLU_MX4, uint8_t>), grid, block, 0, stream, p, n);
  return launch_status(name);
}

int mx4_slots(const Mx4Gemm& up, bool is_f32, const uint8_t* down, const uint8_t* down_scales, const float* weights,
              int64_t T, int64_t H, int64_t k, void* out, hipStream_t stream) {
  const int64_t up_tiles = mx4_few_columns(up.N, MX4_SWIGLU_MX4), down_tiles = (H + 15) / 16;
  MOE_REQUIRE(up.rows * up_tiles < (1ll << 30) && T * down_tiles < (1ll << 30), MOE_ERR_UNSUPPORTED,
              "mx4 experts: too many tiles");
  const dim3 up_grid(static_cast<unsigned>(up.rows * up_tiles)), down_grid(static_cast<unsigned>(T * down_tiles));
  auto launch = [&](auto x) {
    using X = decltype(x);
    hipLaunchKernelGGL((mx4_few_kernel<MX4_SWIGLU_MX4, X>), up_grid, dim3(kFewWaves * kWave), 0, stream, up,
                       static_cast<int>(up_tiles));
    const int rc = launch_status("moe_mx4_experts(gate and up)");
    if (rc) return rc;
    hipLaunchKernelGGL((mx4_slot_down_kernel<X>), down_grid, dim3(kSlotWaves * kWave), 0, stream, up.c_codes,
                       up.c_scales, down, down_scales, up.ids, weights, up.G, static_cast<int>(H),
                       static_cast<int>(up.N), static_cast<int>(k), static_cast<int>(down_tiles), static_cast<X*>(out));
    return launch_status("moe_mx4_experts(down)");
  };
  return is_f32 ? launch(float{}) : launch(bf16_t{});
}

}  // namespace moe
