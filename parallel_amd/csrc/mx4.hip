// Quantisation to microscaled 4-bit values and back, and the entry points of
// the grouped products (format: mx4.h).
//
// Either direction is one pass bound by HBM: a thread takes 8 values (16 bytes
// of bf16), four neighbouring lanes a block of 32, whose largest size two DPP
// moves find; the conversion instruction scales by a power of two and rounds
// to nearest even, saturating at 6.
#include <cmath>
#include <type_traits>
#include <utility>

#include "mx4.h"

namespace moe {

constexpr int kMx4Threads = 256;

__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  v = max(v, static_cast<uint32_t>(dpp_move_i<dpp::kQuadXor1>(0, static_cast<int>(v))));
  return max(v, static_cast<uint32_t>(dpp_move_i<dpp::kQuadXor2>(0, static_cast<int>(v))));
}

// Thread i takes values 8 i .. 8 i + 7 of the rows laid end to end; `pad` is
// the bytes behind each row's scales (0: the scales lie end to end too).
template <class E>
__global__ __launch_bounds__(kMx4Threads) void mx4_quantize_kernel(const E* __restrict__ x, int64_t n8, int64_t K,
                                                                   uint32_t* __restrict__ codes,
                                                                   uint8_t* __restrict__ scales, int pad) {
  const int64_t step = static_cast<int64_t>(gridDim.x) * kMx4Threads;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kMx4Threads + threadIdx.x; i < n8; i += step) {
    uint32_t c = 0, s;
    if constexpr (std::is_same<E, float>::value) {
      const float4 lo = reinterpret_cast<const float4*>(x)[2 * i], hi = reinterpret_cast<const float4*>(x)[2 * i + 1];
      const float f[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(f[e]) & 0x7fffffffu);
      s = mx4_scale(quad_max(top));
      const float by = mx4_scale_f(s);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[0], f[1], by, 0);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[2], f[3], by, 1);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[4], f[5], by, 2);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[6], f[7], by, 3);
    } else {
      const uint4 v = reinterpret_cast<const uint4*>(x)[i];
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) top = max(top, max((w[e] & 0x7fffu) << 16, w[e] & 0x7fff0000u));
      s = mx4_scale(quad_max(top));
      const float by = mx4_scale_f(s);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_t, w[0]), by, 0);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_t, w[1]), by, 1);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_t, w[2]), by, 2);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_t, w[3]), by, 3);
    }
    codes[i] = s == 255u ? 0u : c;
    if ((i & 3) == 0) {
      int64_t at = i >> 2;
      if (pad) {
        const int64_t per = K / 32, row = at / per;
        at += row * pad;
        if (at + 1 == row * (per + pad) + per)  // the row's last block
          for (int b = 1; b <= pad; ++b) scales[at + b] = 0;
      }
      scales[at] = static_cast<uint8_t>(s);
    }
  }
}

// A thread takes U chunks of 8 values together: one is too little a wave's work (256 bytes read, written four- or
// eightfold).  128 x 1536 x 2048 bf16 270, 211, 195, 192 us with 1, 2, 4, 8 (805 MB written, 5.2 TB/s in all); half of
// it fp32 217, 211, 229, 240.  Up to 2^22 chunks one: 48 x 2048 in 2.8 us, 3.8 with 4; 16384 x 2048 20.3, 20.7.
template <class E, int U>
__global__ __launch_bounds__(kMx4Threads) void mx4_dequantize_kernel(const uint32_t* __restrict__ codes,
                                                                     const uint8_t* __restrict__ scales, int64_t n8,
                                                                     int64_t K, E* __restrict__ out, int pad) {
  const int64_t step = static_cast<int64_t>(gridDim.x) * (U * kMx4Threads);
  for (int64_t i0 = static_cast<int64_t>(blockIdx.x) * (U * kMx4Threads) + threadIdx.x; i0 < n8; i0 += step) {
    uint32_t c[U];
    int s[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t i = min(i0 + u * kMx4Threads, n8 - 1);
      int64_t at = i >> 2;
      if (pad) at += at / (K / 32) * pad;
      c[u] = codes[i];
      s[u] = scales[at];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t i = i0 + u * kMx4Threads;
      if (i >= n8) break;
      float f[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t n = (c[u] >> (4 * e)) & 15u, m = n & 7u;  // m: exponent field and mantissa bit; 0.5 is subnormal
        const float size =
            m < 2 ? 0.5f * static_cast<float>(m) : __uint_as_float((126u + (m >> 1)) << 23 | (m & 1u) << 22);
        const float v = s[u] == 255 ? __uint_as_float(0x7fc00000u) : ldexpf(size, s[u] - 127);
        f[e] = (n & 8u) ? -v : v;
      }
      if constexpr (std::is_same<E, float>::value) {
        reinterpret_cast<float4*>(out)[2 * i] = make_float4(f[0], f[1], f[2], f[3]);
        reinterpret_cast<float4*>(out)[2 * i + 1] = make_float4(f[4], f[5], f[6], f[7]);
      } else {
        reinterpret_cast<uint4*>(out)[i] = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]),
                                                      pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
      }
    }
  }
}

// out[t, :] = sum over the token's slots, in slot order, of weight * row (fp32 rows), 8 columns a thread.
template <class E>
__global__ __launch_bounds__(kMx4Threads) void mx4_combine_kernel(const float* __restrict__ y,
                                                                  const int32_t* __restrict__ pos_of_slot,
                                                                  const int32_t* __restrict__ offsets, int experts,
                                                                  const float* __restrict__ weights, int H, int k,
                                                                  int per_row, E* __restrict__ out) {
  const int64_t t = blockIdx.x / per_row;
  const int c = (blockIdx.x % per_row) * kMx4Threads + threadIdx.x;
  if (c >= H / 8) return;
  const int valid = offsets[experts - 1];
  float o[8] = {};
#pragma unroll 4
  for (int j = 0; j < k; ++j) {
    const int64_t pos = pos_of_slot[t * k + j];
    if (pos >= valid) continue;  // the slot's expert is elsewhere
    const float w = weights[t * k + j];
    const float4* row = reinterpret_cast<const float4*>(y + pos * H + 8 * c);
    const float4 a = row[0], b = row[1];
    o[0] += w * a.x; o[1] += w * a.y; o[2] += w * a.z; o[3] += w * a.w;
    o[4] += w * b.x; o[5] += w * b.y; o[6] += w * b.z; o[7] += w * b.w;
  }
  if constexpr (std::is_same<E, float>::value) {
    float4* to = reinterpret_cast<float4*>(out + t * H + 8 * c);
    to[0] = make_float4(o[0], o[1], o[2], o[3]);
    to[1] = make_float4(o[4], o[5], o[6], o[7]);
  } else {
    *reinterpret_cast<uint4*>(out + t * H + 8 * c) = make_uint4(pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]),
                                                                pack_bf16x2(o[4], o[5]), pack_bf16x2(o[6], o[7]));
  }
}

}  // namespace moe

using namespace moe;

namespace {
bool aligned8(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 7u) == 0; }

int check_rows(const char* what, const void* x, const void* codes, const void* scales, int64_t rows, int64_t K) {
  MOE_REQUIRE(rows >= 0 && K > 0, MOE_ERR_INVALID, "%s: bad sizes %lld x %lld", what, (long long)rows, (long long)K);
  MOE_REQUIRE(K % 32 == 0, MOE_ERR_UNSUPPORTED, "%s: rows of %lld values are not whole blocks of 32", what,
              (long long)K);
  MOE_REQUIRE(rows <= (1ll << 40) / K, MOE_ERR_UNSUPPORTED, "%s: too many values", what);
  if (rows == 0) return MOE_OK;
  MOE_REQUIRE(x && codes && scales, MOE_ERR_INVALID, "%s: null pointer", what);
  MOE_REQUIRE(aligned16(x) && aligned16(codes) && aligned8(scales), MOE_ERR_INVALID, "%s: misaligned operand", what);
  return MOE_OK;
}

// Blocks of a pass over n8 chunks of 8 values, a thread taking `chunks` of them, and no more short of 2^30 threads: the
// hardware hands out blocks as others end, and reads stay in order (bf16 weights of 805 MB to codes 176 us, 5.8 TB/s;
// 210 with 16384 blocks that stride over them).
unsigned pass_blocks(int64_t n8, int chunks) {
  const int64_t each = static_cast<int64_t>(chunks) * kMx4Threads, blocks = (n8 + each - 1) / each;
  return static_cast<unsigned>(blocks < (1 << 22) ? blocks : 1 << 22);
}

// Granlund and Montgomery's multiplier: with l = ceil(log2 d), m = floor(2^(31+l) / d) + 1 divides 31-bit numbers.
void set_divisor(Mx4Gemm& p, int64_t d) {
  uint32_t l = 0;
  while ((1ll << l) < d) ++l;
  p.row_div = static_cast<int>(d);
  p.div_magic = static_cast<uint32_t>((1ull << (31 + l)) / static_cast<uint64_t>(d) + 1);
  p.div_shift = 31 + l;
}

// Which kernel, from the sizes alone (the groups' own counts are on the device).
//
// The few-row kernel where it needs at most two blocks (16 rows by 64 weight rows each) per CU: 2048 x 2048, one
// group, 64, 256 and 512 rows (128, 512, 1024 blocks) 7.0, 10.5 and 18.7 us against 11.3, 11.3 and 11.6 with 64-row
// LDS tiles; gate and up of 8 to 128 rows of 8 to 28 groups 5 to 10 against 7 to 11.
//
// Else the tile height whose passes over the CUs cost least, the estimate being a tile for each group at the least
// and a tile's cost 1, 1.6 and 2.5 for 64, 128 and 256 rows (2048 x 2048, one group, 1024 rows, one pass each: 12.3,
// 15.9, 22.8 us; 16384 rows, 8, 4 and 2 passes: 71, 56, 53; gate and up of 128 groups, 2048 x 768, at 32, 64, 96, 256
// and 1024 rows each: 37, 47, 54, 121, 413 with 64, 40, 41, 45, 103, 317 with 128, 48, 51, 54, 98, 286 with 256).
// Up to K 1024, where the epilogue is more of a tile, a 128-row tile costs two of 64 rows and is not taken (down, K 768,
// 64 even groups of 128 and 256 rows 24 and 37 us with 64, 26 and 37 with 128; Zipf ones 25 and 40, 27 and 38).
// Over 315 products, even and Zipf groups of 1 to 1024 rows, the choice is 2% behind the best one in the mean and 31%
// at the worst (64 Zipf groups of 256 rows in the mean: their tiles are more than estimated).
int mx4_product(const Mx4Gemm& p, int epi, hipStream_t stream, const char* what) {
  const int64_t cus = device_cus(current_device()), groups = p.G < p.rows ? p.G : p.rows;
  if ((groups + (p.rows - groups) / 16) * mx4_few_columns(p.N, epi) <= 2 * cus) return mx4_few(p, epi, stream, what);
  const int64_t columns = mx4_tile_columns(p.N, epi);
  int best = 0;
  int64_t least = 0;
  for (const auto& [height, cost] : {std::pair{64, 10}, std::pair{128, p.K > 1024 ? 16 : 20}, std::pair{256, 25}}) {
    const int64_t down = (static_cast<int64_t>(p.rows) + height - 1) / height;
    const int64_t all = ((down > groups ? down : groups) * columns + cus - 1) / cus * cost;
    if (best == 0 || all < least) best = height, least = all;
  }
  return mx4_tile(p, epi, best, stream, what);
}

int run_product(const char* what, const void* a, const void* a_scales, int64_t a_rows, const int32_t* row_index,
                int64_t row_div, const void* w, const void* w_scales, const int32_t* offs, int64_t G, int64_t M,
                int64_t N, int64_t K, void* c, void* c_codes, void* c_scales, int epi, void* stream) {
  const int64_t wide = mx4_glu(epi) ? 2 * N : N;
  MOE_REQUIRE(G > 0 && M >= 0 && a_rows >= 0 && N > 0 && K > 0 && row_div > 0, MOE_ERR_INVALID, "%s: bad sizes", what);
  MOE_REQUIRE(K % 32 == 0 && N % 8 == 0, MOE_ERR_UNSUPPORTED, "%s: K=%lld must be a multiple of 32, N=%lld of 8", what,
              (long long)K, (long long)N);
  MOE_REQUIRE(epi != MX4_SWIGLU_MX4 || N % 32 == 0, MOE_ERR_UNSUPPORTED,
              "%s: 4-bit output of %lld columns is not whole blocks of 32", what, (long long)N);
  MOE_REQUIRE(M < (1ll << 31) && a_rows < (1ll << 31) && G < (1ll << 24) && row_div < (1ll << 31) && N <= (1ll << 20) &&
                  K < (1ll << 28),
              MOE_ERR_UNSUPPORTED, "%s: sizes past 32 bits", what);
  MOE_REQUIRE(a_rows * (K / 2) < (1ll << 31) && wide * (K / 2) < (1ll << 31), MOE_ERR_UNSUPPORTED,
              "%s: the activations and each group's weights must stay below 2 GiB", what);
  MOE_REQUIRE(row_index || a_rows >= M, MOE_ERR_INVALID, "%s: %lld activation rows for %lld", what, (long long)a_rows,
              (long long)M);
  MOE_REQUIRE(w && w_scales && offs && aligned16(w) && aligned8(w_scales), MOE_ERR_INVALID,
              "%s: bad weight or offsets pointer", what);
  if (M == 0) return MOE_OK;
  MOE_REQUIRE(a && a_scales && aligned16(a) && aligned8(a_scales), MOE_ERR_INVALID, "%s: bad activation pointer", what);
  if (epi == MX4_SWIGLU_MX4) {
    MOE_REQUIRE(c_codes && c_scales && aligned16(c_codes) && aligned8(c_scales), MOE_ERR_INVALID,
                "%s: bad output pointer", what);
  } else {
    MOE_REQUIRE(c && aligned16(c), MOE_ERR_INVALID, "%s: bad output pointer", what);
  }
  Mx4Gemm p{};
  p.a = static_cast<const uint8_t*>(a);
  p.a_scales = static_cast<const uint8_t*>(a_scales);
  p.row_index = row_index;
  set_divisor(p, row_div);
  p.a_rows = static_cast<int>(a_rows);
  p.w = static_cast<const uint8_t*>(w);
  p.w_scales = static_cast<const uint8_t*>(w_scales);
  p.offs = offs;
  p.G = static_cast<int>(G);
  p.rows = static_cast<int>(M);
  p.N = static_cast<int>(N);
  p.K = static_cast<int>(K);
  if (epi == MX4_PLAIN_F32) p.c32 = static_cast<float*>(c);
  else p.c = static_cast<bf16_t*>(c);
  p.c_codes = static_cast<uint8_t*>(c_codes);
  p.c_scales = static_cast<uint8_t*>(c_scales);
  return mx4_product(p, epi, as_stream(stream), what);
}
}  // namespace

extern "C" int moe_mx4_quantize(const void* x, int is_f32, int64_t rows, int64_t K, void* codes, void* scales,
                                void* stream) {
  const int rc = check_rows("mx4 quantize", x, codes, scales, rows, K);
  if (rc || rows == 0) return rc;
  const int64_t n8 = rows * K / 8;
  const int pad = static_cast<int>(mx4_pitch(K) - K / 32);
  if (is_f32)
    hipLaunchKernelGGL(mx4_quantize_kernel<float>, dim3(pass_blocks(n8, 1)), dim3(kMx4Threads), 0, as_stream(stream),
                       static_cast<const float*>(x), n8, K, static_cast<uint32_t*>(codes),
                       static_cast<uint8_t*>(scales), pad);
  else
    hipLaunchKernelGGL(mx4_quantize_kernel<bf16_t>, dim3(pass_blocks(n8, 1)), dim3(kMx4Threads), 0, as_stream(stream),
                       static_cast<const bf16_t*>(x), n8, K, static_cast<uint32_t*>(codes),
                       static_cast<uint8_t*>(scales), pad);
  return launch_status("moe_mx4_quantize");
}

extern "C" int moe_mx4_dequantize(const void* codes, const void* scales, int64_t rows, int64_t K, int is_f32,
                                  void* out, void* stream) {
  const int rc = check_rows("mx4 dequantize", out, codes, scales, rows, K);
  if (rc || rows == 0) return rc;
  const int64_t n8 = rows * K / 8;
  const int pad = static_cast<int>(mx4_pitch(K) - K / 32);
  auto launch = [&](auto e, auto chunks) {
    using E = decltype(e);
    constexpr int U = decltype(chunks)::value;
    hipLaunchKernelGGL((mx4_dequantize_kernel<E, U>), dim3(pass_blocks(n8, U)), dim3(kMx4Threads), 0, as_stream(stream),
                       static_cast<const uint32_t*>(codes), static_cast<const uint8_t*>(scales), n8, K,
                       static_cast<E*>(out), pad);
  };
  auto typed = [&](auto e, auto chunks) {
    if (n8 <= 1ll << 22) launch(e, std::integral_constant<int, 1>{});
    else launch(e, chunks);
  };
  if (is_f32) typed(float{}, std::integral_constant<int, 2>{});
  else typed(bf16_t{}, std::integral_constant<int, 4>{});
  return launch_status("moe_mx4_dequantize");
}

extern "C" int moe_mx4_grouped_gemm(const void* a_codes, const void* a_scales, int64_t a_rows,
                                    const int32_t* row_index, int64_t row_divisor, const void* w_codes,
                                    const void* w_scales, const int32_t* offs, int64_t G, int64_t M, int64_t N,
                                    int64_t K, void* c, void* stream) {
  return run_product("moe_mx4_grouped_gemm", a_codes, a_scales, a_rows, row_index, row_divisor, w_codes, w_scales, offs,
                     G, M, N, K, c, nullptr, nullptr, MX4_PLAIN, stream);
}

extern "C" int moe_mx4_grouped_swiglu(const void* a_codes, const void* a_scales, int64_t a_rows,
                                      const int32_t* row_index, int64_t row_divisor, const void* w_codes,
                                      const void* w_scales, const int32_t* offs, int64_t G, int64_t M, int64_t I,
                                      int64_t K, void* act, void* act_codes, void* act_scales, void* stream) {
  return run_product("moe_mx4_grouped_swiglu", a_codes, a_scales, a_rows, row_index, row_divisor, w_codes, w_scales,
                     offs, G, M, I, K, act, act_codes, act_scales, act_codes ? MX4_SWIGLU_MX4 : MX4_SWIGLU, stream);
}

namespace {
// Whether the slots go one by one, in their own order (mx4_few.hip): up to 128 that read at most 48 MB of weights again
// which an expert's rows taken together would read once (the tokens' experts by even routing).  128 experts of 2048 x
// 768, 8 a token: 8, 64, 96 and 128 slots (0, 33, 70, 116 MB) 12, 42, 58, 72 us against 23, 53, 60, 62 sorted; 8 of 1024
// x 512, 2 a token: 32, 48, 64 slots (20, 33, 47 MB) 13, 17, 20 against 18 each; 16 of 4096 x 1536, 2 a token: 8, 16, 32
// slots (15, 57, 165 MB) 26, 44, 73 against 33, 42, 47.
bool slots_apart(int64_t T, int64_t H, int64_t k, int64_t E, int64_t I) {
  const double slots = static_cast<double>(T) * k, share = k < E ? static_cast<double>(k) / E : 1.0;
  const double hit = E * (1.0 - std::pow(1.0 - share, static_cast<double>(T)));
  return slots <= 128 && (slots - hit) * (3.0 * I * H * 17 / 32) <= 48e6;
}
constexpr int kMaxExperts = 1024;  // as many as the sort takes, with or without it

// The experts' workspace, each part 256-byte aligned.
struct ExpertsSpace {
  size_t perm, pos, counts, offsets, sort, x, x_scales, act, act_scales, y, bytes;
  size_t sort_bytes;
  bool f32_rows, sorted;
};
// The down product's rows are held in fp32 for fp32 modules, and while they stay small enough (16 MiB) that their
// bytes do not count; a bf16 row rounds once more, by half a step of the output's type.
ExpertsSpace experts_space(bool is_f32, int64_t T, int64_t H, int64_t k, int64_t E, int64_t I) {
  const int64_t S = T * k;
  ExpertsSpace s{};
  size_t at = 0;
  auto take = [&](int64_t bytes) {
    const size_t here = at;
    at += (static_cast<size_t>(bytes) + 255) / 256 * 256;
    return here;
  };
  s.f32_rows = is_f32 || S * H <= (1ll << 22);
  s.sorted = !slots_apart(T, H, k, E, I);
  s.act = take(S * (I / 2));
  s.act_scales = take(S * mx4_pitch(I));
  if (s.sorted) {
    s.perm = take(4 * S);
    s.pos = take(4 * S);
    s.counts = take(4 * E);
    s.offsets = take(4 * E);
    s.sort_bytes = moe_permute_workspace_bytes(S, E);
    s.sort = take(static_cast<int64_t>(s.sort_bytes));
    s.x = take(T * (H / 2));
    s.x_scales = take(T * mx4_pitch(H));
    s.y = take(S * H * (s.f32_rows ? 4 : 2));
  }
  s.bytes = at;
  return s;
}
bool experts_sizes(int64_t T, int64_t H, int64_t k, int64_t E, int64_t I) {
  return T >= 0 && T < (1ll << 31) && k >= 1 && k <= kMaxSlots && T * k < (1ll << 31) && E >= 1 && H > 0 &&
         H <= (1ll << 20) && I > 0 && I <= (1ll << 20);
}
}  // namespace

extern "C" size_t moe_mx4_experts_workspace_bytes(int is_f32, int64_t T, int64_t H, int64_t k, int64_t E, int64_t I) {
  return experts_sizes(T, H, k, E, I) ? experts_space(is_f32, T, H, k, E, I).bytes : 0;
}

extern "C" int moe_mx4_experts(const void* hidden, int is_f32, const int64_t* ids, const float* weights, int64_t T,
                               int64_t H, int64_t k, int64_t E, int64_t I, const void* gate_up_codes,
                               const void* gate_up_scales, const void* down_codes, const void* down_scales, void* out,
                               void* workspace, size_t workspace_bytes, void* stream) {
  MOE_REQUIRE(experts_sizes(T, H, k, E, I), MOE_ERR_INVALID, "mx4 experts: bad sizes (k at most %d)", kMaxSlots);
  MOE_REQUIRE(H % 32 == 0 && I % 32 == 0, MOE_ERR_UNSUPPORTED, "mx4 experts: H=%lld and I=%lld must be multiples of 32",
              (long long)H, (long long)I);
  MOE_REQUIRE(E <= kMaxExperts, MOE_ERR_UNSUPPORTED, "mx4 experts: more than %d experts", kMaxExperts);
  const int64_t S = T * k;
  if (T == 0) return MOE_OK;
  MOE_REQUIRE(hidden && ids && weights && out && aligned16(hidden) && aligned16(out), MOE_ERR_INVALID,
              "mx4 experts: bad pointer");
  MOE_REQUIRE(gate_up_codes && gate_up_scales && down_codes && down_scales && aligned16(gate_up_codes) &&
                  aligned8(gate_up_scales) && aligned16(down_codes) && aligned8(down_scales),
              MOE_ERR_INVALID, "mx4 experts: bad weight pointer");
  MOE_REQUIRE(T * (H / 2) < (1ll << 31) && S * (I / 2) < (1ll << 31) && I * H < (1ll << 31), MOE_ERR_UNSUPPORTED,
              "mx4 experts: the 4-bit rows and each expert's weights must stay below 2 GiB");
  const ExpertsSpace s = experts_space(is_f32, T, H, k, E, I);
  MOE_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= s.bytes, MOE_ERR_WORKSPACE,
              "mx4 experts: workspace %zu < %zu bytes", workspace_bytes, s.bytes);
  char* ws = static_cast<char*>(workspace);
  int32_t* perm = reinterpret_cast<int32_t*>(ws + s.perm);
  int32_t* pos = reinterpret_cast<int32_t*>(ws + s.pos);
  int32_t* offsets = reinterpret_cast<int32_t*>(ws + s.offsets);
  if (!s.sorted) {
    Mx4Gemm up{};
    up.x = hidden;
    up.ids = ids;
    set_divisor(up, k);
    up.a_rows = static_cast<int>(T);
    up.w = static_cast<const uint8_t*>(gate_up_codes);
    up.w_scales = static_cast<const uint8_t*>(gate_up_scales);
    up.G = static_cast<int>(E);
    up.rows = static_cast<int>(S);
    up.N = static_cast<int>(I);
    up.K = static_cast<int>(H);
    up.c_codes = reinterpret_cast<uint8_t*>(ws + s.act);
    up.c_scales = reinterpret_cast<uint8_t*>(ws + s.act_scales);
    return mx4_slots(up, is_f32, static_cast<const uint8_t*>(down_codes), static_cast<const uint8_t*>(down_scales),
                     weights, T, H, k, out, as_stream(stream));
  }
  int rc = permute_fwd_run(nullptr, T, 0, ids, k, 1, E, nullptr, perm, pos, reinterpret_cast<int32_t*>(ws + s.counts),
                           offsets, ws + s.sort, s.sort_bytes, stream);
  if (rc) return rc;
  rc = moe_mx4_quantize(hidden, is_f32, T, H, ws + s.x, ws + s.x_scales, stream);
  if (rc) return rc;
  rc = run_product("mx4 experts, gate and up", ws + s.x, ws + s.x_scales, T, perm, k, gate_up_codes, gate_up_scales,
                   offsets, E, S, I, H, nullptr, ws + s.act, ws + s.act_scales, MX4_SWIGLU_MX4, stream);
  if (rc) return rc;
  rc = run_product("mx4 experts, down", ws + s.act, ws + s.act_scales, S, nullptr, 1, down_codes, down_scales, offsets,
                   E, S, H, I, ws + s.y, nullptr, nullptr, s.f32_rows ? MX4_PLAIN_F32 : MX4_PLAIN, stream);
  if (rc) return rc;
  if (!s.f32_rows) return moe_combine_fwd(ws + s.y, pos, offsets, E, weights, T, H, k, out, stream);
  const int64_t per_row = (H / 8 + kMx4Threads - 1) / kMx4Threads;
  MOE_REQUIRE(T * per_row < (1ll << 31), MOE_ERR_UNSUPPORTED, "mx4 experts: too many rows");
  const dim3 grid(static_cast<unsigned>(T * per_row)), block(kMx4Threads);
  const float* y = reinterpret_cast<const float*>(ws + s.y);
  if (is_f32)
    hipLaunchKernelGGL(mx4_combine_kernel<float>, grid, block, 0, as_stream(stream), y, pos, offsets,
                       static_cast<int>(E), weights, static_cast<int>(H), static_cast<int>(k),
                       static_cast<int>(per_row), static_cast<float*>(out));
  else
    hipLaunchKernelGGL(mx4_combine_kernel<bf16_t>, grid, block, 0, as_stream(stream), y, pos, offsets,
                       static_cast<int>(E), weights, static_cast<int>(H), static_cast<int>(k),
                       static_cast<int>(per_row), static_cast<bf16_t*>(out));
  return launch_status("moe_mx4_experts(combine)");
}
