// Quantisation to microscaled 4-bit values and back, and the entry points of
// the grouped products (format: mx4.h).
//
// Either direction is one pass bound by HBM: a thread takes 8 values (16 bytes
// of bf16), four neighbouring lanes a block of 32, whose largest size two DPP
// moves find; the conversion instruction scales by a power of two and rounds
// to nearest even, saturating at 6.
#include <type_traits>

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

template <class E>
__global__ __launch_bounds__(kMx4Threads) void mx4_dequantize_kernel(const uint32_t* __restrict__ codes,
                                                                     const uint8_t* __restrict__ scales, int64_t n8,
                                                                     int64_t K, E* __restrict__ out, int pad) {
  const int64_t step = static_cast<int64_t>(gridDim.x) * kMx4Threads;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kMx4Threads + threadIdx.x; i < n8; i += step) {
    int64_t at = i >> 2;
    if (pad) at += at / (K / 32) * pad;
    const uint32_t c = codes[i];
    const int s = scales[at];
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t n = (c >> (4 * e)) & 15u, m = n & 7u;  // m: exponent field and mantissa bit; 0.5 is subnormal
      const float size = m < 2 ? 0.5f * static_cast<float>(m) : __uint_as_float((126u + (m >> 1)) << 23 | (m & 1u) << 22);
      const float v = s == 255 ? __uint_as_float(0x7fc00000u) : ldexpf(size, s - 127);
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

// Blocks of a pass over n8 chunks of 8 values: enough to fill the card, each
// thread taking several chunks of a large pass.
unsigned pass_blocks(int64_t n8) {
  const int64_t blocks = (n8 + kMx4Threads - 1) / kMx4Threads;
  return static_cast<unsigned>(blocks < 16384 ? blocks : 16384);
}

int run_product(const char* what, const void* a, const void* a_scales, int64_t a_rows, const int32_t* row_index,
                int64_t row_div, const void* w, const void* w_scales, const int32_t* offs, int64_t G, int64_t M,
                int64_t N, int64_t K, void* c, void* c_codes, void* c_scales, int epi, void* stream) {
  const int64_t wide = epi == MX4_PLAIN ? N : 2 * N;
  MOE_REQUIRE(G > 0 && M >= 0 && a_rows >= 0 && N > 0 && K > 0 && row_div > 0, MOE_ERR_INVALID, "%s: bad sizes", what);
  MOE_REQUIRE(K % 32 == 0 && N % 8 == 0, MOE_ERR_UNSUPPORTED, "%s: K=%lld must be a multiple of 32, N=%lld of 8", what,
              (long long)K, (long long)N);
  MOE_REQUIRE(epi != MX4_SWIGLU_MX4 || N % 32 == 0, MOE_ERR_UNSUPPORTED,
              "%s: 4-bit output of %lld columns is not whole blocks of 32", what, (long long)N);
  MOE_REQUIRE(M < (1ll << 31) && a_rows < (1ll << 31) && G < (1ll << 24) && row_div < (1ll << 31) && N < (1ll << 28) &&
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
  p.row_div = static_cast<int>(row_div);
  // Granlund and Montgomery's multiplier: with l = ceil(log2 d), m = floor(2^(31+l) / d) + 1 divides 31-bit numbers.
  uint32_t l = 0;
  while ((1ll << l) < row_div) ++l;
  p.div_magic = static_cast<uint32_t>((1ull << (31 + l)) / static_cast<uint64_t>(row_div) + 1);
  p.div_shift = 31 + l;
  p.a_rows = static_cast<int>(a_rows);
  p.w = static_cast<const uint8_t*>(w);
  p.w_scales = static_cast<const uint8_t*>(w_scales);
  p.offs = offs;
  p.G = static_cast<int>(G);
  p.rows = static_cast<int>(M);
  p.N = static_cast<int>(N);
  p.K = static_cast<int>(K);
  p.c = static_cast<bf16_t*>(c);
  p.c_codes = static_cast<uint8_t*>(c_codes);
  p.c_scales = static_cast<uint8_t*>(c_scales);
  const int64_t mean = (M + G - 1) / G;
  if (mean <= 32) return mx4_few(p, epi, as_stream(stream), what);
  return mx4_tile(p, epi, mean <= 64 ? 64 : mean <= 128 ? 128 : 256, as_stream(stream), what);
}
}  // namespace

extern "C" int moe_mx4_quantize(const void* x, int is_f32, int64_t rows, int64_t K, void* codes, void* scales,
                                void* stream) {
  const int rc = check_rows("mx4 quantize", x, codes, scales, rows, K);
  if (rc || rows == 0) return rc;
  const int64_t n8 = rows * K / 8;
  const int pad = static_cast<int>(mx4_pitch(K) - K / 32);
  if (is_f32)
    hipLaunchKernelGGL(mx4_quantize_kernel<float>, dim3(pass_blocks(n8)), dim3(kMx4Threads), 0, as_stream(stream),
                       static_cast<const float*>(x), n8, K, static_cast<uint32_t*>(codes),
                       static_cast<uint8_t*>(scales), pad);
  else
    hipLaunchKernelGGL(mx4_quantize_kernel<bf16_t>, dim3(pass_blocks(n8)), dim3(kMx4Threads), 0, as_stream(stream),
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
  if (is_f32)
    hipLaunchKernelGGL(mx4_dequantize_kernel<float>, dim3(pass_blocks(n8)), dim3(kMx4Threads), 0, as_stream(stream),
                       static_cast<const uint32_t*>(codes), static_cast<const uint8_t*>(scales), n8, K,
                       static_cast<float*>(out), pad);
  else
    hipLaunchKernelGGL(mx4_dequantize_kernel<bf16_t>, dim3(pass_blocks(n8)), dim3(kMx4Threads), 0, as_stream(stream),
                       static_cast<const uint32_t*>(codes), static_cast<const uint8_t*>(scales), n8, K,
                       static_cast<bf16_t*>(out), pad);
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
