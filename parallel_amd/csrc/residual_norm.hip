// The residual stream around a block: the block's output normed (or not),
// gated, scaled and added to the residual, and the sum normed for the next
// block, forward and backward, in one launch each (plus the column sums').
//
// Per row of H values, everything in fp32 from the rows as they are stored:
//   v = y * ry * post (ry = rsqrt(mean(y^2) + eps)), or v = y without post
//   h = residual_scale * residual + branch_scale * g * v
//   x = h * r * gamma,  r = rsqrt(mean(h^2) + eps)
// Only hidden and x are rounded, once each: x is normed from h in fp32, not
// from the rounded hidden, and the backward forms h again from y and residual
// (which it reads either way, so that hidden need not be kept).
// Its gradients, with dH and dX those of hidden and x, e = dX * gamma:
//   dh = dH + r e - (r^3 / H) h sum_j(e_j h_j)
//   d_residual = residual_scale dh,   dz = branch_scale g dh
//   d_gate = branch_scale dh v (summed over what g is broadcast over)
//   dy = dz, or with post, f = dz * post:  ry f - (ry^3 / H) y sum_j(f_j y_j)
//   d_gamma = sum_t dX h r,   d_post = sum_t dz y ry
//
// Both are bound by the row streams (forward 4, backward 6, or 5 where dy and
// d_residual are the same numbers and the caller takes one tensor for both).
// A row is held in registers, by one wave (H <= 512) or by a block of four or,
// backward above 4096, eight (WPR waves per row, NC 8-value chunks per lane).
// The backward's waves walk several rows, as many walkers as run at once, and
// keep the column sums in registers, so that the partials are a few
// thousandths of the streams, and one more launch adds the partial rows in a
// fixed order: no atomics, the same bits every time.  The sums' registers leave
// two or three waves per SIMD, too few to hide a row's loads behind the others'
// sums, so the next row's loads are issued before this one's sums.
//
// Measured, inputs not in cache (a copy of 1 GiB: 5.1 TB/s): forward 16384 x
// 2048 bf16 49 us (268 MB), 8192 x 8192 101 us (537 MB); backward 71 (336 MB)
// and 132 (671 MB).  Backward with post and a gate per token: 5003 x 4096 70 us
// (246 MB), 90 with each row's loads behind the last one's stores; 16384 x 2048
// 103 against 121; 8192 x 8192 190 against 350 with four waves a row, whose 256
// registers leave one wave per SIMD.  The plain sum of one chunk a lane has
// registers for five waves and loses by it (73 against 71): it does not.
#include <type_traits>

#include "common.h"

namespace moe {

enum { kGateNone = 0, kGateToken = 1, kGateChannel = 2, kGateFull = 3 };

// Eight values as they are stored.
template <class T>
struct RnRaw {
  uint4 v[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int j = 0; j < static_cast<int>(sizeof(T) / 2); ++j) v[j] = reinterpret_cast<const uint4*>(p)[j];
  }
  __device__ __forceinline__ void values(float (&f)[8]) const {
    if constexpr (std::is_same<T, float>::value) {
      const float4 a = __builtin_bit_cast(float4, v[0]), b = __builtin_bit_cast(float4, v[1]);
      f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
      f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    } else {
      f[0] = lo_bf16(v[0].x); f[1] = hi_bf16(v[0].x);
      f[2] = lo_bf16(v[0].y); f[3] = hi_bf16(v[0].y);
      f[4] = lo_bf16(v[0].z); f[5] = hi_bf16(v[0].z);
      f[6] = lo_bf16(v[0].w); f[7] = hi_bf16(v[0].w);
    }
  }
};
template <class T>
__device__ __forceinline__ void rn_load8(const T* p, float (&f)[8]) {
  RnRaw<T> raw;
  raw.load(p);
  raw.values(f);
}
template <class T>
__device__ __forceinline__ void rn_store8(T* p, const float (&f)[8]) {
  if constexpr (std::is_same<T, float>::value) {
    reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
  } else {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]),
                                              pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
  }
}
template <class T>
__device__ __forceinline__ float rn_load1(const T* p) {
  if constexpr (std::is_same<T, float>::value) return *p;
  else return bf16_to_f32(*p);
}
template <class T>
__device__ __forceinline__ void rn_store1(T* p, float v) {
  if constexpr (std::is_same<T, float>::value) *p = v;
  else *p = f32_to_bf16(v);
}

// Threads per block: a row's waves (WPR of them), four rows of one wave each.
constexpr int rn_threads(int wpr) { return wpr > 4 ? wpr * kWave : 4 * kWave; }

// Sums over a row's lanes.  A row's waves exchange their sums through one of
// two LDS slots in turn: a slot is written again only after the barrier of the
// sum between, which every wave reaches after it has read the slot.
template <int WPR>
struct RowSum {
  float2 (*slots)[WPR];
  int turn;
  __device__ __forceinline__ float2 operator()(float a, float b) {
    a = wave_sum(a);
    b = wave_sum(b);
    if constexpr (WPR == 1) {
      return make_float2(a, b);
    } else {
      float2* s = slots[turn];
      turn ^= 1;
      if ((threadIdx.x & (kWave - 1)) == 0) s[threadIdx.x >> 6] = make_float2(a, b);
      __syncthreads();
      float2 sum = s[0];
#pragma unroll
      for (int w = 1; w < WPR; ++w) sum = make_float2(sum.x + s[w].x, sum.y + s[w].y);
      return sum;
    }
  }
};

struct RnFwd {
  const void *y, *residual, *post, *gate, *gamma;
  int gate_kind, T, H;
  float branch_scale, residual_scale, eps;
  void *hidden, *x;
  float *rstd_y, *rstd;
};

template <class E, int NC, int WPR>
__global__ __launch_bounds__(rn_threads(WPR)) void residual_norm_fwd_kernel(const RnFwd p) {
  __shared__ float2 slots[2][WPR];
  RowSum<WPR> row_sum{slots, 0};
  constexpr int kLanes = WPR * kWave;
  const int lane = threadIdx.x % kLanes;
  const int t = blockIdx.x * (rn_threads(WPR) / kLanes) + threadIdx.x / kLanes;  // one row per block where WPR is 4
  if (t >= p.T) return;
  const int n = p.H / 8;
  const int64_t base = static_cast<int64_t>(t) * p.H;
  const E* yr = static_cast<const E*>(p.y) + base;
  const E* rr = static_cast<const E*>(p.residual) + base;
  const float inv_h = 1.0f / static_cast<float>(p.H);
  float v[NC][8], res[NC][8];
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int c = lane + i * kLanes;
    if (c < n) {
      rn_load8(yr + 8 * c, v[i]);
      rn_load8(rr + 8 * c, res[i]);
#pragma unroll
      for (int e = 0; e < 8; ++e) ss += v[i][e] * v[i][e];
    }
  }
  float ry = 1.0f;
  if (p.post) {
    ry = rsqrtf(row_sum(ss, 0.0f).x * inv_h + p.eps);
    if (lane == 0 && p.rstd_y) p.rstd_y[t] = ry;
  }
  const float gt = p.gate_kind == kGateToken ? rn_load1(static_cast<const E*>(p.gate) + t) : 1.0f;
  const E* gr = static_cast<const E*>(p.gate) + (p.gate_kind == kGateFull ? base : 0);
  ss = 0.0f;
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int c = lane + i * kLanes;
    if (c < n) {
      if (p.post) {
        float w[8];
        rn_load8(static_cast<const E*>(p.post) + 8 * c, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] = v[i][e] * ry * w[e];
      }
      if (p.gate_kind >= kGateChannel) {
        float g[8];
        rn_load8(gr + 8 * c, g);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] *= g[e];
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] *= gt;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[i][e] = p.residual_scale * res[i][e] + p.branch_scale * v[i][e];
        ss += v[i][e] * v[i][e];
      }
      rn_store8(static_cast<E*>(p.hidden) + base + 8 * c, v[i]);
    }
  }
  const float r = rsqrtf(row_sum(ss, 0.0f).x * inv_h + p.eps);
  if (lane == 0 && p.rstd) p.rstd[t] = r;
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int c = lane + i * kLanes;
    if (c < n) {
      float w[8];
      rn_load8(static_cast<const E*>(p.gamma) + 8 * c, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] = v[i][e] * r * w[e];
      rn_store8(static_cast<E*>(p.x) + base + 8 * c, v[i]);
    }
  }
}

struct RnBwd {
  const void *d_hidden, *d_x, *y, *residual, *post, *gate, *gamma;
  const float *rstd_y, *rstd;
  int gate_kind, T, H, parts;  // parts: row walkers, one row of each kind of partials per walker
  float branch_scale, residual_scale;
  void *d_y, *d_residual, *d_gate;
  float* partials;  // [d_gamma, then d_post if post, then d_gate if per channel][parts][H]
};

// EXTRA: 0 the plain sum, whose registers are all it keeps; 1 with post or a gate; 2 with a gate per channel.
template <class E, int NC, int WPR, int EXTRA>
__global__ __launch_bounds__(rn_threads(WPR)) void residual_norm_bwd_kernel(const RnBwd p) {
  __shared__ float2 slots[2][WPR];
  RowSum<WPR> row_sum{slots, 0};
  constexpr int kLanes = WPR * kWave;
  constexpr bool WHOLE = EXTRA > 0, channel = EXTRA == 2;
  const int lane = threadIdx.x % kLanes;
  const int part = blockIdx.x * (rn_threads(WPR) / kLanes) + threadIdx.x / kLanes;
  if (part >= p.parts) return;
  const int n = p.H / 8;
  const float inv_h = 1.0f / static_cast<float>(p.H);
  const bool post = WHOLE && p.post;
  float sum_gamma[NC][8], sum_post[WHOLE ? NC : 1][8], sum_gate[channel ? NC : 1][8];
#pragma unroll
  for (int i = 0; i < NC; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      sum_gamma[i][e] = 0.0f;
      if constexpr (WHOLE) sum_post[i][e] = 0.0f;
      if constexpr (channel) sum_gate[i][e] = 0.0f;
    }
  // A row as it is read.  Where registers allow, the next row's loads are in flight while this one is summed.
  constexpr bool AHEAD = NC > 1 || EXTRA > 0;
  RnRaw<E> y_in[NC], res_in[NC], dx_in[NC], dh_in[NC];
  float r_in = 0.0f, ry_in = 1.0f, gt_in = 1.0f;
  auto fetch = [&](int t) __attribute__((always_inline)) {
    const int64_t base = static_cast<int64_t>(t) * p.H;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = lane + i * kLanes;
      if (c < n) {
        y_in[i].load(static_cast<const E*>(p.y) + base + 8 * c);
        res_in[i].load(static_cast<const E*>(p.residual) + base + 8 * c);
        if (p.d_x) dx_in[i].load(static_cast<const E*>(p.d_x) + base + 8 * c);
        if (p.d_hidden) dh_in[i].load(static_cast<const E*>(p.d_hidden) + base + 8 * c);
      }
    }
    r_in = p.rstd[t];
    if (post) ry_in = p.rstd_y[t];
    if (WHOLE && p.gate_kind == kGateToken) gt_in = rn_load1(static_cast<const E*>(p.gate) + t);
  };
  if (AHEAD && part < p.T) fetch(part);
  for (int t = part; t < p.T; t += p.parts) {  // the same count for every wave of a row: barriers match
    const int64_t base = static_cast<int64_t>(t) * p.H;
    if (!AHEAD) fetch(t);
    const float r = r_in, ry = ry_in, gt = gt_in;
    const E* gr = static_cast<const E*>(p.gate) + (p.gate_kind == kGateFull ? base : 0);
    float yv[NC][8], h[NC][8], dh[NC][8];
    float dot = 0.0f;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = lane + i * kLanes;
      if (c < n) {
        y_in[i].values(yv[i]);
        res_in[i].values(h[i]);
        float w[8], g[8], v[8], dx[8];
        if (p.d_x) dx_in[i].values(dx);
        if (p.d_hidden) dh_in[i].values(dh[i]);
        else
#pragma unroll
          for (int e = 0; e < 8; ++e) dh[i][e] = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = yv[i][e];
        if constexpr (WHOLE) {
          if (post) {
            rn_load8(static_cast<const E*>(p.post) + 8 * c, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = v[e] * ry * w[e];
          }
          if (p.gate_kind >= kGateChannel) {
            rn_load8(gr + 8 * c, g);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] *= g[e];
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] *= gt;
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) h[i][e] = p.residual_scale * h[i][e] + p.branch_scale * v[e];
        if (p.d_x) {
          rn_load8(static_cast<const E*>(p.gamma) + 8 * c, w);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            sum_gamma[i][e] += dx[e] * h[i][e] * r;
            dot += dx[e] * w[e] * h[i][e];
            dh[i][e] += r * (dx[e] * w[e]);
          }
        }
      }
    }
    if (AHEAD && t + p.parts < p.T) fetch(t + p.parts);
    if (p.d_x) {
      const float k = r * r * r * inv_h * row_sum(dot, 0.0f).x;
#pragma unroll
      for (int i = 0; i < NC; ++i)
        if (lane + i * kLanes < n)
#pragma unroll
          for (int e = 0; e < 8; ++e) dh[i][e] -= k * h[i][e];
    }
    float dot_y = 0.0f, dot_g = 0.0f;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = lane + i * kLanes;
      if (c < n) {
        float o[8];
        if (p.d_residual) {
#pragma unroll
          for (int e = 0; e < 8; ++e) o[e] = p.residual_scale * dh[i][e];
          rn_store8(static_cast<E*>(p.d_residual) + base + 8 * c, o);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) dh[i][e] *= p.branch_scale;
        if constexpr (WHOLE) {
          float w[8], g[8];
          if (post) rn_load8(static_cast<const E*>(p.post) + 8 * c, w);
          if (p.gate_kind >= kGateChannel) rn_load8(gr + 8 * c, g);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float q = post ? yv[i][e] * ry : yv[i][e];  // v without post's weight
            o[e] = dh[i][e] * (post ? q * w[e] : q);          // the gate's gradient
            dot_g += o[e];
            if constexpr (channel) sum_gate[i][e] += o[e];
            const float dz = dh[i][e] * (p.gate_kind >= kGateChannel ? g[e] : gt);
            if (post) {
              sum_post[i][e] += dz * q;
              dh[i][e] = dz * w[e];
              dot_y += dh[i][e] * yv[i][e];
            } else {
              dh[i][e] = dz;
            }
          }
          if (p.gate_kind == kGateFull) rn_store8(static_cast<E*>(p.d_gate) + base + 8 * c, o);
        }
        if (!post && p.d_y) rn_store8(static_cast<E*>(p.d_y) + base + 8 * c, dh[i]);
      }
    }
    if constexpr (WHOLE) {
      if (post || p.gate_kind == kGateToken) {
        const float2 s = row_sum(dot_y, dot_g);
        if (p.gate_kind == kGateToken && lane == 0) rn_store1(static_cast<E*>(p.d_gate) + t, s.y);
        if (post) {
          const float k = ry * ry * ry * inv_h * s.x;
#pragma unroll
          for (int i = 0; i < NC; ++i) {
            const int c = lane + i * kLanes;
            if (c < n) {
              float o[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) o[e] = ry * dh[i][e] - k * yv[i][e];
              rn_store8(static_cast<E*>(p.d_y) + base + 8 * c, o);
            }
          }
        }
      }
    }
  }
  const int64_t kind = static_cast<int64_t>(p.parts) * p.H;
  float* out = p.partials + static_cast<int64_t>(part) * p.H;
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int c = lane + i * kLanes;
    if (c < n) {
      rn_store8(out + 8 * c, sum_gamma[i]);
      if constexpr (WHOLE) {
        if (post) rn_store8(out + kind + 8 * c, sum_post[i]);
      }
      if constexpr (channel) rn_store8(out + (post ? 2 : 1) * kind + 8 * c, sum_gate[i]);
    }
  }
}

// out[j] = sum of column j over the parts: 32 columns per block (a line of
// 128 bytes of each part), 32 threads taking every 32nd part each, then the
// threads' sums in order.
constexpr int kRnSumThreads = 1024;
template <class E>
__global__ __launch_bounds__(kRnSumThreads) void residual_norm_sums_kernel(const float* __restrict__ partials,
                                                                           int parts, int H, E* out0, E* out1,
                                                                           E* out2) {
  __shared__ float part[32][33];
  const int col = threadIdx.x & 31, row = threadIdx.x >> 5;
  const int j = blockIdx.x * 32 + col;
  const float* src = partials + static_cast<int64_t>(blockIdx.y) * parts * H + j;
  float acc = 0.0f;
  if (j < H) {
#pragma unroll 8
    for (int q = row; q < parts; q += 32) acc += src[static_cast<int64_t>(q) * H];
  }
  part[row][col] = acc;
  __syncthreads();
  if (row == 0 && j < H) {
    float s = 0.0f;
#pragma unroll
    for (int q = 0; q < 32; ++q) s += part[q][col];
    E* out = blockIdx.y == 0 ? out0 : blockIdx.y == 1 ? out1 : out2;
    rn_store1(out + j, s);
  }
}

}  // namespace moe

using namespace moe;

namespace {
constexpr int64_t kRnMaxH = 8192;

int check_rn(const char* what, const void* y, const void* residual, const void* gate, int gate_kind, const void* gamma,
             const void* post, int64_t T, int64_t H) {
  // (a walker's next row, at most 4096 on, stays an int)
  MOE_REQUIRE(T >= 0 && T <= (1ll << 30), MOE_ERR_INVALID, "%s: bad row count %lld", what, (long long)T);
  MOE_REQUIRE(H > 0 && H % 8 == 0 && H <= kRnMaxH, MOE_ERR_UNSUPPORTED,
              "%s: H=%lld must be a multiple of 8 and at most %lld", what, (long long)H, (long long)kRnMaxH);
  MOE_REQUIRE(gate_kind >= kGateNone && gate_kind <= kGateFull, MOE_ERR_INVALID, "%s: bad gate kind %d", what,
              gate_kind);
  MOE_REQUIRE(gamma && aligned16(gamma) && aligned16(post), MOE_ERR_INVALID, "%s: bad weight pointer", what);
  if (T == 0) return MOE_OK;
  MOE_REQUIRE(y && residual && (gate || gate_kind == kGateNone), MOE_ERR_INVALID, "%s: null pointer", what);
  MOE_REQUIRE(aligned16(y) && aligned16(residual) && aligned16(gate), MOE_ERR_INVALID,
              "%s: operands must be 16-byte aligned", what);
  return MOE_OK;
}

// Waves per row and chunks per lane for a width: one wave holds a row of up to
// 512 values; wider rows take four.
bool wave_rows(int64_t H) { return H <= 512; }

// Row walkers of the backward, each a row of partials: at most 1024 blocks (the workspace's size), and as many as run
// at once, so that no block starts when the others end.
constexpr int64_t kRnBlocks = 1024;
int64_t rn_parts(int64_t T, int64_t H, int64_t blocks) {
  const int64_t most = (wave_rows(H) ? 4 : 1) * blocks;
  return T < 1 ? 1 : T < most ? T : most;
}

template <bool BWD, class F>
void rn_dispatch(int64_t H, F&& f) {
  using std::integral_constant;
  if (wave_rows(H)) f(integral_constant<int, 1>{}, integral_constant<int, 1>{});
  else if (H <= 2048) f(integral_constant<int, 1>{}, integral_constant<int, 4>{});
  else if (H <= 4096) f(integral_constant<int, 2>{}, integral_constant<int, 4>{});
  else f(integral_constant<int, BWD ? 2 : 4>{}, integral_constant<int, BWD ? 8 : 4>{});
}
}  // namespace

extern "C" int moe_residual_norm_fwd(const void* y, const void* residual, const void* post, const void* gate,
                                     int gate_kind, const void* gamma, int is_f32, int64_t T, int64_t H,
                                     float branch_scale, float residual_scale, float eps, void* hidden, void* x,
                                     float* rstd_y, float* rstd, void* stream) {
  int rc = check_rn("residual_norm fwd", y, residual, gate, gate_kind, gamma, post, T, H);
  if (rc) return rc;
  MOE_REQUIRE(eps >= 0.0f, MOE_ERR_INVALID, "residual_norm fwd: eps must be non-negative");
  if (T == 0) return MOE_OK;
  MOE_REQUIRE(hidden && x && aligned16(hidden) && aligned16(x), MOE_ERR_INVALID,
              "residual_norm fwd: bad output pointer");
  const RnFwd p{y,      residual, post, gate, gamma, gate_kind, static_cast<int>(T), static_cast<int>(H), branch_scale,
                residual_scale, eps, hidden, x, rstd_y, rstd};
  rn_dispatch<false>(H, [&](auto nc, auto wpr) {
    constexpr int NC = decltype(nc)::value, WPR = decltype(wpr)::value, per = rn_threads(WPR) / (WPR * kWave);
    const dim3 grid(static_cast<unsigned>((T + per - 1) / per));
    if (is_f32)
      hipLaunchKernelGGL((residual_norm_fwd_kernel<float, NC, WPR>), grid, dim3(rn_threads(WPR)), 0, as_stream(stream), p);
    else
      hipLaunchKernelGGL((residual_norm_fwd_kernel<bf16_t, NC, WPR>), grid, dim3(rn_threads(WPR)), 0, as_stream(stream), p);
  });
  return launch_status("moe_residual_norm_fwd");
}

extern "C" size_t moe_residual_norm_bwd_workspace_bytes(int64_t T, int64_t H) {
  if (T < 0 || H < 1) return 0;
  return static_cast<size_t>(3 * rn_parts(T, H, kRnBlocks)) * static_cast<size_t>(H) * sizeof(float);
}

extern "C" int moe_residual_norm_bwd(const void* d_hidden, const void* d_x, const void* y, const void* residual,
                                     const void* post, const void* gate, int gate_kind, const void* gamma,
                                     const float* rstd_y, const float* rstd, int is_f32, int64_t T, int64_t H,
                                     float branch_scale, float residual_scale, void* d_y, void* d_residual,
                                     void* d_post, void* d_gate, void* d_gamma, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  int rc = check_rn("residual_norm bwd", y, residual, gate, gate_kind, gamma, post, T, H);
  if (rc) return rc;
  const bool channel = gate_kind == kGateChannel, full = gate_kind == kGateFull;
  MOE_REQUIRE(d_gamma && (d_post || !post) && (d_gate || !channel), MOE_ERR_INVALID,
              "residual_norm bwd: null weight gradient");
  if (T > 0) {
    MOE_REQUIRE(rstd && (rstd_y || !post) && (d_gate || gate_kind == kGateNone), MOE_ERR_INVALID,
                "residual_norm bwd: null pointer");
    MOE_REQUIRE((d_residual || d_y) && (d_y || (!post && gate_kind == kGateNone)), MOE_ERR_INVALID,
                "residual_norm bwd: null input gradient");
    MOE_REQUIRE(aligned16(d_hidden) && aligned16(d_x) && aligned16(d_y) && aligned16(d_residual) &&
                    (!full || aligned16(d_gate)),
                MOE_ERR_INVALID, "residual_norm bwd: operands must be 16-byte aligned");
  }
  const size_t need = moe_residual_norm_bwd_workspace_bytes(T, H);
  MOE_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= need, MOE_ERR_WORKSPACE,
              "residual_norm bwd: workspace %zu < %zu bytes", workspace_bytes, need);
  RnBwd p{d_hidden, d_x, y, residual, post, gate, gamma, rstd_y, rstd, gate_kind, static_cast<int>(T),
          static_cast<int>(H), 0, branch_scale, residual_scale, d_y, d_residual, d_gate,
          static_cast<float*>(workspace)};
  rn_dispatch<true>(H, [&](auto nc, auto wpr) {  // (with T == 0 the one walker writes its zero sums)
    constexpr int NC = decltype(nc)::value, WPR = decltype(wpr)::value, per = rn_threads(WPR) / (WPR * kWave);
    auto launch = [&](auto e, auto extra) {
      const auto kernel = residual_norm_bwd_kernel<decltype(e), NC, WPR, decltype(extra)::value>;
      const int dev = current_device();
      const int64_t fit = static_cast<int64_t>(device_cus(dev)) *
                          cached_blocks_per_cu(dev, reinterpret_cast<const void*>(kernel), rn_threads(WPR), 0);
      p.parts = static_cast<int>(rn_parts(T, H, fit < kRnBlocks ? fit : kRnBlocks));
      hipLaunchKernelGGL(kernel, dim3((p.parts + per - 1) / per), dim3(rn_threads(WPR)), 0, as_stream(stream), p);
    };
    auto typed = [&](auto e) {
      if (channel) launch(e, std::integral_constant<int, 2>{});
      else if (post || gate_kind != kGateNone) launch(e, std::integral_constant<int, 1>{});
      else launch(e, std::integral_constant<int, 0>{});
    };
    if (is_f32) typed(float{});
    else typed(bf16_t{});
  });
  rc = launch_status("moe_residual_norm_bwd(rows)");
  if (rc) return rc;
  const dim3 grid(static_cast<unsigned>((H + 31) / 32), 1 + (post ? 1 : 0) + (channel ? 1 : 0));
  void* second = post ? d_post : d_gate;
  if (is_f32)
    hipLaunchKernelGGL((residual_norm_sums_kernel<float>), grid, dim3(kRnSumThreads), 0, as_stream(stream), p.partials,
                       p.parts, static_cast<int>(H), static_cast<float*>(d_gamma), static_cast<float*>(second),
                       static_cast<float*>(d_gate));
  else
    hipLaunchKernelGGL((residual_norm_sums_kernel<bf16_t>), grid, dim3(kRnSumThreads), 0, as_stream(stream), p.partials,
                       p.parts, static_cast<int>(H), static_cast<bf16_t*>(d_gamma), static_cast<bf16_t*>(second),
                       static_cast<bf16_t*>(d_gate));
  return launch_status("moe_residual_norm_bwd(sums)");
}
