// Grouped products of mx4 operands for groups of many rows: LDS tiles of up to
// BM rows by 256 weight rows (128 act columns with swiglu, gate and up in
// 16-row turns), 256 values deep, so a row of a stage is one 128-byte line.
//
// Eight waves, two by rows and four by columns; wave row wm owns the 16-row
// tiles wm, wm + 2, ... (a partly filled tile then loads both), wave column wn
// the 64 weight rows 64 wn ...  Products are v_mfma_scale_f32_16x16x128 on
// codes and scales as they are stored: lane l multiplies the 32-blocks 2 (l /
// 16) and + 1 of a stage's row, so its two codes chunks are neighbours and its
// two scales one 16-bit read.
//
// Blocks are persistent, one per CU, and run one stream of stages over their
// tiles: a DMA cursor (buffer_load ... lds) fills a ring of STAGES stages
// STAGES - 1 ahead of the compute cursor and runs on across tiles, so that a
// tile's first stage is on its way while the last one's output is written.
// The epilogue turns each 16-row result into whole 16-byte pieces through the
// stage just multiplied (which the DMA reaches a barrier later); it issues the
// same number of stores whatever is in range (out of range ones are dropped by
// the buffer resource), so that the waits that follow can leave them in flight.
#include "dma.h"
#include "mx4.h"

namespace moe {
namespace {

constexpr int kTileWaves = 8, kTileThreads = kTileWaves * kWave;
constexpr int kTileN = 256;     // weight rows per tile
constexpr int kGroupRegs = 4;   // groups held in registers, 64 each
constexpr int kXcds = 8;

// 4 bytes per lane from `rsrc` + voffset into LDS at M0 + 4 lane (dma16 for scales).
__device__ __forceinline__ void dma4(u32x4_t rsrc, uint32_t voffset, uint32_t lds_addr) {
  asm volatile("s_nop 4\n\tbuffer_load_dword %0, %1, 0 offen lds" ::"v"(voffset), "s"(rsrc), "{m0}"(lds_addr)
               : "memory");
}

// The groups' first rows and counts, one group per lane and register.
struct Groups {
  int lo[kGroupRegs], cnt[kGroupRegs];
  __device__ __forceinline__ void load(const Mx4Gemm& p) {
#pragma unroll
    for (int c = 0; c < kGroupRegs; ++c) cnt[c] = mx4_group_rows(p, c * kWave + (threadIdx.x & (kWave - 1)), lo[c]);
  }
  // f(first group, lo, cnt) for each 64 groups until it returns true.
  template <class F>
  __device__ __forceinline__ void each(const Mx4Gemm& p, F&& f) const {
#pragma unroll
    for (int c = 0; c < kGroupRegs; ++c)
      if (c * kWave < p.G && f(c * kWave, lo[c], cnt[c])) return;
    for (int c0 = kGroupRegs * kWave; c0 < p.G; c0 += kWave) {
      int l;
      const int n = mx4_group_rows(p, c0 + (threadIdx.x & (kWave - 1)), l);
      if (f(c0, l, n)) return;
    }
  }
};

template <int BM, int STAGES, int EPI>
__global__ __launch_bounds__(kTileThreads) void mx4_tile_kernel(const Mx4Gemm p, int n_tiles) {
  constexpr bool GLU = EPI != MX4_PLAIN;
  constexpr int WM = 2, MT = BM / 16 / WM, NT = 4;
  constexpr int kCols = GLU ? kTileN / 2 : kTileN;     // output columns per tile
  constexpr int LA = BM / 64, LB = kTileN / 64;        // code DMAs per wave and stage (8 rows each)
  constexpr int LPW = LA + LB + 2;                     // and one for either operand's scales (32 rows each)
  constexpr int kB = BM * 128, kAs = kB + kTileN * 128, kBs = kAs + BM * 8, kSpare = kBs + kTileN * 8;
  constexpr int kStage = (kSpare + 256 + 1023) / 1024 * 1024;  // the spare 256 bytes take scale DMAs of rows past BM
  constexpr int kStores = EPI == MX4_PLAIN ? 2 * MT : EPI == MX4_SWIGLU ? MT : 2 * ((MT * 16 + 63) / 64);
  constexpr int kSlot = 16 * 144;                      // a wave's epilogue staging: 16 rows of 64 bf16, 16 bytes apart
  static_assert(kTileWaves * kSlot <= kStage && MT * 16 * 17 <= kSlot, "the epilogue stages in one ring stage");
  static_assert(STAGES * kStage <= 160 * 1024, "LDS");
  static_assert((STAGES - 2) * LPW + kStores < 64, "vmcnt range");
  __shared__ __attribute__((aligned(1024))) char ring[STAGES * kStage];

  const int lane = threadIdx.x & (kWave - 1), i16 = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave & 1, wn = wave >> 1;
  const int64_t wide = GLU ? 2 * static_cast<int64_t>(p.N) : p.N;
  const uint32_t half_k = static_cast<uint32_t>(p.K) / 2, pitch = static_cast<uint32_t>(mx4_pitch(p.K));
  const int blocks = p.K / 32, nk = (p.K + 255) / 256;

  Groups groups;
  groups.load(p);
  int total = 0;
  groups.each(p, [&](int, int, int cnt) {
    total += __builtin_amdgcn_readlane(wave_inclusive_scan((cnt + BM - 1) / BM), kWave - 1);
    return false;
  });
  total = __builtin_amdgcn_readfirstlane(total) * n_tiles;
  // This block's tiles: every nbx-th of its XCD's contiguous share.
  const int nbx = gridDim.x / kXcds, xcd = blockIdx.x % kXcds, xidx = blockIdx.x / kXcds;
  const int share = (total + kXcds - 1) / kXcds, first = xcd * share + xidx;
  const int span = min(share, total - xcd * share);
  const int ntiles = span > xidx ? (span - xidx + nbx - 1) / nbx : 0;
  if (ntiles <= 0) return;  // the whole block

  auto find = [&](int j) __attribute__((always_inline)) {  // tile j of the block's (j < ntiles)
    Mx4Tile t{0, 0, 0, 0};
    const int tile = first + j * nbx;
    int base = 0;
    groups.each(p, [&](int c0, int lo, int cnt) {
      const int n = n_tiles * ((cnt + BM - 1) / BM);
      const int incl = wave_inclusive_scan(n);
      const int tot = __builtin_amdgcn_readlane(incl, kWave - 1);
      if (tile >= base + tot) {
        base += tot;
        return false;
      }
      const int w = __builtin_amdgcn_readfirstlane(__builtin_ctzll(__ballot(base + incl > tile)));
      const int local = tile - base - __builtin_amdgcn_readlane(incl - n, w);
      const int rows = __builtin_amdgcn_readlane(cnt, w), parts = (rows + BM - 1) / BM;
      const int per = ((rows + parts - 1) / parts + 15) & ~15;
      const int nt = local / parts, part = local - nt * parts;
      t = Mx4Tile{c0 + w, __builtin_amdgcn_readlane(lo, w) + part * per, min(per, rows - part * per), nt};
      return true;
    });
    t.g = __builtin_amdgcn_readfirstlane(t.g);
    t.r0 = __builtin_amdgcn_readfirstlane(t.r0);
    t.rows = __builtin_amdgcn_readfirstlane(t.rows);
    t.n = __builtin_amdgcn_readfirstlane(t.n);
    return t;
  };

  // ------------------------------------------------------------ DMA cursor
  // Code DMA j of a wave fills rows 8 (wave L + j) .. + 7 of an operand, lane l
  // the 16-byte slot l % 8 of row l / 8; slot s of row r holds chunk s ^ ((r /
  // 2) % 8), so that the 16 rows of a fragment read lie on distinct banks.
  // The scale DMA of a wave fills rows 32 wave .. + 31, lane l half l % 2 of row l / 2.
  const uint32_t lds0 = lds_address(ring);
  const u32x4_t ra = rsrc_words(p.a, static_cast<uint32_t>(p.a_rows) * half_k);
  const u32x4_t ras = rsrc_words(p.a_scales, static_cast<uint32_t>(p.a_rows) * pitch);
  u32x4_t rb = ra, rbs = ra;
  uint32_t a_off[LA], b_off[LB], as_off, bs_off;  // at stage 0; kOOB for rows past the end
  int next_row[LA + 1];  // the source rows of the tile behind the cursor's (gathered activations), -1 past its end
  const int l8 = lane >> 3, slot = lane & 7;
  auto chunk_of = [&](int r) { return static_cast<uint32_t>(slot ^ ((r >> 1) & 7)); };
  auto tile_row = [&](int j) { return j < LA ? 8 * (wave * LA + j) + l8 : 32 * wave + (lane >> 1); };
  int dj = -1, dk = nk;
  auto fetch_rows = [&](int j) __attribute__((always_inline)) {
    Mx4Tile t{0, 0, 0, 0};
    if (j < ntiles) t = find(j);
#pragma unroll
    for (int n = 0; n <= LA; ++n) {
      const int r = tile_row(n);
      next_row[n] = r < t.rows ? t.r0 + r : -1;
      if (p.row_index && r < t.rows) next_row[n] = p.row_index[t.r0 + r] / p.row_div;
    }
  };
  auto seek = [&]() __attribute__((always_inline)) {  // to the next tile's first stage
    ++dj;
    dk = 0;
    const bool live = dj < ntiles;
    Mx4Tile t{0, 0, 0, 0};
    if (live) t = find(dj);
    auto source = [&](int n) { return next_row[n] >= 0 && next_row[n] < p.a_rows; };
#pragma unroll
    for (int j = 0; j < LA; ++j)
      a_off[j] = source(j) ? static_cast<uint32_t>(next_row[j]) * half_k + 16u * chunk_of(tile_row(j)) : kOOB;
    as_off = source(LA) ? static_cast<uint32_t>(next_row[LA]) * pitch + 4u * (lane & 1) : kOOB;
    auto weight_row = [&](int r, bool& in) {
      const int n = t.n * kCols + (GLU ? (r >> 5) * 16 + (r & 15) : r);
      in = live && n < p.N;
      return static_cast<uint32_t>(GLU && (r & 16) ? p.N + n : n);
    };
    bool in;
#pragma unroll
    for (int j = 0; j < LB; ++j) {
      const int r = 8 * (wave * LB + j) + l8;
      const uint32_t w = weight_row(r, in);
      b_off[j] = in ? w * half_k + 16u * chunk_of(r) : kOOB;
    }
    const uint32_t w = weight_row(32 * wave + (lane >> 1), in);
    bs_off = in ? w * pitch + 4u * (lane & 1) : kOOB;
    rb = rsrc_words(p.w + t.g * wide * half_k, static_cast<uint32_t>(wide) * half_k);
    rbs = rsrc_words(p.w_scales + t.g * wide * pitch, static_cast<uint32_t>(wide) * pitch);
    fetch_rows(dj + 1);
  };
  auto issue = [&](int stage) __attribute__((always_inline)) {  // the cursor's stage into the ring, and on
    const uint32_t at = lds0 + stage * kStage;
    const uint32_t ahead = 128u * dk;
    auto chunk_in = [&](int r) { return 8 * dk + static_cast<int>(chunk_of(r)) < blocks; };
#pragma unroll
    for (int j = 0; j < LA; ++j) {
      const bool in = a_off[j] != kOOB && chunk_in(tile_row(j));
      dma16(ra, in ? a_off[j] + ahead : kOOB, __builtin_amdgcn_readfirstlane(at + 1024 * (wave * LA + j)));
    }
#pragma unroll
    for (int j = 0; j < LB; ++j) {
      const bool in = b_off[j] != kOOB && chunk_in(8 * (wave * LB + j) + l8);
      dma16(rb, in ? b_off[j] + ahead : kOOB, __builtin_amdgcn_readfirstlane(at + kB + 1024 * (wave * LB + j)));
    }
    dma4(ras, as_off != kOOB ? as_off + 8u * dk : kOOB,
         __builtin_amdgcn_readfirstlane(at + (32 * wave < BM ? kAs + 256 * wave : kSpare)));
    dma4(rbs, bs_off != kOOB ? bs_off + 8u * dk : kOOB, __builtin_amdgcn_readfirstlane(at + kBs + 256 * wave));
    if (++dk == nk) seek();
  };

  // -------------------------------------------------------- compute cursor
  const int a_lane = i16 * 128, swz = (i16 >> 1) & 7;
  f32x4_t acc[MT][NT];
  auto multiply = [&](const char* st, int k, int rows) __attribute__((always_inline)) {
    const int left = blocks - (8 * k + 2 * q);  // the lane's blocks inside K (scale padding may hold anything)
    const uint32_t keep = left > 1 ? 0xffffu : left > 0 ? 0xffu : 0u;
    uint32_t sw[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j)
      sw[j] = *reinterpret_cast<const uint16_t*>(st + kBs + (64 * wn + 16 * j + i16) * 8 + 2 * q) & keep;
    uint4 w[2][NT];
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int j = 0; j < NT; ++j)
        w[s][j] = *reinterpret_cast<const uint4*>(st + kB + (64 * wn + 16 * j) * 128 + a_lane + (((2 * q + s) ^ swz) << 4));
    // The next 16 rows' fragments are read while these are multiplied; tiles
    // without rows skip their products.
    uint4 a[2][2];
    uint32_t sa[2];
    auto read = [&](int i) __attribute__((always_inline)) {
      const int r = 16 * (wm + WM * i);
      sa[i & 1] = *reinterpret_cast<const uint16_t*>(st + kAs + (r + i16) * 8 + 2 * q) & keep;
#pragma unroll
      for (int s = 0; s < 2; ++s)
        a[i & 1][s] = *reinterpret_cast<const uint4*>(st + r * 128 + a_lane + (((2 * q + s) ^ swz) << 4));
    };
    read(0);
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      if (i + 1 < MT) read(i + 1);
      if (16 * (wm + WM * i) < rows) {  // wave-uniform
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = mx4_mfma<0>(w[0][j], a[i & 1][0], acc[i][j], sw[j], sa[i & 1]);
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = mx4_mfma<1>(w[1][j], a[i & 1][1], acc[i][j], sw[j], sa[i & 1]);
      }
    }
  };
  auto store = [&](char* st, const Mx4Tile& t) __attribute__((always_inline)) {
    char* mine = st + wave * kSlot;
    const int n0 = t.n * kCols + wn * (kCols / 4);  // the wave's first output column
    if constexpr (EPI == MX4_SWIGLU_MX4) {
      const auto rc = make_rsrc(p.c_codes + static_cast<int64_t>(t.r0) * (p.N / 2), static_cast<uint32_t>(t.rows) * (p.N / 2));
      const uint32_t out_pitch = static_cast<uint32_t>(mx4_pitch(p.N));
      const auto rs = make_rsrc(p.c_scales + static_cast<int64_t>(t.r0) * out_pitch, static_cast<uint32_t>(t.rows) * out_pitch);
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        float act[2][4];
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          act[e / 4][e % 4] = silu_f(acc[i][2 * (e / 4)][e % 4]) * acc[i][2 * (e / 4) + 1][e % 4];
          top = max(top, __float_as_uint(act[e / 4][e % 4]) & 0x7fffffffu);
        }
        top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 16)));
        top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 32)));
        const uint32_t s = mx4_scale(top);
        const float f = mx4_scale_f(s);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t c = 0;
          c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, act[h][0], act[h][1], f, 0);
          c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, act[h][2], act[h][3], f, 1);
          *reinterpret_cast<uint16_t*>(mine + (16 * i + i16) * 16 + 8 * h + 2 * q) =
              static_cast<uint16_t>(s == 255u ? 0u : c);
        }
        if (q == 0) mine[MT * 256 + 16 * i + i16] = static_cast<char>(s);
      }
#pragma unroll
      for (int h = 0; h < (MT * 16 + 63) / 64; ++h) {
        const int m = 64 * h + lane;                              // of the wave's rows
        const int row = 16 * (wm + WM * (m >> 4)) + (m & 15);     // of the tile's
        const bool in = m < MT * 16 && row < t.rows && n0 < p.N;
        const uint4 v = *reinterpret_cast<const uint4*>(mine + (m < MT * 16 ? m : 0) * 16);
        const uint8_t s = static_cast<uint8_t>(mine[MT * 256 + (m < MT * 16 ? m : 0)]);
        __builtin_amdgcn_raw_buffer_store_b128(u32x4_t{v.x, v.y, v.z, v.w}, rc,
                                               in ? static_cast<uint32_t>(row) * (p.N / 2) + n0 / 2 : kOOB, 0, 0);
        __builtin_amdgcn_raw_buffer_store_b8(s, rs, in ? static_cast<uint32_t>(row) * out_pitch + n0 / 32 : kOOB, 0, 0);
      }
    } else {
      constexpr int W = GLU ? 32 : 64;         // the wave's output columns
      constexpr int kRow = 2 * W + 16;         // staged row: neighbouring rows on other banks
      constexpr int kPieces = W / 8, kPass = 64 / kPieces;
      const auto rc = make_rsrc(p.c + static_cast<int64_t>(t.r0) * p.N, static_cast<uint32_t>(t.rows) * p.N * 2u);
#pragma unroll
      for (int i = 0; i < MT; ++i) {
#pragma unroll
        for (int j = 0; j < W / 16; ++j) {
          float o[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if constexpr (GLU) o[e] = silu_f(acc[i][2 * j][e]) * acc[i][2 * j + 1][e];
            else o[e] = acc[i][j][e];
          }
          *reinterpret_cast<uint2*>(mine + i16 * kRow + (16 * j + 4 * q) * 2) =
              make_uint2(pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]));
        }
#pragma unroll
        for (int h = 0; h < 16 / kPass; ++h) {
          const int r = h * kPass + lane / kPieces, piece = lane % kPieces;
          const uint4 v = *reinterpret_cast<const uint4*>(mine + r * kRow + 16 * piece);
          const int row = 16 * (wm + WM * i) + r, n = n0 + 8 * piece;
          const bool in = row < t.rows && n < p.N;
          __builtin_amdgcn_raw_buffer_store_b128(u32x4_t{v.x, v.y, v.z, v.w}, rc,
                                                 in ? (static_cast<uint32_t>(row) * p.N + n) * 2u : kOOB, 0, 0);
        }
      }
    }
  };

  fetch_rows(0);
  seek();
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) issue(s);
  int at = 0, since = STAGES;  // the ring's stage, steps since an epilogue
  for (int j = 0; j < ntiles; ++j) {
    const Mx4Tile t = find(j);
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int n = 0; n < NT; ++n) acc[i][n] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    for (int k = 0; k < nk; ++k) {
      // This stage has landed once what is younger alone is outstanding: the DMA of STAGES - 2 stages, and
      // an epilogue's stores in the STAGES - 1 steps behind it.
      if (since < STAGES - 1) {
        wait_vmcnt<(STAGES - 2) * LPW + kStores>();
      } else {
        wait_vmcnt<(STAGES - 2) * LPW>();
      }
      wait_lgkmcnt0();               // this wave's reads of the stage before are done
      __builtin_amdgcn_s_barrier();  // every wave's share landed, and all have left the stage the DMA turns to
      asm volatile("" ::: "memory");
      issue(at ? at - 1 : STAGES - 1);
      __builtin_amdgcn_s_setprio(1);
      multiply(ring + at * kStage, k, t.rows);
      __builtin_amdgcn_s_setprio(0);
      ++since;
      if (k + 1 < nk) at = at + 1 == STAGES ? 0 : at + 1;
    }
    asm volatile("" ::: "memory");
    wait_lgkmcnt0();
    __builtin_amdgcn_s_barrier();  // all have read the stage that the epilogue writes through
    asm volatile("" ::: "memory");
    store(ring + at * kStage, t);
    since = 0;
    at = at + 1 == STAGES ? 0 : at + 1;
    wait_lgkmcnt0();  // the staging is read before the next barrier lets the DMA into it
  }
  wait_vmcnt<0>();  // the trailing DMA (out of range: zeros) before the LDS is released
}

template <int BM, int STAGES>
int launch(const Mx4Gemm& p, int epi, hipStream_t stream, const char* name) {
  const int cols = epi == MX4_PLAIN ? kTileN : kTileN / 2;
  const int n_tiles = (p.N + cols - 1) / cols;
  const int64_t most = mx4_most_tiles(p.rows, p.G, BM) * n_tiles;
  MOE_REQUIRE(most < (1ll << 30), MOE_ERR_UNSUPPORTED, "%s: too many tiles", name);
  const int64_t cus = device_cus(current_device()) / kXcds * kXcds;
  const int64_t want = (most + kXcds - 1) / kXcds * kXcds;
  const dim3 grid(static_cast<unsigned>(want < cus ? want : cus)), block(kTileThreads);
  if (epi == MX4_PLAIN)
    hipLaunchKernelGGL((mx4_tile_kernel<BM, STAGES, MX4_PLAIN>), grid, block, 0, stream, p, n_tiles);
  else if (epi == MX4_SWIGLU)
    hipLaunchKernelGGL((mx4_tile_kernel<BM, STAGES, MX4_SWIGLU>), grid, block, 0, stream, p, n_tiles);
  else
    hipLaunchKernelGGL((mx4_tile_kernel<BM, STAGES, MX4_SWIGLU_MX4>), grid, block, 0, stream, p, n_tiles);
  return launch_status(name);
}

}  // namespace

int mx4_tile(const Mx4Gemm& p, int epi, int bm, hipStream_t stream, const char* name) {
  return bm <= 64 ? launch<64, 3>(p, epi, stream, name)
                  : bm <= 128 ? launch<128, 3>(p, epi, stream, name) : launch<256, 2>(p, epi, stream, name);
}

}  // namespace moe
