// Grouped products of mx4 operands for groups of many rows: LDS tiles of up to
// BM rows by 256 weight rows (128 act columns with swiglu, gate and up), 256
// values deep, so a row of a stage is one 128-byte line.
//
// Eight waves, two by rows and four by columns; wave row wm owns the 16-row
// tiles wm, wm + 2, ... (a partly filled tile then loads both), wave column wn
// the 64 weight rows 64 wn ...  Products are v_mfma_scale_f32_16x16x128 on
// codes and scales as they are stored: lane l multiplies the 32-blocks 2 (l /
// 16) and + 1 of a stage's row, so its two codes chunks are neighbours and its
// two scales one 16-bit read.  The scales come 16 bytes (two stages) of a row
// at a time into a ring of their own: fetched stage by stage they were as many
// L2 requests as the codes' whole lines.  The wave's 64 weight rows are dealt to
// its four fragments four rows at a time, so that a lane's results are twice 8
// (with swiglu once) neighbouring output columns of one row, stored as they are.
//
// Blocks are persistent, one per CU, and run one stream of stages over their
// tiles: a DMA cursor (buffer_load ... lds, fired between the products) fills a
// ring of STAGES stages STAGES - 1 ahead of the compute cursor and runs on
// across tiles, so that a tile's first stage is on its way while the last one's
// output is written.  The epilogue issues the same number of stores whatever is
// in range (out of range ones are dropped by the buffer resource), so that the
// waits that follow can leave them in flight.
//
// Measured at 1024 rows of each of 128 groups: gate and up, 2048 x 768, 308 us
// (825 GFLOP, 2.7 PFLOP/s), down with bf16 rows 235 (537 MB written).  Parts
// switched off: LDS reads alone 79 us of gate and up's, with the products 193
// (bare products 142 at the power limit), with the DMA 250; the rest is the
// epilogue, which nothing covers: one tile's results fill the registers, and
// two blocks of half the rows per CU lost as much to the L1's bytes (344).
// Where weights stream once (384 rows) it is HBM: 41 us for 204 MB.
#include "dma.h"
#include "mx4.h"

namespace moe {
namespace {

constexpr int kTileWaves = 8, kTileThreads = kTileWaves * kWave;
constexpr int kTileN = 256;     // weight rows per tile
constexpr int kXcds = 8;

// f(first group, rows below it in its 64, lo, cnt) for every 64 groups, a group per lane.
template <class F>
__device__ __forceinline__ void each_groups(const Mx4Gemm& p, F&& f) {
  for (int c0 = 0; c0 < p.G; c0 += kWave) {
    int lo;
    const int cnt = mx4_group_rows(p, c0 + (threadIdx.x & (kWave - 1)), lo);
    f(c0, lo, cnt);
  }
}

template <int BM, int STAGES, int EPI>
__global__ __launch_bounds__(kTileThreads) void mx4_tile_kernel(const Mx4Gemm p, int n_tiles) {
  constexpr bool GLU = mx4_glu(EPI);
  constexpr int WM = 2, MT = BM / 16 / WM, NT = 4;
  constexpr int kCols = GLU ? kTileN / 2 : kTileN;     // output columns per tile
  constexpr int LA = BM / 64, LB = kTileN / 64;        // code DMAs per wave and stage (8 rows each)
  constexpr int LPW = LA + LB;
  constexpr int kB = BM * 128, kStage = kB + kTileN * 128;
  constexpr int kScaleWaves = (BM + kTileN) / 64;      // waves that fetch scales, 64 rows each: A's, then B's
  constexpr int kScales = kScaleWaves * 1024, kBs = BM * 16;
  // Scale slots: a fetch serves two stages, so where a tile has an even number of them two slots do for a DMA cursor
  // two stages ahead; otherwise one per stage.
  constexpr int kSlots = STAGES * (kStage + kScales) <= 160 * 1024 ? STAGES : 2;
  constexpr int kStores = EPI == MX4_SWIGLU ? MT : EPI == MX4_PLAIN_F32 ? 4 * MT : 2 * MT;  // store instructions per wave and tile
  // Groups of products between which the next stage's DMA is fired: a ring of two needs it early.
  constexpr int kFire = STAGES == 2 ? MT : 2 * MT;
  static_assert(kScaleWaves <= kTileWaves && STAGES <= 3 && STAGES * kStage + kSlots * kScales <= 160 * 1024, "LDS");
  static_assert((STAGES - 2) * LPW + kStores < 64, "vmcnt range");
  __shared__ __attribute__((aligned(1024))) char ring[STAGES * kStage + kSlots * kScales];  // the stages, then their scales

  const int lane = threadIdx.x & (kWave - 1), i16 = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave & 1, wn = wave >> 1;
  const int64_t wide = GLU ? 2 * static_cast<int64_t>(p.N) : p.N;
  const uint32_t half_k = static_cast<uint32_t>(p.K) / 2, pitch = static_cast<uint32_t>(mx4_pitch(p.K));
  const int blocks = p.K / 32, deep = (p.K + 255) / 256;
  const int nk = kSlots < STAGES ? (deep + 1) / 2 * 2 : deep;  // stages per tile (the last may lie past K)

  int total = 0;
  each_groups(p, [&](int, int, int cnt) {
    total += __builtin_amdgcn_readlane(wave_inclusive_scan((cnt + BM - 1) / BM), kWave - 1);
  });
  total = __builtin_amdgcn_readfirstlane(total) * n_tiles;
  // This block's tiles: every nbx-th of its XCD's contiguous share.
  const int nbx = gridDim.x / kXcds, xcd = blockIdx.x % kXcds, xidx = blockIdx.x / kXcds;
  const int share = (total + kXcds - 1) / kXcds, first = xcd * share + xidx;
  const int span = min(share, total - xcd * share);
  const int ntiles = span > xidx ? (span - xidx + nbx - 1) / nbx : 0;
  if (ntiles <= 0) return;  // the whole block

  // Lane l holds the block's tile seen + l, so that a tile costs four lane
  // reads; the lanes move on when a cursor passes them.
  Mx4Tile held{0, 0, 0, 0};
  int seen = 0;
  auto hold = [&](int j0) __attribute__((always_inline)) {
    seen = j0;
    held = Mx4Tile{0, 0, 0, 0};
    const int tile = first + (j0 + lane) * nbx;
    const bool live = j0 + lane < ntiles;
    int base = 0;
    each_groups(p, [&](int c0, int lo, int cnt) {
      const int n = n_tiles * ((cnt + BM - 1) / BM);
      const int incl = wave_inclusive_scan(n);
      const int tot = __builtin_amdgcn_readlane(incl, kWave - 1);
      const int local = tile - base;
      int w = 0;  // the first lane whose sum passes `local`
#pragma unroll
      for (int step = kWave / 2; step >= 1; step >>= 1)
        if (__shfl(incl, w + step - 1) <= local) w += step;
      const int rows = __shfl(cnt, w), start = __shfl(lo, w), before = __shfl(incl - n, w);
      if (live && local >= 0 && local < tot) {
        const int parts = (rows + BM - 1) / BM, per = ((rows + parts - 1) / parts + 15) & ~15;
        const int nt = (local - before) / parts, part = local - before - nt * parts;
        held = Mx4Tile{c0 + w, start + part * per, min(per, rows - part * per), nt};
      }
      base += tot;
    });
  };
  auto find = [&](int j) __attribute__((always_inline)) {  // tile j of the block's, seen <= j < seen + 64
    const int l = j - seen;
    return Mx4Tile{__builtin_amdgcn_readlane(held.g, l), __builtin_amdgcn_readlane(held.r0, l),
                   __builtin_amdgcn_readlane(held.rows, l), __builtin_amdgcn_readlane(held.n, l)};
  };

  // ------------------------------------------------------------ DMA cursor
  // Code DMA j of a wave fills rows 8 (wave L + j) .. + 7 of an operand, lane l
  // the 16-byte slot l % 8 of row l / 8; chunk 2 q + s of row r is at slot
  // (4 s + q) ^ key(r).  A pass of ds_read_b128 takes rows 0-3 and 12-15 of one
  // lane quarter with rows 4-11 of the next: with chunk numbers that differ by
  // one between quarters and the eight keys of a fragment's row pairs (a_key of
  // neighbouring rows, b_key of rows 16 a + 4 j + b) its lanes lie on distinct
  // banks.
  // Every second stage, wave w's scale DMA takes 16 bytes of each of 64 rows: of
  // A rows 64 w + lane, or behind them of B the rows of wave column w - BM / 64,
  // fragment by fragment (position 16 j + 4 a + b: row 16 a + 4 j + b).
  const uint32_t lds0 = lds_address(ring);
  const u32x4_t ra = rsrc_words(p.a, static_cast<uint32_t>(p.a_rows) * half_k);
  const u32x4_t ras = rsrc_words(p.a_scales, static_cast<uint32_t>(p.a_rows) * pitch);
  u32x4_t rb = ra, rs = ra;
  uint32_t a_off[LA], b_off[LB], s_off;  // at stage 0; kOOB for rows past the end
  int next_row[LA + 1], next_rows = 0;  // of the tile behind the cursor's: its entries of row_index, its rows
  const int l8 = lane >> 3, slot = lane & 7;
  auto a_key = [](int r) { return (r >> 1) & 7; };
  auto b_key = [](int r) { return ((r >> 1) & 1) | ((r >> 4) & 3) << 1; };
  auto chunk_at = [&](int key) { return ((slot ^ key) & 3) << 1 | (slot ^ key) >> 2; };
  auto a_chunk = [&](int j) { return chunk_at(a_key(8 * (wave * LA + j) + l8)); };
  auto b_chunk = [&](int j) { return chunk_at(b_key(8 * (wave * LB + j) + l8)); };
  auto tile_row = [&](int j) { return j < LA ? 8 * (wave * LA + j) + l8 : 64 * wave + lane; };
  int cj = 0, dj = -1, dk = nk;  // the compute cursor's tile; the DMA cursor's tile and stage
  auto fetch_rows = [&](int j) __attribute__((always_inline)) {
    if (j - seen >= kWave) hold(cj);  // (the DMA cursor is a few tiles ahead at most)
    const Mx4Tile t = find(j);        // past the last tile: no rows
    next_rows = t.rows;
#pragma unroll
    for (int n = 0; n <= LA; ++n) next_row[n] = min(t.r0 + tile_row(n), p.rows - 1);
    if (p.row_index) {
#pragma unroll
      for (int n = 0; n <= LA; ++n) next_row[n] = p.row_index[next_row[n]];
    }
  };
  auto seek = [&]() __attribute__((always_inline)) {  // to the next tile's first stage
    ++dj;
    dk = 0;
    const bool live = dj < ntiles;
    const Mx4Tile t = find(dj);
    auto source = [&](int n, uint32_t row_bytes, uint32_t off) {
      const int r = p.row_index ? mx4_source_row(p, next_row[n]) : next_row[n];
      return tile_row(n) < next_rows && r >= 0 && r < p.a_rows ? static_cast<uint32_t>(r) * row_bytes + off : kOOB;
    };
#pragma unroll
    for (int j = 0; j < LA; ++j) a_off[j] = source(j, half_k, 16u * a_chunk(j));
    auto weight = [&](int r, uint32_t row_bytes, uint32_t off) {  // row r of the tile's: fragment (r / 4) % 4
      const int j = (r >> 2) & 3;
      const int n = t.n * kCols + (GLU ? (r >> 6) * 32 + ((r >> 4) & 3) * 8 + (j >> 1) * 4 + (r & 3)
                                      : (r & ~63) + (j >> 1) * 32 + ((r >> 4) & 3) * 8 + (j & 1) * 4 + (r & 3));
      const int w = GLU && (j & 1) ? p.N + n : n;
      return live && n < p.N ? static_cast<uint32_t>(w) * row_bytes + off : kOOB;
    };
#pragma unroll
    for (int j = 0; j < LB; ++j) b_off[j] = weight(8 * (wave * LB + j) + l8, half_k, 16u * b_chunk(j));
    rb = rsrc_words(p.w + t.g * wide * half_k, static_cast<uint32_t>(wide) * half_k);
    if (wave < BM / 64) {
      s_off = source(LA, pitch, 0);
      rs = ras;
    } else {
      s_off = weight(64 * (wave - BM / 64) + ((lane >> 2) & 3) * 16 + (lane >> 4) * 4 + (lane & 3), pitch, 0);
      rs = rsrc_words(p.w_scales + t.g * wide * pitch, static_cast<uint32_t>(wide) * pitch);
    }
    fetch_rows(dj + 1);
  };
  // DMA n of the cursor's stage into the ring stage at `at` (an offset out of range stays so).
  auto fire = [&](int n, uint32_t at) __attribute__((always_inline)) {
    const bool whole = 8 * dk + 8 <= blocks;
    auto off = [&](uint32_t o, int chunk) { return whole || 8 * dk + chunk < blocks ? o + 128u * dk : kOOB; };
    auto to = [&](int b) { return __builtin_amdgcn_readfirstlane(at + b); };
    if (n < LB) {
      dma16(rb, off(b_off[n], b_chunk(n)), to(kB + 1024 * (wave * LB + n)));
    } else {
      dma16(ra, off(a_off[n - LB], a_chunk(n - LB)), to(1024 * (wave * LA + n - LB)));
    }
  };
  int scales_to = 0, scales_at = 0;  // the scale ring's slots of the DMA and of the compute cursor
  auto fire_scales = [&]() __attribute__((always_inline)) {  // with the first of two stages
    if (dk & 1) return;
    if (wave < kScaleWaves)
      dma16(rs, s_off + 8u * dk, __builtin_amdgcn_readfirstlane(lds0 + STAGES * kStage + scales_to * kScales + 1024 * wave));
    scales_to = scales_to + 1 == kSlots ? 0 : scales_to + 1;
  };
  auto advance = [&]() __attribute__((always_inline)) {
    if (++dk == nk) seek();
  };

  // -------------------------------------------------------- compute cursor
  const int swz = i16 >> 1;  // a_key and b_key of the lane's fragment rows
  const int a_lane = i16 * 128, b_row = 64 * wn + 16 * (i16 >> 2) + (i16 & 3);  // fragment j: rows b_row + 4 j
  f32x4_t acc[MT][NT];
  // acc += the stage at `st`, firing the DMA into the one at `to` on the way.
  auto multiply = [&](const char* st, int k, int rows, uint32_t to) __attribute__((always_inline)) {
    const char* sc = ring + STAGES * kStage + scales_at * kScales + (k & 1) * 8 + 2 * q;
    const int left = blocks - (8 * k + 2 * q);  // the lane's blocks inside K (scale padding may hold anything)
    const uint32_t keep = left > 1 ? 0xffffu : left > 0 ? 0xffu : 0u;
    uint32_t sw[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) 
      sw[j] = *reinterpret_cast<const uint16_t*>(sc + kBs + (64 * wn + 16 * j + i16) * 16) & keep;
    // The products of a stage's first 32-blocks go over all row tiles before those of the second: half of B's
    // fragments are read while the first half multiplies, and each tile's next fragment a tile ahead.  Tiles
    // without rows skip their products.
    uint4 w[2][NT], a[2];
    uint32_t sa[MT];
    auto read_b = [&](int s, int j) __attribute__((always_inline)) {
      w[s][j] = *reinterpret_cast<const uint4*>(st + kB + (b_row + 4 * j) * 128 + (((4 * s + q) ^ swz) << 4));
    };
    auto read_a = [&](int n) __attribute__((always_inline)) {
      const int s = n / MT, r = 16 * (wm + WM * (n % MT));
      if (s == 0) sa[n] = *reinterpret_cast<const uint16_t*>(sc + (r + i16) * 16) & keep;
      a[n & 1] = *reinterpret_cast<const uint4*>(st + r * 128 + a_lane + (((4 * s + q) ^ swz) << 4));
    };
#pragma unroll
    for (int j = 0; j < NT; ++j) read_b(0, j);
    read_a(0);
#pragma unroll
    for (int n = 0; n < 2 * MT; ++n) {
      const int s = n / MT, i = n % MT;
      if (n + 1 < 2 * MT) read_a(n + 1);
#pragma unroll
      for (int j = 0; j < NT; ++j)
        if (s == 0 && j * MT / NT == i) read_b(1, j);
      if (16 * (wm + WM * i) < rows) {  // wave-uniform
#pragma unroll
        for (int j = 0; j < NT; ++j)
          acc[i][j] = s == 0 ? mx4_mfma<0>(w[0][j], a[n & 1], acc[i][j], sw[j], sa[i])
                             : mx4_mfma<1>(w[1][j], a[n & 1], acc[i][j], sw[j], sa[i]);
      }
      if (n == 0) fire_scales();
#pragma unroll
      for (int f = n * LPW / kFire; n < kFire && f < (n + 1) * LPW / kFire; ++f) fire(f, to);
    }
    advance();
    if ((k & 1) || k + 1 == nk) scales_at = scales_at + 1 == kSlots ? 0 : scales_at + 1;
  };
  // The tile's results: lane l holds row 16 (wm + 2 i) + l % 16, and of the wave's columns 32 (j / 2) + 8 q + 4 (j %
  // 2) .. + 3 in acc[i][j], or gate and up of act columns 8 q + 4 h .. + 3 in acc[i][2 h] and [2 h + 1].
  auto store = [&](const Mx4Tile& t) __attribute__((always_inline)) {
    // An offset past the compiler's sight, so that it does not branch on its choice and split the store: the waits
    // count one store instruction for each below.
    auto at = [](bool in, uint32_t off) __attribute__((always_inline)) {
      uint32_t v = in ? off : kOOB;
      asm("" : "+v"(v));
      return v;
    };
    auto put16 = [](__amdgpu_buffer_rsrc_t rs, uint32_t off, const float (&o)[8]) {
      __builtin_amdgcn_raw_buffer_store_b128(u32x4_t{pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]),
                                                     pack_bf16x2(o[4], o[5]), pack_bf16x2(o[6], o[7])}, rs, off, 0, 0);
    };
    const uint32_t N = p.N;
    const uint32_t n0 = t.n * kCols + wn * (kCols / 4);  // the wave's first output column
    const auto rc = EPI == MX4_PLAIN_F32
                        ? make_rsrc(p.c32 + static_cast<int64_t>(t.r0) * N, static_cast<uint32_t>(t.rows) * N * 4u)
                        : make_rsrc(p.c + static_cast<int64_t>(t.r0) * N, static_cast<uint32_t>(t.rows) * N * 2u);
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const uint32_t row = 16 * (wm + WM * i) + i16;
      const bool in = static_cast<int>(row) < t.rows;
      if constexpr (EPI == MX4_PLAIN_F32) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const uint32_t n = n0 + 32 * (j / 2) + 8 * q + 4 * (j % 2);
          __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, acc[i][j]), rc,
                                                 at(in && n < N, (row * N + n) * 4u), 0, 0);
        }
      } else if constexpr (EPI == MX4_PLAIN) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t n = n0 + 32 * h + 8 * q;
          float o[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) o[e] = acc[i][2 * h + e / 4][e % 4];
          put16(rc, at(in && n < N, (row * N + n) * 2u), o);
        }
      } else {
        float act[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) act[e] = mx4_act(acc[i][2 * (e / 4)][e % 4], acc[i][2 * (e / 4) + 1][e % 4]);
        if constexpr (EPI == MX4_SWIGLU) {
          const uint32_t n = n0 + 8 * q;
          put16(rc, at(in && n < N, (row * N + n) * 2u), act);
        } else {  // quantised from fp32: one rounding, to 4 bits
          const uint32_t out_pitch = static_cast<uint32_t>(mx4_pitch(N));
          const auto rcc = make_rsrc(p.c_codes + static_cast<int64_t>(t.r0) * (N / 2), static_cast<uint32_t>(t.rows) * (N / 2));
          const auto rcs = make_rsrc(p.c_scales + static_cast<int64_t>(t.r0) * out_pitch,
                                     static_cast<uint32_t>(t.rows) * out_pitch);
          uint32_t top = 0;
#pragma unroll
          for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(act[e]) & 0x7fffffffu);
          top = quarters_max(top);
          const uint32_t s = mx4_scale(top);
          const float f = mx4_scale_f(s);
          uint32_t c = 0;
          c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, act[0], act[1], f, 0);
          c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, act[2], act[3], f, 1);
          c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, act[4], act[5], f, 2);
          c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, act[6], act[7], f, 3);
          const bool w = in && n0 < N;
          __builtin_amdgcn_raw_buffer_store_b32(s == 255u ? 0u : c, rcc, at(w, row * (N / 2) + n0 / 2 + 4 * q), 0, 0);
          __builtin_amdgcn_raw_buffer_store_b8(static_cast<uint8_t>(s), rcs, at(w && q == 0, row * out_pitch + n0 / 32), 0, 0);
        }
      }
    }
  };

  hold(0);
  fetch_rows(0);
  seek();
  for (int s = 0; s < STAGES - 1; ++s) {
    fire_scales();
#pragma unroll
    for (int n = 0; n < LPW; ++n) fire(n, lds0 + s * kStage);
    advance();
  }
  int at = 0, since = STAGES;  // the ring's stage, steps since an epilogue
  for (; cj < ntiles; ++cj) {
    const Mx4Tile t = find(cj);
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
      multiply(ring + at * kStage, k, k < deep ? t.rows : 0, lds0 + (at ? at - 1 : STAGES - 1) * kStage);
      ++since;
      at = at + 1 == STAGES ? 0 : at + 1;
    }
    store(t);
    since = 0;
  }
  wait_vmcnt<0>();  // the trailing DMA (out of range: zeros) before the LDS is released
}

template <int BM, int STAGES>
int launch(const Mx4Gemm& p, int epi, hipStream_t stream, const char* name) {
  static_assert(kTileN == 256, "mx4_tile_columns");
  const int n_tiles = static_cast<int>(mx4_tile_columns(p.N, epi));
  const int64_t most = mx4_most_tiles(p.rows, p.G, BM) * n_tiles;
  MOE_REQUIRE(most < (1ll << 30), MOE_ERR_UNSUPPORTED, "%s: too many tiles", name);
  const int64_t cus = device_cus(current_device()) / kXcds * kXcds;
  const int64_t want = (most + kXcds - 1) / kXcds * kXcds;
  const dim3 grid(static_cast<unsigned>(want < cus ? want : cus)), block(kTileThreads);
  if (epi == MX4_PLAIN)
    hipLaunchKernelGGL((mx4_tile_kernel<BM, STAGES, MX4_PLAIN>), grid, block, 0, stream, p, n_tiles);
  else if (epi == MX4_PLAIN_F32)
    hipLaunchKernelGGL((mx4_tile_kernel<BM, STAGES, MX4_PLAIN_F32>), grid, block, 0, stream, p, n_tiles);
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
