// 8-bit integer products on CDNA4 matrix cores (gfx950): the grouped gate/up and
// down products of int8 experts and a Linear's dense product.
//
// v_mfma_i32_16x16x64_i8 takes 16 consecutive codes of a row per lane where
// v_mfma_f32_16x16x32_bf16 takes 8 bf16 values: the same 16 bytes, in the same
// time, for twice the products. A row of kp codes is therefore staged, swizzled
// and read like a bf16 row of kp / 2 values (mfma_tile.h), a K step is 128 codes,
// and the tiles, the walk and the waves' roles are those of moe_gemm_mfma.hip;
// only the sums (32-bit integers, exact in any order) and the epilogue differ:
//   sum * (scale of the row * scale of the column) (+ bias), or
//   silu(g) u of two such products,
// rounded once to the output's type. Sums being exact, every tile, split and order
// gives the same bits.
#include <algorithm>
#include <cmath>

#include "mfma_pick.h"
#include "mfma_tile.h"
#include "moe_int8.h"
#include "wave_lanes.h"

#include <type_traits>

// Set to 1 by moe_gemm_int8_ragged.hip, which builds these kernels a second time
// for rows that are no whole number of 128-byte steps, or outputs whose rows are no
// whole number of 16-byte stores.
#ifndef ASTRAI_MOE_RAGGED_K
#define ASTRAI_MOE_RAGGED_K 0
#endif

namespace astrai_moe {
namespace {

constexpr bool kRagged = ASTRAI_MOE_RAGGED_K != 0;

typedef int i32x4_t __attribute__((ext_vector_type(4)));

// The row tiles of a launch: those of the list, or one expert's n_rows rows.
struct RowTiles {
  const int32_t* tiles;
  int n_rows, block_m;
  __device__ int live(int capacity) const {
    return tiles == nullptr ? capacity : min(load_scalar(tiles), min(load_scalar(tiles + 2), capacity));
  }
  __device__ int height() const { return tiles == nullptr ? block_m : load_scalar(tiles + 1); }
  __device__ void get(int mt, int& e, int& row0, int& end) const {
    if (tiles == nullptr) {
      e = 0;
      row0 = mt * block_m;
      end = n_rows;
    } else {
      const int32_t* ti = tiles + ASTRAI_MOE_TILE_HEADER + (int64_t)uniform(mt) * ASTRAI_MOE_TILE_STRIDE;
      e = load_scalar(ti);
      row0 = load_scalar(ti + 1);
      end = load_scalar(ti + 2);
    }
  }
};

struct Args {
  const int8_t* a;
  const float* a_scale;
  const int32_t* row_src;
  RowTiles tiles;
  const int8_t *w0, *w1;
  const float *s0, *s1;
  const void* bias;
  const void* x;  // rows to quantise in the kernel, and their columns
  int64_t k;
  int kp, n, n_tiles_n, capacity;
  void* c;
  float* part;     // partial sums of a split last round, or null
  int32_t* sched;  // run-time claims (their counter cleared by the quantiser before), or null
};

// Per-tile global bases (bytes).
template <int BM, int BN, bool kGateUp, bool kGather>
struct I8Src {
  const char* a_base = nullptr;
  const char* b_base0 = nullptr;
  const char* b_base1 = nullptr;
  int e = 0, row0 = 0, rows = 0, b_rows = 0;
  __device__ void setup(const Args& p, int mt, int nt, int row_off = 0) {
    int end;
    p.tiles.get(mt, e, row0, end);
    row0 += row_off;
    rows = min(BM, end - row0);
    constexpr int kTileRows = kGateUp ? BN / 2 : BN;
    b_rows = min(kTileRows, p.n - nt * kTileRows);
    a_base = reinterpret_cast<const char*>(kGather ? p.a : p.a + (int64_t)row0 * p.kp);
    const int64_t at = ((int64_t)e * p.n + (int64_t)nt * kTileRows) * p.kp;
    b_base0 = reinterpret_cast<const char*>(p.w0 + at);
    b_base1 = kGateUp ? reinterpret_cast<const char*>(p.w1 + at) : b_base0;
  }
  template <bool kTail>
  __device__ void dma_a_rows(const DmaLane& dl, uint32_t row_off, int q, uint32_t kp, char* lds) const {
    if constexpr (kTail)
      dma_16_or_zero(a_base, row_off + dl.chunk(q), dl.chunk(q), kp, lds);
    else
      lds_dma_16(a_base + (row_off + dl.chunk(q)), lds);
  }
  template <bool kTail>
  __device__ void dma_b(const DmaLane& dl, int q, uint32_t kp, char* lds) const {
    const int r0 = q * 8;
    const char* bb = (kGateUp && r0 >= BN / 2) ? b_base1 : b_base0;
    const int rq = (kGateUp && r0 >= BN / 2) ? r0 - BN / 2 : r0;
    const uint32_t off = (uint32_t)min(rq + dl.row, b_rows - 1) * kp + dl.chunk(q);
    if constexpr (kTail)
      dma_16_or_zero(bb, off, dl.chunk(q), kp, lds);
    else
      lds_dma_16(bb + off, lds);
  }
};

// Byte offsets of the activation rows one lane loads in its NQ DMA ops of a tile
// (pad rows re-read the tile's last row), gathered through row_src or not. Gathered
// rows lie anywhere in a (under 4 GiB), others behind the tile's first.
template <int NQ, bool kGather>
struct RowOffsets {
  uint32_t off[NQ];
  __device__ void load(const int32_t* row_src, int row0, int rows, int qbase, int lane, uint32_t kp) {
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      const int r = min((qbase + i) * 8 + (lane >> 3), rows - 1);
      off[i] = (kGather ? (uint32_t)row_src[row0 + r] : (uint32_t)r) * kp;
    }
  }
};

// The scales of four columns of expert e from column n on; columns past the
// matrix get 0.
__device__ __forceinline__ f32x4_t four(const float* s, int64_t e, int n, int n_all) {
  typedef float f32x4_u __attribute__((ext_vector_type(4), aligned(4)));  // (scales start anywhere)
  const float* const at = s + e * n_all + n;
  if (!kRagged) return n < n_all ? (f32x4_t)*reinterpret_cast<const f32x4_u*>(at) : f32x4_t{0, 0, 0, 0};
  f32x4_t v;
#pragma unroll
  for (int r = 0; r < 4; ++r) v[r] = n + r < n_all ? at[r] : 0.0f;
  return v;
}

template <typename T>
struct Out4 {
  typedef bf16x4_t type;
};
template <>
struct Out4<float> {
  typedef f32x4_t type;
};

// Four output values of a lane: columns n .. n + 3 of a row.
template <typename T, bool kGateUp>
__device__ __forceinline__ typename Out4<T>::type out_of(const i32x4_t& g, const i32x4_t& u, float sa, const f32x4_t& s0,
                                                         const f32x4_t& s1, const f32x4_t& bias) {
  typename Out4<T>::type o;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    float v;
    if constexpr (kGateUp)
      v = swiglu<T>(g[r], u[r], sa, s0[r], s1[r]);
    else
      v = (float)g[r] * (sa * s0[r]) + bias[r];
    if constexpr (std::is_same_v<T, bf16_t>)
      o[r] = (__bf16)v;
    else
      o[r] = v;
  }
  return o;
}

template <typename T>
__device__ __forceinline__ f32x4_t bias_of(const void* bias, int n, int n_all) {
  f32x4_t v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (n + r < n_all) v[r] = Elem<T>::to_f32(static_cast<const T*>(bias)[n + r]);
  return v;
}

// The epilogue of one wave's WM x WN sums: the accumulator layout gives lane l
// columns 4 (l / 16) .. + 3 of row l % 16 of each 16 x 16 tile. bf16 outputs are
// transposed in pairs of tiles to 16-byte stores; fp32 ones are 16 bytes as they
// lie. Outputs whose rows are no whole number of 16 bytes are stored by element.
template <typename T, bool kGateUp, bool kBias, int WM, int WN, int BN>
__device__ __forceinline__ void store_sums(const i32x4_t (&acc)[WM / 16][WN / 16], const Args& p, int e, int wm, int wn,
                                           int t_row0, int t_rows, int t_nt) {
  constexpr int MT16 = WM / 16, NT16 = WN / 16, NJ = kGateUp ? NT16 / 2 : NT16;
  static_assert(NJ % 2 == 0, "tiles are stored in pairs");
  const int el = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
  const int row_l = el & 15, q = el >> 4;
  const int n_base = kGateUp ? t_nt * (BN / 2) + wn * (WN / 2) : t_nt * BN + wn * WN;
  const int N = p.n;
  T* const C = static_cast<T*>(p.c);
  const bool whole = !kRagged || ((N * (int)sizeof(T)) % 16 == 0 && reinterpret_cast<uintptr_t>(p.c) % 16 == 0);
#pragma unroll
  for (int jp = 0; jp < NJ; jp += 2) {
    f32x4_t s0[2], s1[2], b[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int n = n_base + (jp + h) * 16 + 4 * q;
      s0[h] = four(p.s0, e, n, N);
      if constexpr (kGateUp) s1[h] = four(p.s1, e, n, N);
      b[h] = kBias ? bias_of<T>(p.bias, n, N) : f32x4_t{0, 0, 0, 0};
    }
#pragma unroll
    for (int i = 0; i < MT16; ++i) {
      const int gm = wm * WM + i * 16 + row_l;
      const int row = t_row0 + min(gm, t_rows - 1);
      const float sa = p.a_scale[row];
      const int64_t row_off = (int64_t)row * N;
      typename Out4<T>::type o[2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
        o[h] = out_of<T, kGateUp>(acc[i][jp + h], acc[i][kGateUp ? jp + h + NJ : jp + h], sa, s0[h], s1[h], b[h]);
      if (whole) {
        if constexpr (std::is_same_v<T, bf16_t>) {
          transpose2(o);
          const int n = n_base + jp * 16 + 8 * q;
          bf16x8_t v;
#pragma unroll
          for (int r = 0; r < 4; ++r) v[r] = o[0][r], v[4 + r] = o[1][r];
          if (gm < t_rows && n < N) *reinterpret_cast<bf16x8_t*>(C + row_off + n) = v;
        } else {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int n = n_base + (jp + h) * 16 + 4 * q;
            if (gm < t_rows && n < N) *reinterpret_cast<f32x4_t*>(C + row_off + n) = o[h];
          }
        }
      } else if (gm < t_rows) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int n = n_base + (jp + h) * 16 + 4 * q;
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (n + r < N) {
              using E = std::conditional_t<std::is_same_v<T, bf16_t>, __bf16, T>;
              reinterpret_cast<E*>(C)[row_off + n + r] = o[h][r];
            }
        }
      }
    }
  }
}

// ===========================================================================
// 32-, 64- and 128-row tiles: every wave issues DMA, several stages in flight. Bound by
// reading the weights where an expert has few rows (64 tokens, 128 experts, top-8, D
// 4096, F 1536: 2.4 GB of codes, the layer 405 us, 5.9 TB/s, as a plain read), by the
// rounds of tiles otherwise (333 tokens, 64 experts, top-6 and a shared one, D 2048, F
// 1408: 77 and 47 us of 157; 32- and 128-row tiles there, or a stage more, took as long).
// ===========================================================================
template <int BM_, int BN_, int STAGES_, int WGM_, int WGN_, int GM_>
struct TileCfg {
  static constexpr int BM = BM_, BN = BN_, STAGES = STAGES_, WGM = WGM_, WGN = WGN_, GM = GM_;
  static constexpr int WAVES = WGM * WGN;
  static constexpr int THREADS = WAVES * 64;
  static constexpr int WM = BM / WGM;  // rows per wave
  static constexpr int WN = BN / WGN;  // columns per wave
  static constexpr int A_BYTES = BM * kRowBytes;
  static constexpr int B_BYTES = BN * kRowBytes;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int A_PER_WAVE = A_BYTES / 1024 / WAVES;  // 1 KB DMA ops per wave
  static constexpr int B_PER_WAVE = B_BYTES / 1024 / WAVES;
  static constexpr int DMA_PER_WAVE = A_PER_WAVE + B_PER_WAVE;
  static_assert(A_BYTES % (1024 * WAVES) == 0 && B_BYTES % (1024 * WAVES) == 0, "DMA ops split over waves");
  static_assert(WM % 16 == 0 && WN % 32 == 0, "16x16 MFMA tiles; gate/up halves");
  static_assert(STAGES >= 2 && STAGES * STAGE_BYTES <= 160 * 1024, "LDS");
  static_assert(DMA_PER_WAVE * (STAGES - 1) <= 63, "vmcnt range");
};

// kHalves: the list holds 256-row tiles, each walked as two of 128 rows.
template <typename Cfg, typename T, bool kGateUp, bool kGather, bool kHalves>
__global__ __launch_bounds__(Cfg::THREADS, 1) void gemm_i8_kernel(const Args p) {
  constexpr int S = Cfg::STAGES;
  constexpr int DPW = Cfg::DMA_PER_WAVE;
  __shared__ __attribute__((aligned(1024))) char smem[S * Cfg::STAGE_BYTES];
  static_assert(!kHalves || Cfg::BM == 128, "halves of 256-row tiles");
  const TileWalk<Cfg::GM> walk(p.tiles.live(p.capacity), kHalves ? 2 * p.n_tiles_n : p.n_tiles_n);
  int mt = 0, nt = 0;
  // the workgroup's first tile from `logical` on that has rows (a tile of at
  // most 128 rows has no second half)
  auto seek = [&](int logical_, int& mt_, int& nt_) {
    int at = walk.seek(logical_, mt_, nt_);
    if constexpr (kHalves) {
      while (at < walk.total && (nt_ & 1) != 0) {
        int e, row0, end;
        p.tiles.get(mt_, e, row0, end);
        if (row0 + 128 < end) break;
        at = walk.seek(at + walk.G, mt_, nt_);
      }
    }
    return at;
  };
  int logical = seek(walk.first_slot(), mt, nt);
  if (logical >= walk.total) return;

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int wm = wave / Cfg::WGN;
  const int wn = wave % Cfg::WGN;
  const uint32_t kp = (uint32_t)p.kp;
  I8Src<Cfg::BM, Cfg::BN, kGateUp, kGather> src;
  RowOffsets<Cfg::A_PER_WAVE, kGather> rows;
  const int KT = (int)((kp + kRowBytes - 1) / kRowBytes);
  // K steps start at step (7 e) mod KT, so that workgroups streaming different
  // experts read their weight rows at different offsets (as in moe_gemm_mfma.hip)
  int k_start = 0;
  auto setup_tile = [&](int mt_, int nt_) {
    if constexpr (kHalves)
      src.setup(p, mt_, nt_ >> 1, (nt_ & 1) * 128);
    else
      src.setup(p, mt_, nt_);
    k_start = (src.e * 7) % KT;
    rows.load(p.row_src, src.row0, src.rows, wave * Cfg::A_PER_WAVE, lane, kp);
  };
  auto stage_ops = [&](auto tail_c, int ks, int buf) {
    constexpr bool kTail = decltype(tail_c)::value;
    char* sa = smem + buf * Cfg::STAGE_BYTES;
    char* sb = sa + Cfg::A_BYTES;
    const DmaLane dl(lane, ks);
#pragma unroll
    for (int i = 0; i < Cfg::A_PER_WAVE; ++i) {
      const int q = wave * Cfg::A_PER_WAVE + i;
      src.template dma_a_rows<kTail>(dl, rows.off[i], q, kp, sa + q * 1024);
    }
#pragma unroll
    for (int i = 0; i < Cfg::B_PER_WAVE; ++i) {
      const int q = wave * Cfg::B_PER_WAVE + i;
      src.template dma_b<kTail>(dl, q, kp, sb + q * 1024);
    }
  };
  auto issue_stage = [&](int kstep, int buf) {  // the tile's kstep-th step
    const int ks = kstep + k_start < KT ? kstep + k_start : kstep + k_start - KT;  // K step loaded
    if (kRagged && (uint32_t)(ks + 1) * kRowBytes > kp)
      stage_ops(std::true_type{}, ks, buf);
    else
      stage_ops(std::false_type{}, ks, buf);
  };

  // ---- fragment reads (16x16x64: lane l holds row l % 16, codes 16 (l / 16) .. + 15) ----
  constexpr int MT16 = Cfg::WM / 16, NT16 = Cfg::WN / 16;
  const int frag_row = lane & 15;
  const int fq = lane >> 4;
  const int fsw = (frag_row >> 1) & 7;  // row bases are multiples of 16
  int a_off[MT16];
#pragma unroll
  for (int i = 0; i < MT16; ++i) a_off[i] = (wm * Cfg::WM + i * 16 + frag_row) * kRowBytes;
  int b_off[NT16];
#pragma unroll
  for (int j = 0; j < NT16; ++j) {
    int r;
    if (kGateUp) {
      constexpr int half = NT16 / 2;
      r = (j < half) ? wn * (Cfg::WN / 2) + j * 16 : Cfg::BN / 2 + wn * (Cfg::WN / 2) + (j - half) * 16;
    } else {
      r = wn * Cfg::WN + j * 16;
    }
    b_off[j] = (r + frag_row) * kRowBytes;
  }
  i32x4_t fa[2][MT16], fb[2][NT16];
  auto read_frags = [&](int buf, int kh, int slot_) {
    const char* sa = smem + buf * Cfg::STAGE_BYTES;
    const char* sb = sa + Cfg::A_BYTES;
    const int sw = ((kh * 4 + fq) ^ fsw) << 4;
#pragma unroll
    for (int i = 0; i < MT16; ++i) fa[slot_][i] = *reinterpret_cast<const i32x4_t*>(sa + a_off[i] + sw);
#pragma unroll
    for (int j = 0; j < NT16; ++j) fb[slot_][j] = *reinterpret_cast<const i32x4_t*>(sb + b_off[j] + sw);
  };
  i32x4_t acc[MT16][NT16];
  auto mfmas = [&](int slot_) {
#pragma unroll
    for (int i = 0; i < MT16; ++i)
#pragma unroll
      for (int j = 0; j < NT16; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fb[slot_][j], fa[slot_][i], acc[i][j], 0, 0, 0);
  };
  // pair each fragment read of the next half with an MFMA of this one
  auto interleave = [&]() {
#pragma unroll
    for (int q = 0; q < MT16 + NT16; ++q) {
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    }
    if constexpr (MT16 * NT16 > MT16 + NT16)
      __builtin_amdgcn_sched_group_barrier(0x008, MT16 * NT16 - (MT16 + NT16), 0);
  };

  setup_tile(mt, nt);
#pragma unroll
  for (int s = 0; s < S; ++s)
    if (s < KT) issue_stage(s, s);
  wait_groups<DPW, S - 1>(min(S - 1, KT - 1));  // step 0 landed
  lds_barrier();
  while (true) {
#pragma unroll
    for (int i = 0; i < MT16; ++i)
#pragma unroll
      for (int j = 0; j < NT16; ++j) acc[i][j] = i32x4_t{0, 0, 0, 0};
    read_frags(0, 0, 0);
    int buf = 0;
    for (int kt = 0; kt < KT; ++kt) {
      read_frags(buf, 1, 1);
      interleave();
      mfmas(0);
      const int nbuf = (buf + 1 == S) ? 0 : buf + 1;
      if (kt + 1 < KT) {
        wait_groups<DPW, S - 2>(min(S - 2, KT - 2 - kt));
        __builtin_amdgcn_sched_barrier(0);
        lds_barrier();
        __builtin_amdgcn_sched_barrier(0);
        read_frags(nbuf, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
        if (kt + S < KT) issue_stage(kt + S, buf);
        __builtin_amdgcn_sched_barrier(0);
      }
      mfmas(1);
      buf = nbuf;
    }

    // ---- next tile's first stages, then this tile's epilogue ----
    int nmt = 0, nnt = 0;
    const int nlogical = seek(logical + walk.G, nmt, nnt);
    const bool has_next = nlogical < walk.total;
    const int t_e = src.e, t_row0 = src.row0, t_rows = src.rows, t_nt = kHalves ? nt >> 1 : nt;
    __builtin_amdgcn_sched_barrier(0);
    lds_barrier();  // every wave is done reading the stage buffers
    __builtin_amdgcn_sched_barrier(0);
    if (has_next) {
      setup_tile(nmt, nnt);
#pragma unroll
      for (int s = 0; s < S; ++s)
        if (s < KT) issue_stage(s, s);
    }
    if (!kGateUp && p.bias != nullptr)
      store_sums<T, kGateUp, true, Cfg::WM, Cfg::WN, Cfg::BN>(acc, p, t_e, wm, wn, t_row0, t_rows, t_nt);
    else
      store_sums<T, kGateUp, false, Cfg::WM, Cfg::WN, Cfg::BN>(acc, p, t_e, wm, wn, t_row0, t_rows, t_nt);
    if (!has_next) break;
    logical = nlogical;
    mt = nmt;
    nt = nnt;
    wait_vmcnt<0>();  // the next tile's stages (and this wave's stores) are done
    lds_barrier();
  }
}

// ===========================================================================
// Streaming kernel: 256 x 256 tiles, 8 matrix-core waves + 4 DMA waves, as
// gemm_stream_kernel of moe_gemm_mfma.hip, whose comments give the reasons of its
// schedule: two activation and three weight stages, one barrier a K step, the
// matrix-core waves' fragments in rings, the priority drops. 16384 tokens, 8 experts,
// top-2, D 4096, F 14336: gate/up 2.73 to 2.86 ms (2.7 to 2.8 Pop/s), down 1.34 to 1.43
// (2.7 to 2.9); one expert, 8192 rows, 4096 to 14336 364 to 443 us (2.2 to 2.64). A K
// step of a tile takes about 1.46 us, of which the matrix instructions alone, with their
// operands in registers on every compute unit at once, take 1.07 (4.0 Pop/s; those of
// 32 x 32 x 32 3.5); a tile's epilogue and first fragments take about 3 us, of which the
// gate/up product's shorter K has more (matrix cores busy 79%, down 83%).
// ===========================================================================
template <bool kGateUp>
struct StreamCfg {
  static constexpr int BM = 256, BN = 256, GM = kGateUp ? 8 : 16;
  static constexpr int WGM = 2, WGN = 4, MW = 8, DW = 4;  // matrix-core waves (WGM x WGN), DMA waves
  static constexpr int WAVES = MW + DW, THREADS = WAVES * 64;
  static constexpr int WM = BM / WGM, WN = BN / WGN;  // 128 x 64 per matrix-core wave
  static constexpr int A_BYTES = BM * kRowBytes, B_BYTES = BN * kRowBytes;  // 32 KB per K step each
  static constexpr int A_STAGES = 2, B_STAGES = 3;
  static constexpr int A_OFF = 0, B_OFF = A_STAGES * A_BYTES;
  static constexpr int LDS = B_OFF + B_STAGES * B_BYTES;  // 160 KB
  static constexpr int OPS = A_BYTES / 1024 / DW;         // 1 KB DMA ops per DMA wave per operand and step
  static constexpr int RG = 2, AR = 4, PD = 2;
};

// Position of a DMA wave in its workgroup's sequence of K steps.
template <int BM, int BN, int GM, bool kGateUp, bool kGather>
struct StepCursor {
  int idx, mt, nt, kt, k1, unit;
  bool live;
  I8Src<BM, BN, kGateUp, kGather> src;
  __device__ void enter(const SplitWalk<GM>& walk, int logical, const Args& p) {
    walk.item(logical, mt, nt, kt, k1, unit);
    src.setup(p, mt, nt);
  }
  __device__ void start(const SplitWalk<GM>& walk, const ItemSeq& seq, const Args& p) {
    idx = 0, live = true;
    enter(walk, seq.id(0), p);
  }
  // true when the cursor moved on to the next work item
  __device__ bool advance(const SplitWalk<GM>& walk, const ItemSeq& seq, const Args& p) {
    if (++kt < k1) return false;
    const int nxt = seq.id(++idx);
    live = nxt >= 0;
    if (live) enter(walk, nxt, p);
    return live;
  }
};

template <typename T, bool kGateUp, bool kGather, bool kBias>
__global__ __launch_bounds__(StreamCfg<kGateUp>::THREADS, 1) void gemm_i8_stream_kernel(const Args p) {
  using Cfg = StreamCfg<kGateUp>;
  __shared__ __attribute__((aligned(1024))) char smem[Cfg::LDS];
  const uint32_t kp = (uint32_t)p.kp;
  const int KT = (int)((kp + kRowBytes - 1) / kRowBytes);
  const SplitWalk<Cfg::GM> walk(p.tiles.live(p.capacity), p.n_tiles_n, KT, !kGateUp && p.part != nullptr);
  const ItemSeq seq(walk, KT, p.sched);
  if (seq.m == 0) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;

  if (wave >= Cfg::MW) {
    // ---------------- DMA waves ----------------
    const int dw = wave - Cfg::MW;
    StepCursor<Cfg::BM, Cfg::BN, Cfg::GM, kGateUp, kGather> ca;  // next A step
    StepCursor<Cfg::BM, Cfg::BN, Cfg::GM, kGateUp, false> cb;    // next B step
    RowOffsets<Cfg::OPS, kGather> rows;
    auto load_rows = [&]() { rows.load(p.row_src, ca.src.row0, ca.src.rows, dw * Cfg::OPS, lane, kp); };
    ca.start(walk, seq, p);
    cb.start(walk, seq, p);
    load_rows();
    auto tail_step = [&](int kt) { return kRagged && (uint32_t)(kt + 1) * kRowBytes > kp; };
    auto ops_a = [&](auto tail_c, int buf) {
      const DmaLane dl(lane, ca.kt);
      char* base = smem + Cfg::A_OFF + buf * Cfg::A_BYTES;
#pragma unroll
      for (int i = 0; i < Cfg::OPS; ++i) {
        const int q = dw * Cfg::OPS + i;
        ca.src.template dma_a_rows<decltype(tail_c)::value>(dl, rows.off[i], q, kp, base + q * 1024);
      }
    };
    auto issue_a = [&](int buf) {
      if (tail_step(ca.kt))
        ops_a(std::true_type{}, buf);
      else
        ops_a(std::false_type{}, buf);
      if (ca.advance(walk, seq, p)) load_rows();  // the next item's rows
    };
    auto ops_b = [&](auto tail_c, int buf) {
      const DmaLane dl(lane, cb.kt);
      char* base = smem + Cfg::B_OFF + buf * Cfg::B_BYTES;
#pragma unroll
      for (int i = 0; i < Cfg::OPS; ++i) {
        const int q = dw * Cfg::OPS + i;
        cb.src.template dma_b<decltype(tail_c)::value>(dl, q, kp, base + q * 1024);
      }
    };
    auto issue_b = [&](int buf) {
      if (tail_step(cb.kt))
        ops_b(std::true_type{}, buf);
      else
        ops_b(std::false_type{}, buf);
      cb.advance(walk, seq, p);
    };
    // prologue in issue order B0, A0, B1, A1, B2 (as far as the steps exist)
    int a_iss = 0, b_iss = 0;
    issue_b(0), ++b_iss;
    issue_a(0), ++a_iss;
    if (cb.live) issue_b(1), ++b_iss;
    if (ca.live) issue_a(1), ++a_iss;
    if (cb.live) issue_b(2), ++b_iss;
    wait_groups<Cfg::OPS, 3>((a_iss - 1) + (b_iss - 1));  // A0 and B0 landed
    __builtin_amdgcn_s_barrier();                          // X_{-1}
    for (int g = 0;; ++g) {
      // A(g + 1) and B(g + 1) landed; B(g + 2), issued after A(g + 1), may stay in flight
      wait_groups<Cfg::OPS, 1>(b_iss > g + 2 ? 1 : 0);
      __builtin_amdgcn_s_barrier();  // X_g
      const bool more = ca.live;
      if (ca.live) issue_a(g & 1), ++a_iss;  // A(g + 2)
      if (cb.live) issue_b(g % 3), ++b_iss;  // B(g + 3)
      if (!more && g + 1 >= a_iss) break;    // X_g was the last step's barrier
    }
    return;
  }

  // ---------------- matrix-core waves ----------------
  const int wm = wave / Cfg::WGN;
  const int wn = wave % Cfg::WGN;
  constexpr int MT16 = Cfg::WM / 16, NT16 = Cfg::WN / 16;
  constexpr int AR = Cfg::AR, PD = Cfg::PD;
  const int frag_row = lane & 15;
  const int fq = lane >> 4;
  const uint32_t v_lane = frag_row * kRowBytes + ((fq ^ ((frag_row >> 1) & 7)) << 4);
  const uint32_t b_row = kGateUp ? wn * (Cfg::WN / 2) : wn * Cfg::WN;
  uint32_t vA = (uint32_t)Cfg::A_OFF + (uint32_t)(wm * Cfg::WM) * kRowBytes + v_lane;
  uint32_t vB = (uint32_t)Cfg::B_OFF + b_row * kRowBytes + v_lane;
  constexpr uint32_t kBEnd = (uint32_t)Cfg::LDS;
  auto next_b = [&](uint32_t v) -> uint32_t {
    const uint32_t n = v + Cfg::B_BYTES;
    return n >= kBEnd ? n - Cfg::B_STAGES * Cfg::B_BYTES : n;
  };
  auto rotate = [&]() {
    vA ^= (uint32_t)Cfg::A_BYTES;
    vB = next_b(vB);
    asm volatile("" : "+v"(vA), "+v"(vB));
  };
  i32x4_t fa[AR], fb[NT16];
  i32x4_t acc[MT16][NT16];
  auto lds128 = [&](uint32_t addr) -> i32x4_t { return *reinterpret_cast<const i32x4_t*>(smem + addr); };
  auto rdA = [&](uint32_t base, int kh, int i) -> i32x4_t {
    return lds128((base ^ (kh ? 64u : 0u)) + i * 16 * kRowBytes);
  };
  auto rdB = [&](uint32_t base, int kh, int j) -> i32x4_t {
    constexpr int half = NT16 / 2;
    const int r = kGateUp ? ((j < half) ? j * 16 : Cfg::BN / 2 + (j - half) * 16) : j * 16;
    return lds128((base ^ (kh ? 64u : 0u)) + r * kRowBytes);
  };
  // one K step as 16 rows of 16 (two halves x 8 row blocks) in groups of RG
  constexpr int RG = Cfg::RG;
  auto step = [&]() {
    uint32_t nA = 0, nB = 0;
    static_for<16 / RG>([&](auto gg) {
      constexpr int r0 = decltype(gg)::value * RG;
      if constexpr (r0 == 0) __builtin_amdgcn_s_setprio(1);
      if constexpr (kGateUp ? (r0 == 8 || r0 == 12) : r0 == 10) __builtin_amdgcn_s_setprio(0);
      if constexpr (kGateUp ? r0 == 10 : r0 == 12) __builtin_amdgcn_s_setprio(1);
      if constexpr (r0 + PD >= 16 && r0 + PD < 16 + RG) {
        __builtin_amdgcn_sched_barrier(0);
        lds_barrier();  // X_g
        __builtin_amdgcn_sched_barrier(0);
        nA = vA ^ (uint32_t)Cfg::A_BYTES;
        nB = next_b(vB);
      }
      static_for<RG>([&](auto qq) {
        constexpr int rp = r0 + PD + decltype(qq)::value;
        if constexpr (rp < 16)
          fa[rp % AR] = rdA(vA, rp / 8, rp % 8);
        else
          fa[rp % AR] = rdA(nA, 0, rp - 16);
      });
#pragma unroll
      for (int j = 0; j < NT16; ++j) {
        static_for<RG>([&](auto qq) {
          constexpr int r = r0 + decltype(qq)::value;
          acc[r % 8][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fb[j], fa[r % AR], acc[r % 8][j], 0, 0, 0);
        });
        if constexpr (r0 + RG == 8) fb[j] = rdB(vB, 1, j);
        if constexpr (r0 + RG == 16) fb[j] = rdB(nB, 0, j);
      }
    });
  };

  lds_barrier();  // X_{-1}
  int mt = 0, nt = 0, k0 = 0, k1 = 0, unit = -1;
  bool claiming = wave == 0;  // matrix-core wave 0 makes the run-time claims
  // Waves of padding rows only idle where gemm_stream_kernel's do.
  const int idle_row0 = __builtin_amdgcn_readfirstlane(wm * Cfg::WM);
  const int idle_mt0 =
      __builtin_amdgcn_readfirstlane(KT < kIdleMaxSteps || p.tiles.tiles == nullptr ? 0 : load_scalar(p.tiles.tiles + 3));
  walk.item(seq.id(0), mt, nt, k0, k1, unit);
  for (int idx = 0;; ++idx) {
    const int claim_at = (claiming && seq.claims_next(idx)) ? k1 - kClaimLead : -1;
    int e, t_row0, t_end;
    p.tiles.get(mt, e, t_row0, t_end);
    const int t_rows = min(Cfg::BM, t_end - t_row0);
    const bool idle = idle_threshold(mt >= idle_mt0, idle_row0) >= t_rows;
    // The item's first fragments. (The step before has read them already; read again,
    // their registers are the epilogue's in between, which spilled without.)
#pragma unroll
    for (int j = 0; j < NT16; ++j) fb[j] = rdB(vB, 0, j);
#pragma unroll
    for (int r = 0; r < PD; ++r) fa[r % AR] = rdA(vA, 0, r);
    int zero;
    asm("s_mov_b32 %0, 0" : "=s"(zero));
#pragma unroll
    for (int i = 0; i < MT16; ++i)
#pragma unroll
      for (int j = 0; j < NT16; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[i][j][r] = zero;
    if (idle) {
      for (int kt = k0; kt < k1; ++kt) {
        __builtin_amdgcn_sched_barrier(0);
        lds_barrier();  // X_g
        __builtin_amdgcn_sched_barrier(0);
        rotate();
      }
    } else {
      for (int kt = k0, stop = claim_at >= 0 ? claim_at : k1;; stop = k1) {
        for (; kt < stop; ++kt) {
          step();
          rotate();
        }
        if (kt == k1) break;
        claiming = seq.claim(idx, p.sched);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    const int nxt = seq.id(idx + 1);
    if (kGateUp || unit < 0) {
      if (!idle)
        store_sums<T, kGateUp, kBias, Cfg::WM, Cfg::WN, Cfg::BN>(acc, p, e, wm, wn, t_row0, t_rows, nt);
    } else {
      store_partial(reinterpret_cast<const f32x4_t(&)[MT16][NT16]>(acc), p.part, unit, wave, lane);
    }
    if (nxt < 0) break;
    walk.item(nxt, mt, nt, k0, k1, unit);
  }
}

// The epilogue of the split tail tiles (SplitWalk): workgroup (t, w), one wave,
// adds the partial sums of matrix-core wave w of tail tile t.
template <typename T, bool kBias>
__global__ __launch_bounds__(64) void i8_split_reduce_kernel(const Args p, int G) {
  using Cfg = StreamCfg<false>;
  const int KT = (p.kp + kRowBytes - 1) / kRowBytes;
  const SplitWalk<Cfg::GM> walk(p.tiles.live(p.capacity), p.n_tiles_n, KT, true, G);
  const int t = blockIdx.x;
  if (walk.S < 2 || t >= walk.total - walk.full) return;
  int mt = 0, nt = 0;
  walk.decode(walk.full + t, mt, nt);
  int e, t_row0, t_end;
  p.tiles.get(mt, e, t_row0, t_end);
  const int t_rows = min(Cfg::BM, t_end - t_row0);
  const int wave = blockIdx.y, lane = threadIdx.x;
  constexpr int MT16 = Cfg::WM / 16, NT16 = Cfg::WN / 16;
  constexpr int kUnitVecs = kSplitUnitFloats / 4;
  const i32x4_t* at = reinterpret_cast<const i32x4_t*>(p.part) + (int64_t)t * walk.S * kUnitVecs +
                      wave * (MT16 * NT16 * 64) + lane;
  i32x4_t acc[MT16][NT16];
#pragma unroll
  for (int i = 0; i < MT16; ++i)
#pragma unroll
    for (int j = 0; j < NT16; ++j) acc[i][j] = at[(i * NT16 + j) * 64];
  for (int s = 1; s < walk.S; ++s) {
    const i32x4_t* ps = at + (int64_t)s * kUnitVecs;
#pragma unroll
    for (int i = 0; i < MT16; ++i)
#pragma unroll
      for (int j = 0; j < NT16; ++j) acc[i][j] += ps[(i * NT16 + j) * 64];
  }
  store_sums<T, false, kBias, Cfg::WM, Cfg::WN, Cfg::BN>(acc, p, e, wave / Cfg::WGN, wave % Cfg::WGN, t_row0,
                                                         t_rows, nt);
}

using SmallCfg = TileCfg<kMfmaSmallBM, 256, 4, 1, 4, 8>;
using MidCfg = TileCfg<kMfmaMidBM, 256, 3, 2, 4, 8>;
using Mid2Cfg = TileCfg<kMfmaMid2BM, 256, 3, 2, 4, 8>;
using NarrowCfg = TileCfg<kMfmaMid2BM, 128, 4, 4, 2, 8>;
using NarrowMidCfg = TileCfg<kMfmaMidBM, 128, 3, 2, 2, 8>;

#if ASTRAI_MOE_RAGGED_K
// ===========================================================================
// Few rows: as gemm_few_kernel of moe_gemm_few.hip, bound by reading the weights
// once with every compute unit. A column tile is 32 or 16 weight rows; the four waves
// of a workgroup take every fourth K step of it, each through an LDS ring of its own,
// and their sums meet in LDS, 32 rows at a time. (For every shape: whole K steps gain
// nothing here.)
// ===========================================================================
template <int BM_, int BN_>
struct FewCfg {
  static constexpr int BM = BM_, BN = BN_, WAVES = 4, STAGES = BM == 64 ? 3 : BN == 32 ? 4 : 6;
  static constexpr int NR = BM / 16, NC = BN / 16;  // 16-row and 16-column blocks
  static constexpr int A_BYTES = BM * kRowBytes, B_BYTES = BN * kRowBytes, STAGE = A_BYTES + B_BYTES;
  static constexpr int OPS = STAGE / 1024;                     // DMA ops per wave and step
  static constexpr int RED_ROWS = 32;                          // rows whose sums meet at a time
  static constexpr int RED_WAVE = RED_ROWS * BN * 4;           // one wave's sums of these
  static constexpr int RED_OFF = WAVES * STAGES * STAGE;       // 128 or 144 KB of rings
  static constexpr int RED_BUFS = BM == 64 ? 1 : 2;            // places they meet in
  static constexpr int LDS = RED_OFF + RED_BUFS * WAVES * RED_WAVE;  // 160 KB
  static_assert(LDS <= 160 * 1024, "LDS");
  static_assert(OPS * (STAGES - 1) <= 63, "vmcnt range");
};

// Position of a wave in its sequence of K steps: run `sub` of BM rows of tile `unit`,
// the wave's step j of n.
template <typename Cfg, bool kGateUp, bool kGather>
struct FewCursor {
  int unit, mt, nt, e, row0, rows, sub, j, n, rot;
  bool live;
  const char *a, *b0, *b1;
  uint32_t off[Cfg::BM / 8];  // byte offsets of the rows a lane loads of the activation tile
  int b_rows;

  __device__ void enter(const Args& p) {
    constexpr int kCols = kGateUp ? Cfg::BN / 2 : Cfg::BN;
    mt = unit / p.n_tiles_n;
    nt = unit - mt * p.n_tiles_n;
    int end;
    p.tiles.get(mt, e, row0, end);
    e = uniform(e), row0 = uniform(row0);
    rows = min(uniform(p.tiles.height()), uniform(end) - row0);
    b_rows = min(kCols, p.n - nt * kCols);
    const int64_t at = ((int64_t)e * p.n + (int64_t)nt * kCols) * p.kp;
    b0 = reinterpret_cast<const char*>(p.w0 + at);
    b1 = kGateUp ? reinterpret_cast<const char*>(p.w1 + at) : b0;
    rot = n > 0 ? (7 * e + 3 * nt) % n : 0;
    sub = 0;
  }
  __device__ void enter_rows(const Args& p, int lane) {
    j = 0;
    a = reinterpret_cast<const char*>(kGather ? p.a : p.a + (int64_t)(row0 + sub * Cfg::BM) * p.kp);
    const int last = rows - sub * Cfg::BM - 1;  // pad rows re-read the last row
#pragma unroll
    for (int q = 0; q < Cfg::BM / 8; ++q) {
      const int r = min(q * 8 + (lane >> 3), last);
      off[q] = (kGather ? (uint32_t)p.row_src[row0 + sub * Cfg::BM + r] : (uint32_t)r) * (uint32_t)p.kp;
    }
  }
  __device__ void advance(const Args& p, int total, int G, int lane) {
    if (++j < n) return;
    const int old_mt = mt, old_sub = sub;
    if ((sub + 1) * Cfg::BM < rows) {
      ++sub;
    } else {
      unit += G;
      live = unit < total;
      if (!live) return;
      enter(p);
    }
    if (mt == old_mt && sub == old_sub)
      j = 0;
    else
      enter_rows(p, lane);
  }
  // the wave's next step into LDS at `lds`
  __device__ void issue(const Args& p, int wave, int lane, char* lds) const {
    int jr = j + rot;
    if (jr >= n) jr -= n;
    const int ks = wave + Cfg::WAVES * jr;
    const uint32_t kp = (uint32_t)p.kp;
    const DmaLane dl(lane, ks);
    const bool tail = (uint32_t)(ks + 1) * kRowBytes > kp;
#pragma unroll
    for (int q = 0; q < Cfg::BM / 8; ++q) {
      if (tail)
        dma_16_or_zero(a, off[q] + dl.chunk(q), dl.chunk(q), kp, lds + q * 1024);
      else
        lds_dma_16(a + (off[q] + dl.chunk(q)), lds + q * 1024);
    }
    lds += Cfg::A_BYTES;
#pragma unroll
    for (int q = 0; q < Cfg::BN / 8; ++q) {
      constexpr int kHalf = Cfg::BN / 16;  // gate/up: ops of the gate rows, then of the up rows
      const char* b = kGateUp && q >= kHalf ? b1 : b0;
      const int q_in = kGateUp ? q % kHalf : q;
      const uint32_t o = (uint32_t)min(q_in * 8 + dl.row, b_rows - 1) * kp + dl.chunk(q);
      if (tail)
        dma_16_or_zero(b, o, dl.chunk(q), kp, lds + q * 1024);
      else
        lds_dma_16(b + o, lds + q * 1024);
    }
  }
};

template <typename Cfg, typename T, bool kGateUp, bool kGather>
__global__ __launch_bounds__(Cfg::WAVES * 64, 1) void gemm_i8_few_kernel(const Args p) {
  constexpr int NR = Cfg::NR, NC = Cfg::NC;
  __shared__ __attribute__((aligned(1024))) char smem[Cfg::LDS];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int G = gridDim.x;
  const int total = uniform(p.tiles.live(p.capacity)) * p.n_tiles_n;
  if ((int)blockIdx.x >= total) return;
  char* const ring = smem + wave * (Cfg::STAGES * Cfg::STAGE);

  FewCursor<Cfg, kGateUp, kGather> ld;  // the next step to load
  const int KT = (p.kp + kRowBytes - 1) / kRowBytes;
  const int n_steps = KT > wave ? (KT - wave + Cfg::WAVES - 1) / Cfg::WAVES : 0;
  ld.n = n_steps;
  ld.unit = blockIdx.x;
  ld.enter(p);
  ld.enter_rows(p, lane);
  ld.live = n_steps > 0;
  int issued = 0, used = 0;  // steps loaded and consumed so far; step i sits in stage i % STAGES
  auto issue = [&]() {
    ld.issue(p, wave, lane, ring + (issued % Cfg::STAGES) * Cfg::STAGE);
    ++issued;
    ld.advance(p, total, G, lane);
  };
#pragma unroll 1
  for (int i = 0; i < Cfg::STAGES; ++i)
    if (ld.live) issue();

  const int frag_row = lane & 15, fq = lane >> 4, fsw = (frag_row >> 1) & 7;
  int parity = 0;
  for (int unit = blockIdx.x; unit < total; unit += G) {
    const int mt = unit / p.n_tiles_n, nt = unit - mt * p.n_tiles_n;
    int e, row0, end;
    p.tiles.get(mt, e, row0, end);
    const int rows = uniform(min(p.tiles.height(), end - row0));
    for (int r0 = 0; r0 < rows; r0 += Cfg::BM) {
      i32x4_t acc[NR][NC];
#pragma unroll
      for (int i = 0; i < NR; ++i)
#pragma unroll
        for (int c = 0; c < NC; ++c) acc[i][c] = i32x4_t{0, 0, 0, 0};
      for (int step = 0; step < n_steps; ++step) {
        wait_groups<Cfg::OPS, Cfg::STAGES - 1>(issued - used - 1);  // this step has landed
        const char* sa = ring + (used % Cfg::STAGES) * Cfg::STAGE + frag_row * kRowBytes;
        i32x4_t fa[2][NR], fb[2][NC];
#pragma unroll
        for (int kh = 0; kh < 2; ++kh) {
          const int chunk = ((kh * 4 + fq) ^ fsw) << 4;
#pragma unroll
          for (int i = 0; i < NR; ++i)
            fa[kh][i] = *reinterpret_cast<const i32x4_t*>(sa + i * 16 * kRowBytes + chunk);
#pragma unroll
          for (int c = 0; c < NC; ++c)
            fb[kh][c] = *reinterpret_cast<const i32x4_t*>(sa + Cfg::A_BYTES + c * 16 * kRowBytes + chunk);
        }
        wait_lds();  // the stage has been read: it may be loaded again
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("" ::: "memory");
        ++used;
        if (ld.live) issue();
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int kh = 0; kh < 2; ++kh)
#pragma unroll
          for (int i = 0; i < NR; ++i)
#pragma unroll
            for (int c = 0; c < NC; ++c)
              acc[i][c] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fb[kh][c], fa[kh][i], acc[i][c], 0, 0, 0);
      }
      // the waves' sums meet, 32 rows at a time: row r's 16-byte piece c at piece
      // c ^ (r % pieces)
      static_for<Cfg::BM / Cfg::RED_ROWS>([&](auto half) {
        constexpr int i0 = decltype(half)::value * 2;  // the first of these rows' two 16-row blocks
        const int rh = r0 + i0 * 16;
        if (rh >= rows) return;
        constexpr int PIECES = Cfg::BN / 4, ROW = Cfg::BN * 4;
        char* const red = smem + Cfg::RED_OFF + parity * (Cfg::WAVES * Cfg::RED_WAVE);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            const int r = i * 16 + frag_row;
            *reinterpret_cast<i32x4_t*>(red + wave * Cfg::RED_WAVE + r * ROW +
                                        (((c * 4 + fq) ^ (r & (PIECES - 1))) << 4)) = acc[i0 + i][c];
          }
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        auto sum = [&](int r, int piece) {
          i32x4_t v = {0, 0, 0, 0};
#pragma unroll
          for (int w = 0; w < Cfg::WAVES; ++w)
            v += *reinterpret_cast<const i32x4_t*>(red + w * Cfg::RED_WAVE + r * ROW + ((piece ^ (r & (PIECES - 1))) << 4));
          return v;
        };
        constexpr int CP = kGateUp ? PIECES / 2 : PIECES;  // pieces of output columns
        const int r = threadIdx.x / CP, c = threadIdx.x % CP, n = nt * (CP * 4) + c * 4;
        if (r < Cfg::RED_ROWS && rh + r < rows && n < p.n) {
          const int64_t row = row0 + rh + r;
          const f32x4_t zero = {0.0f, 0.0f, 0.0f, 0.0f};
          const f32x4_t s0 = four(p.s0, e, n, p.n), s1 = kGateUp ? four(p.s1, e, n, p.n) : zero;
          const f32x4_t bias = !kGateUp && p.bias != nullptr ? bias_of<T>(p.bias, n, p.n) : zero;
          const i32x4_t g = sum(r, c);
          const auto o = out_of<T, kGateUp>(g, kGateUp ? sum(r, CP + c) : g, p.a_scale[row], s0, s1, bias);
          using E = std::conditional_t<std::is_same_v<T, bf16_t>, __bf16, T>;
          E* const at = static_cast<E*>(p.c) + row * p.n + n;
          if (p.n % 4 == 0) {
            *reinterpret_cast<typename Out4<T>::type*>(at) = o;
          } else {
#pragma unroll
            for (int q = 0; q < 4; ++q)
              if (n + q < p.n) at[q] = o[q];
          }
        }
        if constexpr (Cfg::RED_BUFS == 2)
          parity ^= 1;
        else  // the next sums go to the same place
          asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
      });
    }
  }
}

// ===========================================================================
// A few tokens: the product quantises its rows itself. Every workgroup reads the (at
// most 16) rows of its row tile, whose codes stay in LDS, behind its first weight
// loads: for one token the launch and the trip through memory that a quantiser of its
// own takes (4 to 5 us) are most of a small product's time. Otherwise as above. The rows
// are held in two units of 512 values a wave (UNITS); a third and fourth cost 1.2 to 1.7
// us, as much as a quantiser of its own or more (us a product with them / a quantiser:
// 4096 to 14336, 2 rows 20.2 / 19.0; 2048 to 5632, 4 rows 9.3 / 7.8; 1024 to 4096, 8 rows
// 7.8 / 7.3; of two units 4096 to 14336, 1 row 18.4, 2048 to 5632 6.6, 512 to 1536 4.3).
// ===========================================================================
struct QuantCfg {
  static constexpr int BM = 16, BN = 32, WAVES = 4, STAGES = 8, UNITS = 2;
  static constexpr int STAGE = BN * kRowBytes;                 // weights only
  static constexpr int CODES = UNITS * WAVES * 512 + BM * kRowBytes;  // bytes of the rows' codes, in whole steps
  static constexpr int RED_WAVE = BM * BN * 4;                 // one wave's sums
  static constexpr int CODE_OFF = WAVES * STAGES * STAGE, RED_OFF = CODE_OFF + CODES;
  static constexpr int LDS = RED_OFF + 2 * WAVES * RED_WAVE;   // 150 KB
  static_assert(LDS + 256 <= 160 * 1024, "LDS");
};

template <typename T, bool kGateUp, bool kGather, bool kVec>
__global__ __launch_bounds__(QuantCfg::WAVES * 64, 1) void gemm_i8_quant_kernel(const Args p) {
  using Cfg = QuantCfg;
  using C = typename CodeType<T>::type;
  constexpr int NC = Cfg::BN / 16, OPS = Cfg::STAGE / 1024;
  __shared__ __attribute__((aligned(1024))) char smem[Cfg::LDS];
  __shared__ uint32_t s_top[Cfg::BM];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int G = gridDim.x;
  const int total = uniform(p.tiles.live(p.capacity)) * p.n_tiles_n;
  if ((int)blockIdx.x >= total) return;
  char* const ring = smem + wave * (Cfg::STAGES * Cfg::STAGE);
  char* const codes = smem + Cfg::CODE_OFF;
  const uint32_t kp = (uint32_t)p.kp;
  const int KT = (p.kp + kRowBytes - 1) / kRowBytes, row_bytes = KT * kRowBytes;
  const int n_steps = KT > wave ? (KT - wave + Cfg::WAVES - 1) / Cfg::WAVES : 0;
  constexpr int kCols = kGateUp ? Cfg::BN / 2 : Cfg::BN;

  // ---- weights: the wave's next step to load ----
  int l_unit = blockIdx.x, l_j = 0, l_rot = 0, l_rows = 0;
  bool l_live = n_steps > 0;
  const char *b0 = nullptr, *b1 = nullptr;
  auto enter = [&]() {
    const int mt = l_unit / p.n_tiles_n, nt = l_unit - mt * p.n_tiles_n;
    int e, row0, end;
    p.tiles.get(mt, e, row0, end);
    e = uniform(e);
    l_rows = min(kCols, p.n - nt * kCols);
    const int64_t at = ((int64_t)e * p.n + (int64_t)nt * kCols) * p.kp;
    b0 = reinterpret_cast<const char*>(p.w0 + at);
    b1 = kGateUp ? reinterpret_cast<const char*>(p.w1 + at) : b0;
    l_rot = n_steps > 0 ? (7 * e + 3 * nt) % n_steps : 0;
    l_j = 0;
  };
  int issued = 0, used = 0;
  auto issue = [&]() {
    int jr = l_j + l_rot;
    if (jr >= n_steps) jr -= n_steps;
    const int ks = wave + Cfg::WAVES * jr;
    char* const lds = ring + (issued % Cfg::STAGES) * Cfg::STAGE;
    const DmaLane dl(lane, ks);
    const bool tail = (uint32_t)(ks + 1) * kRowBytes > kp;
#pragma unroll
    for (int q = 0; q < OPS; ++q) {
      constexpr int kHalf = OPS / 2;
      const char* b = kGateUp && q >= kHalf ? b1 : b0;
      const int q_in = kGateUp ? q % kHalf : q;
      const uint32_t o = (uint32_t)min(q_in * 8 + dl.row, l_rows - 1) * kp + dl.chunk(q);
      if (tail)
        dma_16_or_zero(b, o, dl.chunk(q), kp, lds + q * 1024);
      else
        lds_dma_16(b + o, lds + q * 1024);
    }
    ++issued;
    if (++l_j == n_steps) {
      l_unit += G;
      l_live = l_unit < total;
      if (l_live) enter();
    }
  };
  enter();

  // ---- the rows of one tile: unit i of the wave is the 512 columns of chunk wave + 4 i,
  // the chunks of one row after those of the one before ----
  const int chunks = (p.kp + 511) / 512;
  Unit<T> v[Cfg::UNITS];
  int unit_row[Cfg::UNITS], unit_col[Cfg::UNITS];
#pragma unroll
  for (int i = 0; i < Cfg::UNITS; ++i) {
    unit_row[i] = (wave + 4 * i) / chunks;
    unit_col[i] = (wave + 4 * i - unit_row[i] * chunks) * 512 + lane * 8;
  }
  // (a unit without a row loads the first one's again)
  auto load_rows = [&](int row0, int rows) {
#pragma unroll
    for (int i = 0; i < Cfg::UNITS; ++i) {
      const int r = unit_row[i] < rows ? unit_row[i] : 0;
      const int64_t src = kGather ? p.row_src[row0 + r] : row0 + r;
      v[i].template load<kVec>(static_cast<const T*>(p.x) + src * p.k, unit_col[i], p.k);
    }
  };
  // (after a barrier behind the last reads of the tile before) the rows' codes and maxima.
  // Every unit's load is used: one left in flight would have the loop below wait for all.
  auto quantise = [&](int rows) {
    if (threadIdx.x < Cfg::BM) s_top[threadIdx.x] = 0;
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
    for (int i = 0; i < Cfg::UNITS; ++i) {
      const int r = unit_row[i];
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) top = max(top, v[i].bits(j) & 0x7fffffffu);
      top = lanes_max<64>(top);
      if (lane == 0 && r < rows) atomicMax(&s_top[r], top);
    }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
    for (int i = 0; i < Cfg::UNITS; ++i) {
      const int r = unit_row[i], col = unit_col[i];
      if (r >= rows) break;
      const uint32_t top = s_top[r];
      const float most = __uint_as_float(top), shift = range_shift(most);
      const C m = (C)most * (C)shift, inv = (C)127 / m;
      const bool zero = top == 0 || top >= 0x7f800000u;
      // 16-byte piece x of a step's 8 at piece x ^ (r & 7)
      if (col < row_bytes) {
        const int piece = (col >> 4 & 7) ^ (r & 7);
        *reinterpret_cast<uint2*>(codes + r * row_bytes + (col & ~127) + piece * 16 + (col & 8)) =
            zero ? make_uint2(0, 0) : v[i].template codes<C>(shift, m, inv);
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  };

  const int frag_row = lane & 15, fq = lane >> 4, fsw = (frag_row >> 1) & 7;
  int parity = 0, have = -1;
  for (int unit = blockIdx.x; unit < total; unit += G) {
    const int mt = unit / p.n_tiles_n, nt = unit - mt * p.n_tiles_n;
    int e, row0, end;
    p.tiles.get(mt, e, row0, end);
    e = uniform(e), row0 = uniform(row0);
    const int rows = min(Cfg::BM, uniform(end) - row0);
    if (mt != have) {
      load_rows(row0, rows);
      if (have < 0)  // the first weights right behind the rows
#pragma unroll 1
        for (int i = 0; i < Cfg::STAGES; ++i)
          if (l_live) issue();
      quantise(rows);
      have = mt;
    }
    const int my_row = min(frag_row, rows - 1);
    const char* const ca = codes + my_row * row_bytes;
    i32x4_t acc[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) acc[c] = i32x4_t{0, 0, 0, 0};
    const int rot = n_steps > 0 ? (7 * e + 3 * nt) % n_steps : 0;
    for (int step = 0; step < n_steps; ++step) {
      int jr = step + rot;
      if (jr >= n_steps) jr -= n_steps;
      const int ks = wave + Cfg::WAVES * jr;
      wait_groups<OPS, Cfg::STAGES - 1>(issued - used - 1);  // this step has landed
      const char* sb = ring + (used % Cfg::STAGES) * Cfg::STAGE + frag_row * kRowBytes;
      i32x4_t fa[2], fb[2][NC];
#pragma unroll
      for (int kh = 0; kh < 2; ++kh) {
        const int chunk = kh * 4 + fq;
        fa[kh] = *reinterpret_cast<const i32x4_t*>(ca + ks * kRowBytes + ((chunk ^ (my_row & 7)) << 4));
#pragma unroll
        for (int c = 0; c < NC; ++c)
          fb[kh][c] = *reinterpret_cast<const i32x4_t*>(sb + c * 16 * kRowBytes + ((chunk ^ fsw) << 4));
      }
      wait_lds();  // the stage has been read: it may be loaded again
      __builtin_amdgcn_sched_barrier(0);
      asm volatile("" ::: "memory");
      ++used;
      if (l_live) issue();
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int kh = 0; kh < 2; ++kh)
#pragma unroll
        for (int c = 0; c < NC; ++c)
          acc[c] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fb[kh][c], fa[kh], acc[c], 0, 0, 0);
    }
    constexpr int PIECES = Cfg::BN / 4, ROW = Cfg::BN * 4;
    char* const red = smem + Cfg::RED_OFF + parity * (Cfg::WAVES * Cfg::RED_WAVE);
#pragma unroll
    for (int c = 0; c < NC; ++c)
      *reinterpret_cast<i32x4_t*>(red + wave * Cfg::RED_WAVE + frag_row * ROW +
                                  (((c * 4 + fq) ^ (frag_row & (PIECES - 1))) << 4)) = acc[c];
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    auto sum = [&](int r, int piece) {
      i32x4_t t = {0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < Cfg::WAVES; ++w)
        t += *reinterpret_cast<const i32x4_t*>(red + w * Cfg::RED_WAVE + r * ROW + ((piece ^ (r & (PIECES - 1))) << 4));
      return t;
    };
    constexpr int CP = kGateUp ? PIECES / 2 : PIECES;  // pieces of output columns
    const int r = threadIdx.x / CP, c = threadIdx.x % CP, n = nt * kCols + c * 4;
    if (r < rows && n < p.n) {
      const int64_t row = row0 + r;
      const f32x4_t zero = {0.0f, 0.0f, 0.0f, 0.0f};
      const f32x4_t s0 = four(p.s0, e, n, p.n), s1 = kGateUp ? four(p.s1, e, n, p.n) : zero;
      const f32x4_t bias = !kGateUp && p.bias != nullptr ? bias_of<T>(p.bias, n, p.n) : zero;
      const uint32_t top = s_top[r];
      const float sa = top >= 0x7f800000u ? NAN : __uint_as_float(top) / 127.0f;
      const i32x4_t g = sum(r, c);
      const auto o = out_of<T, kGateUp>(g, kGateUp ? sum(r, CP + c) : g, sa, s0, s1, bias);
      using E = std::conditional_t<std::is_same_v<T, bf16_t>, __bf16, T>;
      E* const at = static_cast<E*>(p.c) + row * p.n + n;
      if (p.n % 4 == 0) {
        *reinterpret_cast<typename Out4<T>::type*>(at) = o;
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (n + q < p.n) at[q] = o[q];
      }
    }
    parity ^= 1;
    // (the next tile's quantise() clears the maxima: not before these have been read)
    if (unit + G < total && (unit + G) / p.n_tiles_n != mt) asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  }
}
#endif  // ASTRAI_MOE_RAGGED_K

Args args_of(const Int8Gemm& g) {
  Args a{};
  a.a = g.a, a.a_scale = g.a_scale, a.row_src = g.row_src;
  a.tiles = RowTiles{g.tiles, (int)g.n_rows, g.block_m};
  a.w0 = g.w0, a.w1 = g.w1, a.s0 = g.s0, a.s1 = g.s1, a.bias = g.bias;
  a.x = g.x, a.k = g.k;
  a.kp = (int)g.kp, a.n = (int)g.n, a.capacity = (int)g.capacity, a.c = g.c;
  return a;
}

template <typename Cfg, typename T, bool kGateUp, bool kGather, bool kHalves = false>
int launch_tiles(const Int8Gemm& g, hipStream_t s) {
  if (g.capacity == 0) return ASTRAI_MOE_OK;
  Args a = args_of(g);
  const int64_t n_tiles_n = ceil_div(g.n, kGateUp ? Cfg::BN / 2 : Cfg::BN);  // the last may be partial
  a.n_tiles_n = (int)n_tiles_n;
  int64_t grid = 0;
  if (int rc = persistent_grid(g.capacity, kHalves ? 2 * n_tiles_n : n_tiles_n, &grid)) return rc;
  hipLaunchKernelGGL((gemm_i8_kernel<Cfg, T, kGateUp, kGather, kHalves>), dim3((unsigned)grid), dim3(Cfg::THREADS), 0, s,
                     a);
  return check_launch(kGateUp ? "gemm_i8_kernel<gate_up>" : "gemm_i8_kernel<down>");
}

template <typename T, bool kGateUp, bool kGather, bool kBias>
int launch_stream(const Int8Gemm& g, hipStream_t s) {
  if (g.capacity == 0) return ASTRAI_MOE_OK;
  using Cfg = StreamCfg<kGateUp>;
  Args a = args_of(g);
  const int64_t n_tiles_n = ceil_div(g.n, kGateUp ? Cfg::BN / 2 : Cfg::BN);  // the last may be partial
  a.n_tiles_n = (int)n_tiles_n;
  int64_t grid = 0;
  if (int rc = persistent_grid(g.capacity, n_tiles_n, &grid)) return rc;
  const int64_t ksteps = ceil_div(g.kp, kRowBytes);
  const bool have_ws = g.ws.base != nullptr && g.ws.bytes >= kSchedBytes && grid <= kMaxSchedGroups;
  a.sched = have_ws && ksteps >= kDynamicMinSteps ? static_cast<int32_t*>(g.ws.base) : nullptr;
  a.part = !kGateUp && have_ws && splits_tail(g.kp / 2) &&
                   g.ws.bytes >= kSchedBytes + grid * (int64_t)sizeof(float) * kSplitUnitFloats
               ? reinterpret_cast<float*>(static_cast<char*>(g.ws.base) + kSchedBytes)
               : nullptr;
  hipLaunchKernelGGL((gemm_i8_stream_kernel<T, kGateUp, kGather, kBias>), dim3((unsigned)grid), dim3(Cfg::THREADS), 0,
                     s, a);
  if (int rc = check_launch(kGateUp ? "gemm_i8_stream_kernel<gate_up>" : "gemm_i8_stream_kernel<down>")) return rc;
  if constexpr (!kGateUp) {
    if (a.part == nullptr) return ASTRAI_MOE_OK;
    // whether the tail was split is decided on the device: at most G / 2 tail tiles
    hipLaunchKernelGGL((i8_split_reduce_kernel<T, kBias>), dim3((unsigned)((grid + 1) / 2), Cfg::MW), dim3(64), 0, s, a,
                       (int)grid);
    return check_launch("i8_split_reduce_kernel");
  }
  return ASTRAI_MOE_OK;
}

template <typename T, bool kGateUp, bool kGather>
int launch_typed(const Int8Gemm& g, hipStream_t s) {
  const Tiles pick = pick_tiles(g.rows, g.block_m, g.kp / 2, g.n, kGateUp).tiles;
  if (pick == Tiles::kHalves) return launch_tiles<Mid2Cfg, T, kGateUp, kGather, true>(g, s);
  if (pick == Tiles::kNarrowMid) return launch_tiles<NarrowMidCfg, T, kGateUp, kGather>(g, s);
  if (pick == Tiles::kNarrow) return launch_tiles<NarrowCfg, T, kGateUp, kGather>(g, s);
  if (pick == Tiles::kNarrowHalves) return launch_tiles<NarrowCfg, T, kGateUp, kGather, true>(g, s);
  if (g.block_m == kMfmaBigBM) {
    // (an fp32 h, taken in 64 bits, does not fit the streaming kernel's registers)
    if constexpr (kGateUp && std::is_same_v<T, float>)
      return launch_tiles<Mid2Cfg, T, kGateUp, kGather, true>(g, s);
    else if constexpr (!kGateUp)
      if (g.bias != nullptr) return launch_stream<T, kGateUp, kGather, true>(g, s);
    if constexpr (!(kGateUp && std::is_same_v<T, float>)) return launch_stream<T, kGateUp, kGather, false>(g, s);
  }
  if (g.block_m == kMfmaMidBM) return launch_tiles<MidCfg, T, kGateUp, kGather>(g, s);
  if (g.block_m == kMfmaMid2BM) return launch_tiles<Mid2Cfg, T, kGateUp, kGather>(g, s);
  return launch_tiles<SmallCfg, T, kGateUp, kGather>(g, s);
}

#if ASTRAI_MOE_RAGGED_K
template <typename Cfg, typename T, bool kGateUp, bool kGather>
int launch_few_cfg(const Int8Gemm& g, hipStream_t s) {
  if (g.capacity == 0) return ASTRAI_MOE_OK;
  Args a = args_of(g);
  const int64_t n_cols = ceil_div(g.n, kGateUp ? Cfg::BN / 2 : Cfg::BN);  // the last may be partial
  a.n_tiles_n = (int)n_cols;
  int64_t grid = 0;
  if (int rc = persistent_grid(g.capacity, n_cols, &grid)) return rc;
  hipLaunchKernelGGL((gemm_i8_few_kernel<Cfg, T, kGateUp, kGather>), dim3((unsigned)grid), dim3(Cfg::WAVES * 64), 0, s, a);
  return check_launch(kGateUp ? "gemm_i8_few_kernel<gate_up>" : "gemm_i8_few_kernel<down>");
}

// Tiles of 64 rows where lists are as high and most experts, or one, have more than
// 32; of 16 weight rows for one expert's single run of rows where these fill the
// compute units better (the rules of launch_few_tiles in moe_gemm_few.hip).
template <typename T, bool kGateUp, bool kGather>
int launch_few(const Int8Gemm& g, hipStream_t s) {
  const int64_t most = g.rows.dense() ? 2 * FewCfg<32, 32>::BM : 24 * (int64_t)(g.rows.experts + g.rows.exact);
  if (g.block_m >= FewCfg<64, 32>::BM && g.rows.total() > most)
    return launch_few_cfg<FewCfg<64, 32>, T, kGateUp, kGather>(g, s);
  auto fill = [](int64_t tiles) {  // share of the compute units' time that they fill
    const double rounds = (double)tiles / cu_count();
    return rounds / std::ceil(rounds);
  };
  if (g.rows.dense() && g.rows.total() <= FewCfg<32, 16>::BM &&
      fill(ceil_div(g.n, kGateUp ? 8 : 16)) > 1.05 * fill(ceil_div(g.n, kGateUp ? 16 : 32)))
    return launch_few_cfg<FewCfg<32, 16>, T, kGateUp, kGather>(g, s);
  return launch_few_cfg<FewCfg<32, 32>, T, kGateUp, kGather>(g, s);
}

template <typename T, bool kGateUp, bool kGather>
int launch_quant(const Int8Gemm& g, hipStream_t s) {
  if (g.capacity == 0) return ASTRAI_MOE_OK;
  Args a = args_of(g);
  const int64_t n_cols = ceil_div(g.n, kGateUp ? QuantCfg::BN / 2 : QuantCfg::BN);  // the last may be partial
  a.n_tiles_n = (int)n_cols;
  int64_t grid = 0;
  if (int rc = persistent_grid(g.capacity, n_cols, &grid)) return rc;
  const bool vec = g.k * (int64_t)sizeof(T) % 16 == 0 && aligned16(g.x);  // (the rows' 16-byte pieces)
  hipLaunchKernelGGL((vec ? gemm_i8_quant_kernel<T, kGateUp, kGather, true> : gemm_i8_quant_kernel<T, kGateUp, kGather, false>),
                     dim3((unsigned)grid), dim3(QuantCfg::WAVES * 64), 0, s, a);
  return check_launch(kGateUp ? "gemm_i8_quant_kernel<gate_up>" : "gemm_i8_quant_kernel<down>");
}
#endif

}  // namespace

#if ASTRAI_MOE_RAGGED_K
// Where the registers and the LDS hold the rows, and a workgroup meets few row tiles,
// each of which it quantises anew: one expert's rows, or at most two tiles a workgroup.
bool int8_quantises(int64_t most_rows, int64_t k, int64_t row_tiles, int64_t n, bool gate_up) {
  const int64_t tiles = row_tiles * ceil_div(n, gate_up ? QuantCfg::BN / 2 : QuantCfg::BN);
  return (row_tiles == 1 || tiles <= 2 * cu_count()) && most_rows <= QuantCfg::BM &&
         most_rows * ceil_div(k, 512) <= QuantCfg::WAVES * QuantCfg::UNITS;
}

// Where the few-row kernels replace the tiles of 64 or 128 rows: as few_rows says of
// the bf16 ones, but for more than 32 rows of one expert only where a round holds all
// the column tiles, each of which stages every row again (us a product with / without
// them: 4096 to 14336, 448 tiles, 40 rows 31.9 / 25.5, 100 38.2 / 26.4; 14336 to 4096,
// 128 tiles, 40 25.5 / 63.5, 128 34.7 / 64.7; 2048 to 5632, 176 tiles, 64 11.5 / 14.6);
// and in 64-row lists where a round holds the tiles of all runs of 64 rows (512 to 512, 500
// rows 7.2 / 8.5; 1000 to 2664, 130 rows 8.9 / 12.2; 4096 to 1024, 333 rows 13.7 / 22.6;
// in two rounds 1000 to 2664, 333 rows 12.5 / 12.7, 512 to 2048 9.4 / 8.6, 1024 to 4096
// 15.5 / 11.9).
// And routed rows of short products only where two rounds hold their column tiles:
// with fewer than kFewMinSteps K steps, of which a wave takes every fourth, a tile's
// sums cost more than its loads (us a layer with / without: 64 experts, top-6 and a
// shared one, D 2048, F 1408, 2 tokens 49.4 / 42.6, 8 95 / 84; 128 experts, top-8, D
// 4096, F 1536, 16 335 / 300; long ones gain: 8 experts, D 4096, F 14336, 2 tokens 132 /
// 175, 32 275 / 297).
constexpr int kFewMinSteps = 20;
bool int8_few_rows(const RowCounts& rows, int block_m, int64_t kp, int64_t n, bool gate_up) {
  const double cols = (double)ceil_div(n, gate_up ? 16 : 32);
  if (rows.dense()) {
    if (rows.exact_rows > 32 && cols > cu_count()) return false;
    if (block_m == kMfmaMidBM && ceil_div(rows.exact_rows, kMfmaMidBM) * cols <= cu_count()) return true;
  } else if (ceil_div(kp, kRowBytes) < kFewMinSteps) {
    const double e = rows.experts, live = e > 0 ? e * (1.0 - std::pow(1.0 - 1.0 / e, (double)rows.rows)) : 0.0;
    if ((live + rows.exact) * cols > 2.0 * cu_count()) return false;
  }
  return few_rows(rows, block_m, kp / 2, n, gate_up);
}

namespace ragged {

int launch_int8_quant(const Int8Gemm& g, hipStream_t s) {
  if (g.dtype == ASTRAI_MOE_BF16)
    return g.w1 != nullptr ? launch_quant<bf16_t, true, true>(g, s) : launch_quant<bf16_t, false, false>(g, s);
  return g.w1 != nullptr ? launch_quant<float, true, true>(g, s) : launch_quant<float, false, false>(g, s);
}

int launch_int8_few(const Int8Gemm& g, hipStream_t s) {
  if (g.dtype == ASTRAI_MOE_BF16)
    return g.w1 != nullptr ? launch_few<bf16_t, true, true>(g, s) : launch_few<bf16_t, false, false>(g, s);
  return g.w1 != nullptr ? launch_few<float, true, true>(g, s) : launch_few<float, false, false>(g, s);
}

#endif

int launch_int8_mfma(const Int8Gemm& g, hipStream_t s) {
#if !ASTRAI_MOE_RAGGED_K
  if (g.a == nullptr) return ragged::launch_int8_quant(g, s);
  if (aligned16(g.c) && int8_few_rows(g.rows, g.block_m, g.kp, g.n, g.w1 != nullptr)) return ragged::launch_int8_few(g, s);
  const int size = g.dtype == ASTRAI_MOE_BF16 ? 2 : 4;
  if (g.kp % kRowBytes != 0 || g.n * size % 16 != 0 || g.n % 4 != 0 || !aligned16(g.c))
    return ragged::launch_int8_mfma(g, s);
#endif
  // (the gate/up products gather their rows, the others take them as they lie)
  if (g.dtype == ASTRAI_MOE_BF16)
    return g.w1 != nullptr ? launch_typed<bf16_t, true, true>(g, s) : launch_typed<bf16_t, false, false>(g, s);
  return g.w1 != nullptr ? launch_typed<float, true, true>(g, s) : launch_typed<float, false, false>(g, s);
}

#if ASTRAI_MOE_RAGGED_K
}  // namespace ragged
#endif

}  // namespace astrai_moe
