// The permutation and tile list of one chunk of tokens, written by the workgroup
// that routed it (moe_route.hip, moe_route_scores.hip).
#pragma once

#include "moe_common.h"
#include "moe_gemm.h"

namespace astrai_moe {
namespace {

constexpr int kRouteThreads = 1024;  // 16 waves: a 32-token chunk is 2 rounds of 16 tokens at E >= 64

static_assert(ASTRAI_MOE_CHUNK_TOKENS == 32, "an expert's tokens of a chunk are a 32-bit mask");
static_assert(ASTRAI_MOE_MAX_EXPERTS <= kRouteThreads && ASTRAI_MOE_CHUNK_TOKENS * ASTRAI_MOE_MAX_TOPK <= kRouteThreads,
              "one thread per expert, one per (token, slot)");

// The permutation and tile list of one chunk from the experts' token masks
// (columns n_experts .. are the shared experts') and the (token, slot) entries
// s_e, s_w. Called by the whole workgroup after a barrier behind their writes.
template <typename T>
__device__ void write_chunk_list(const uint32_t* mask, int* base, const int* s_e, const T* s_w, int n_tokens,
                                 int columns, int slots, const RouteList& out) {
  __shared__ int s_wave[kRouteThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int count = tid < columns ? __popc(mask[tid]) : 0;
  // rows in the low half, tiles (one of at least 32 rows per live expert) above
  const int own = count | (count > 0 ? 1 << 16 : 0);
  int incl = own;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int o = __shfl_up(incl, off, 64);
    if (lane >= off) incl += o;
  }
  if (lane == 63) s_wave[wave] = incl;
  __syncthreads();
  int before = incl - own, total = 0;
#pragma unroll
  for (int w = 0; w < kRouteThreads / 64; ++w) {
    if (w < wave) before += s_wave[w];
    total += s_wave[w];
  }
  const int row0 = before & 0xffff, slot = before >> 16;
  if (tid < columns) base[tid] = row0;
  if (count > 0 && slot < out.tile_capacity) {
    int32_t* t = out.tiles + ASTRAI_MOE_TILE_HEADER + (int64_t)slot * ASTRAI_MOE_TILE_STRIDE;
    t[0] = tid;
    t[1] = row0;
    t[2] = row0 + count;
  }
  if (tid == 0) {
    const int n_tiles = total >> 16;
    out.tiles[0] = n_tiles;
    out.tiles[1] = out.block_m;
    out.tiles[2] = (int32_t)out.tile_capacity;
    out.tiles[3] = 0;  // no expert has a whole group of tiles
  }
  __syncthreads();
  if (tid < n_tokens * slots) {
    const int e = s_e[tid], t = tid / slots;
    const int pos = base[e] + __popc(mask[e] & ((1u << t) - 1u));
    out.token_pos[tid] = pos;
    out.sorted_token[pos] = t;
    static_cast<T*>(out.sorted_w)[pos] = s_w[tid];
  }
}

}  // namespace
}  // namespace astrai_moe
