// The keys that rows of a sliding window with sinks see, without the gap between the two.
//
// Query t of a sequence sees key j <= t iff t - j <= left or j < sinks.  A group of rows at tokens q0, q0 + 1, ... takes its keys in tiles of
// 128 from the list
//     column u:  key u                for u < room,      room = sinks rounded up to 8 rows (the swizzle's unit),
//                key u + shift        for u >= room,     shift = max(0, q0 - left - room),
// so the window starts at the first key that any of the rows sees, wherever that lies, and the sinks fill the head of the first tile
// instead of costing a tile of their own.  The tile in which the list jumps is loaded by two TMA boxes.  Columns [sinks, room) are hidden from
// every row where there is a gap (their keys lie in front of the window), and are ordinary keys where there is none.
#pragma once
#include <type_traits>

#include "tc5.cuh"

namespace nsa {

// Boxes of the two parts of the tile in which the list jumps: room % 128 rows, and the rest; and the tensors themselves, for the rows that
// are computed one by one (sink_exact.cuh).
struct SinkMaps {
  CUtensorMap k[2], v[2];
  const void *q, *keys, *values, *dout;
  long long q_sn, q_sh, k_sn, k_sh, v_sn, v_sh, do_sn, do_sh;
};
struct NoMaps {};
template <bool SINKS>
using TileMaps = std::conditional_t<SINKS, SinkMaps, NoMaps>;

__host__ __device__ __forceinline__ int sink_room(int sinks) { return (sinks + 7) & ~7; }
__device__ __forceinline__ int sink_shift(int q0, int left, int room) { return max(0, q0 - left - room); }

// Tile i of the list into shared memory, PANELS panels of PANEL bytes; one thread, with the barrier's bytes announced.  `row0` is the
// sequence's first key row, `whole` the map with boxes of 128 rows, `part` those of the split tile.
template <int PANELS, int PANEL>
__device__ __forceinline__ void load_key_tile(uint8_t* sm, const CUtensorMap* whole, const CUtensorMap* part, uint64_t* bar, int head, int row0, int i,
                                              int room, int shift) {
  const int u = i * 128, first = room - u;  // rows of the tile in front of the jump
#pragma unroll
  for (int pn = 0; pn < PANELS; ++pn) {
    if (shift == 0 || first <= 0 || first >= 128) {
      tma_load_3d(sm + pn * PANEL, whole, bar, pn * 64, head, row0 + u + (first <= 0 ? shift : 0));
    } else {
      tma_load_3d(sm + pn * PANEL, part, bar, pn * 64, head, row0 + u);
      tma_load_3d(sm + pn * PANEL + first * 128, part + 1, bar, pn * 64, head, row0 + room + shift);
    }
  }
}

// The rows of tile i that stand for no key of the rows' list: behind its last column `n`, and between the sinks and the window.
template <int PANELS, int PANEL>
__device__ __forceinline__ void clean_key_tile(uint32_t tile, int i, int n, int sinks, int shift) {
  const int end = n - i * 128;
  if (end < 128) zero_tile_rows<PANELS, PANEL>(tile, max(0, end), 128);
  const int hide0 = sinks - i * 128, hide1 = sink_room(sinks) - i * 128;
  if (shift > 0 && hide1 > hide0 && hide0 < 128 && hide1 > 0) zero_tile_rows<PANELS, PANEL>(tile, max(0, hide0), min(128, hide1));
}

// Rows of G heads from `head` on that belong to no sequence (a padded batch), [first, rows), as zeros; block x of n takes every n-th.  A warp.
template <typename T, int D>
__device__ __forceinline__ void zero_rows_behind(void* x, long long sn, long long sh, int first, int rows, int block, int blocks, int head, int G) {
  for (long long n = (long long)first + block; n < rows; n += blocks)
    for (int c = lane_id(); c < G * (D / 8); c += 32)
      *reinterpret_cast<uint4*>(static_cast<T*>(x) + n * sn + (head + c / (D / 8)) * sh + c % (D / 8) * 8) = make_uint4(0, 0, 0, 0);
}

}  // namespace nsa
