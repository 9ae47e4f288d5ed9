// The keys that rows of a sliding window with sinks see, without the gap between the two.
//
// Query t of a sequence sees key j <= t iff t - j <= left or j < sinks.  A group of rows at tokens q0, q0 + 1, ... takes its keys in tiles
// from the list
//     column u:  key u                for u < room,      room = sinks rounded up to 8 rows (the swizzle's unit),
//                key u + shift        for u >= room,     shift = max(0, q0 - left - room),
// so the window starts at the first key that any of the rows sees, wherever that lies, and the sinks fill the head of the first tile
// instead of costing a tile of their own.  The tile in which the list jumps is loaded by two TMA boxes.  Columns [sinks, room) are hidden from
// every row where there is a gap (their keys lie in front of the window), and are ordinary keys where there is none.
#pragma once
#include "tc5.cuh"
#include "work_steal.cuh"

namespace nsa {

// Boxes of the two parts of the tile in which the list jumps: room % (rows of a tile), and the rest; and the tensors themselves, for the rows that
// are computed one by one (sink_exact.cuh).
struct SinkMaps {
  CUtensorMap k[2], v[2];
  const void *q, *keys, *values, *dout;
  long long q_sn, q_sh, k_sn, k_sh, v_sn, v_sh, do_sn, do_sh;
};

inline void sink_inputs(SinkMaps& m, const void* q, const void* k, const void* v, const void* dout, const long long* S) {
  m.q = q; m.keys = k; m.values = v; m.dout = dout;
  m.q_sn = S[0]; m.q_sh = S[1]; m.k_sn = S[2]; m.k_sh = S[3]; m.v_sn = S[4]; m.v_sh = S[5]; m.do_sn = S[6]; m.do_sh = S[7];
}

__host__ __device__ __forceinline__ int sink_room(int sinks) { return (sinks + 7) & ~7; }
__device__ __forceinline__ int sink_shift(int q0, int left, int room) { return max(0, q0 - left - room); }

// Tile i of the list, KEYS rows of PANELS panels, into shared memory; one thread, with the barrier's bytes announced.  `row0` is the
// sequence's first key row, `whole` the map with boxes of KEYS rows, `part` those of the split tile.
template <int KEYS, int PANELS>
__device__ __forceinline__ void load_key_tile(uint8_t* sm, const CUtensorMap* whole, const CUtensorMap* part, uint64_t* bar, int head, int row0, int i,
                                              int room, int shift) {
  const int u = i * KEYS, first = room - u;  // rows of the tile in front of the jump
#pragma unroll
  for (int pn = 0; pn < PANELS; ++pn) {
    uint8_t* dst = sm + pn * KEYS * 128;
    if (shift == 0 || first <= 0 || first >= KEYS) {
      tma_load_3d(dst, whole, bar, pn * 64, head, row0 + u + (first <= 0 ? shift : 0));
    } else {
      tma_load_3d(dst, part, bar, pn * 64, head, row0 + u);
      tma_load_3d(dst + first * 128, part + 1, bar, pn * 64, head, row0 + room + shift);
    }
  }
}

// The rows of tile i behind the list's last column n, which are other sequences' or nobody's, as zeros.  (Rows that are not finite are computed
// again one by one in any case, see sink_exact.cuh; but what lies behind a batch may well not be, and should not cost that.)
template <int KEYS, int PANELS>
__device__ __forceinline__ void clean_key_tile(uint32_t tile, int i, int n) {
  const int end = n - i * KEYS;
  if (end < KEYS) zero_tile_rows<PANELS, KEYS * 128>(tile, max(0, end), KEYS);
}

// What the rounding of the output o took away, rounded itself (what the products gave is then known to 2^-16 of itself in bf16, in fp16 to 2^-22, or
// 2^-25 where that is more; the forward's cubics, 7.5e-5 of a third of P in tiles that are seen in full, are in those): 16-byte chunk c of a row, in an
// order in which the rows of a warp are neighbours.  The backward pass needs sum_d o dO next to single dO v: where a row looks at few keys the
// two all but cancel, and what is left of o's rounding becomes as large as dS (one key of weight 1 - w: dS is w of its parts).
__device__ __forceinline__ long long rest_chunk(int c, int kvh, int Hkv, int rows, int n, int G, int g) {
  return (((long long)c * Hkv + kvh) * rows + n) * G + g;
}

// A row tile (find_row_tile) of a batch of `rows` rows.  What cu says is held against the rows there are: a tile outside of them is none, a sequence
// that ends behind them ends with them, and either raises the status.  A whole warp.
__device__ __forceinline__ bool find_tile_of_rows(const int* cu, int nseq, int rows, int log_per, int want, const Status& st, int& b, int& start,
                                                  int& len, int& tile) {
  if (!find_row_tile(cu, nseq, log_per, want, b, start, len, tile)) return false;
  if (start >= 0 && tile >= 0 && len <= rows - start) return true;
  if (lane_id() == 0) st.raise(kErrBadIndex);
  if (start < 0 || start >= rows || tile < 0) return false;
  len = min(len, rows - start);
  return ((long long)tile << log_per) < len;
}
// The end of the last sequence, within the rows there are.
__device__ __forceinline__ int end_of_rows(const int* cu, int nseq, int rows, const Status& st) {
  const int end = load_fresh(cu + nseq);
  if ((end < 0 || end > rows || load_fresh(cu) < 0) && lane_id() == 0) st.raise(kErrBadIndex);
  return max(0, min(end, rows));
}

// Rows of G heads from `head` on that belong to no sequence (a padded batch), [first, rows), as zeros; block x of n takes every n-th.  A warp.
template <typename T, int D>
__device__ __forceinline__ void zero_rows_behind(void* x, long long sn, long long sh, int first, int rows, int block, int blocks, int head, int G) {
  for (long long n = (long long)first + block; n < rows; n += blocks)
    for (int c = lane_id(); c < G * (D / 8); c += 32)
      *reinterpret_cast<uint4*>(static_cast<T*>(x) + n * sn + (head + c / (D / 8)) * sh + c % (D / 8) * 8) = make_uint4(0, 0, 0, 0);
}

}  // namespace nsa
