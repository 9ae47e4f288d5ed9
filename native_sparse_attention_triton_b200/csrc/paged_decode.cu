// Attention of one new token per sequence over a paged key-value cache, all of it or a sliding window and sinks.
//
// With L = seqlens[b] rows in the cache of sequence b (the new token's own row among them) row j is visible iff
//     j < L  and  (no window, or j >= L - 1 - window, or j < sinks),
// which is what the query at position L - 1 sees in the varlen form (sink_window_attention).  For every query head
//     o = sum_j p_j v_j,   p_j = 2^(x_j - m) / l,   x_j = scale log2(e) <q, k_j>,   m = max x_j,   l = sum_j 2^(x_j - m).
// Row j lies in page table[b][j / page], slot j % page.  The visible rows are counted without the gap between the sinks and the
// window, so that neither costs a tile of masked keys.
//
// What bounds it is HBM: 4 D bytes of K and V per visible row and KV head against 4 D G flops, which 16 x 8 x 16 products of one warp
// (rows = the G query heads of a KV head) take with room to spare.
//
// The tiles of all (sequence, KV head) pairs form one list, which is cut evenly over the CTAs and their warps whatever the lengths are:
// a warp walks a run of tiles that may end one pair and begin others.  It gathers tiles of kTileRows rows with cp.async, a row's address
// from its page, into a ring of its own, keeps a running maximum and sum and writes a pair that lies in its run whole.  Parts of a pair
// are joined in the order of the list, within a CTA through shared memory and between CTAs through scratch, by the CTA that finishes
// last: the result does not depend on who that is.
//
// The probabilities are rounded to 16 bits twice, p = hi + lo, for two products instead of one: their rounding (2^-9 in bf16, as much as
// the output's own) then costs nothing that can be seen, and the products are not what bounds the kernel.
#include "attn_tile.cuh"
#include "dispatch.h"
#include "host_util.h"
#include "nsa_b200.h"

#include <algorithm>

namespace nsa {

namespace {
constexpr int kPagedWarps = 4;
constexpr int kPagedStages = 3;
constexpr int kPagedTileBytes = 32 * 128 * 2;  // of K, and of V: 32 rows of 128 elements or 64 of 64
}  // namespace

struct PagedDecodeParams {
  const void* q;
  const void* k;
  const void* v;
  void* o;
  const int* table;
  const int* seqlens;
  float* logits;  // [pairs][G][cap] base-2 logits by visible row, or nullptr
  float* lse;     // [pairs][G], with logits
  unsigned* ctrl;
  float* part;    // [CTAs][2][16][D + 2]
  long long q_sb, q_sh, k_sp, k_ss, k_sh, v_sp, v_ss, v_sh, o_sb, o_sh, t_sb;
  int B, Hkv, G, page, max_pages, num_pages, cap;
  int window, sinks;  // window < 0: every row
  float scale2;
  Status st;
};

// Visible rows of a sequence: [0, gap_at) and [gap_at + gap, gap + n).
struct Rows {
  int n, gap_at, gap;
};
__device__ __forceinline__ Rows visible_rows(int len, int window, int sinks, int cap) {
  Rows r;
  len = max(0, min(len, cap));
  const int first = window < 0 ? 0 : max(0, len - 1 - window);
  r.gap_at = min(sinks, first);
  r.gap = first - r.gap_at;
  r.n = len - r.gap;
  return r;
}

// A position in the list of tiles.
template <int ROWS>
struct TileCursor {
  int b, h, t, ntiles;
  Rows rows;
  __device__ __forceinline__ void load(const PagedDecodeParams& p) {
    rows = visible_rows(__ldg(p.seqlens + b), p.window, p.sinks, p.cap);
    ntiles = max(1, (rows.n + ROWS - 1) / ROWS);
  }
  __device__ __forceinline__ void next(const PagedDecodeParams& p) {
    if (++t < ntiles) return;
    t = 0;
    if (++h < p.Hkv) return;
    h = 0;
    if (++b < p.B) load(p);
  }
};

template <int ROWS>
__device__ __forceinline__ int tiles_of(const PagedDecodeParams& p, int b) {
  return max(1, (visible_rows(__ldg(p.seqlens + b), p.window, p.sinks, p.cap).n + ROWS - 1) / ROWS);
}

// Tiles of the whole list.  A whole warp.
template <int ROWS>
__device__ __forceinline__ long long count_tiles(const PagedDecodeParams& p) {
  long long sum = 0;
  for (int b = lane_id(); b < p.B; b += 32) {
    sum += tiles_of<ROWS>(p, b);
    if (blockIdx.x == 0 && __ldg(p.seqlens + b) > p.cap) p.st.raise(kErrBadIndex);  // more rows than its pages hold
  }
#pragma unroll
  for (int s = 16; s; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
  return sum * p.Hkv;
}

// The cursor of tile number x.  A whole warp.
template <int ROWS>
__device__ __forceinline__ TileCursor<ROWS> find_tile(const PagedDecodeParams& p, long long x) {
  TileCursor<ROWS> c;
  long long before = 0;
  for (int b0 = 0;; b0 += 32) {
    const int b = b0 + lane_id();
    const int mine = b < p.B ? tiles_of<ROWS>(p, b) : 0;
    long long upto = (long long)mine * p.Hkv;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, upto, s);
      if (lane_id() >= s) upto += y;
    }
    const unsigned past = __ballot_sync(0xffffffffu, before + upto > x);
    if (past || b0 + 32 >= p.B) {
      const int src = past ? __ffs(past) - 1 : 31;
      const long long start = before + __shfl_sync(0xffffffffu, upto, src) - (long long)__shfl_sync(0xffffffffu, mine, src) * p.Hkv;
      c.b = min(b0 + src, p.B - 1);
      c.load(p);
      const long long at = x - start;
      c.h = (int)(at / c.ntiles);
      c.t = (int)(at - (long long)c.h * c.ntiles);
      return c;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
}

// A part of a pair's result: rows of [D] with their running maximum and sum.
template <int D>
struct Part {
  float o[16][D];
  float m[16], l[16];
};

template <typename T, int D>
__global__ void __launch_bounds__(kPagedWarps * 32, 1) paged_decode_kernel(PagedDecodeParams p) {
  constexpr int ROWS = kPagedTileBytes / (D * 2);  // rows of a tile
  constexpr int NT = ROWS / 8;
  constexpr int RPL = ROWS / 32;                   // rows a lane knows the page of
  constexpr int CH = D / 8;                        // 16-byte chunks of a row
  extern __shared__ __align__(1024) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* ring = smem + warp * (kPagedStages * 2 * kPagedTileBytes);
  Part<D>* head_part = reinterpret_cast<Part<D>*>(smem + kPagedWarps * kPagedStages * 2 * kPagedTileBytes) + warp;
  Part<D>* tail_part = reinterpret_cast<Part<D>*>(ring);  // once the ring is empty
  unsigned* seen_sm = reinterpret_cast<unsigned*>(smem + kPagedWarps * (kPagedStages * 2 * kPagedTileBytes + sizeof(Part<D>))) +
                      warp * kPagedStages * RPL;
  // of every warp: pair of its first and of its last part (-1: none), what the CTA joins
  int* part_pair = reinterpret_cast<int*>(smem + kPagedWarps * (kPagedStages * 2 * kPagedTileBytes + sizeof(Part<D>)) +
                                          kPagedWarps * kPagedStages * RPL * 4);
  __shared__ int s_last;

  // ---- this CTA's and this warp's run of tiles ----
  const long long total = count_tiles<ROWS>(p);
  const int nc = (int)min((long long)gridDim.x, (total + kPagedWarps - 1) / kPagedWarps);  // CTAs with work
  const int cta = blockIdx.x;
  if (cta >= nc) return;
  const long long c_begin = cta * total / nc, c_end = (cta + 1) * total / nc;
  const long long begin = c_begin + warp * (c_end - c_begin) / kPagedWarps, end = c_begin + (warp + 1) * (c_end - c_begin) / kPagedWarps;
  const int count = (int)(end - begin);

  if (lane == 0) part_pair[2 * warp] = part_pair[2 * warp + 1] = -1;
  if (count > 0) {
    TileCursor<ROWS> cur = find_tile<ROWS>(p, begin), ld = cur;
    // pages of the tile that is loaded next, a tile ahead of its use
    int page_id[RPL], slot[RPL];
    unsigned ok[RPL];
    auto look_up = [&](bool more) {
#pragma unroll
      for (int r = 0; r < RPL; ++r) {
        const int u = ld.t * ROWS + r * 32 + lane;
        const bool in = more && u < ld.rows.n;
        const int j = u < ld.rows.gap_at ? u : u + ld.rows.gap;
        const int pg = in ? j / p.page : 0;
        slot[r] = j - pg * p.page;
        page_id[r] = in ? __ldg(p.table + (long long)ld.b * p.t_sb + pg) : -1;
        ok[r] = in;
      }
    };
    auto fetch = [&](int i) {  // tile number i of the run into its stage
      const int s = i % kPagedStages;
      const uint32_t ks = smem_u32(ring + s * 2 * kPagedTileBytes), vs = ks + kPagedTileBytes;
#pragma unroll
      for (int r = 0; r < RPL; ++r) {
        const bool good = ok[r] && (unsigned)page_id[r] < (unsigned)p.num_pages;
        if (ok[r] && !good) p.st.raise(kErrBadIndex);
        const unsigned see = __ballot_sync(0xffffffffu, good);
        if (lane == 0) seen_sm[s * RPL + r] = see;
        if (!good) page_id[r] = -1;
      }
      const T* kb = static_cast<const T*>(p.k) + (long long)ld.h * p.k_sh;
      const T* vb = static_cast<const T*>(p.v) + (long long)ld.h * p.v_sh;
#pragma unroll
      for (int c = 0; c < ROWS * CH / 32; ++c) {
        const int flat = c * 32 + lane;
        const int row = flat / CH, chunk = flat % CH;
        const int r = c * 32 / CH / 32;  // the same for all lanes
        const int pg = __shfl_sync(0xffffffffu, page_id[r], row & 31), sl = __shfl_sync(0xffffffffu, slot[r], row & 31);
        const bool good = pg >= 0;
        const uint32_t off = swz_addr<ROWS>(0, row, chunk);
        cp_async16(ks + off, good ? kb + (long long)pg * p.k_sp + (long long)sl * p.k_ss + chunk * 8 : kb, good);
        cp_async16(vs + off, good ? vb + (long long)pg * p.v_sp + (long long)sl * p.v_ss + chunk * 8 : vb, good);
      }
    };
    look_up(true);
#pragma unroll
    for (int i = 0; i < kPagedStages - 1; ++i) {
      if (i < count) {
        fetch(i);
        ld.next(p);
        look_up(i + 1 < count);
      }
      cp_async_commit();
    }

    uint32_t qf[D / 16][4];
    float o[D / 8][4], m[2], l[2];
    bool fresh = true;
    int seg_t0 = 0;  // first tile of the present pair in this run
    bool first_seg = true;
    for (int i = 0; i < count; ++i) {
      if (i + kPagedStages - 1 < count) {
        fetch(i + kPagedStages - 1);
        ld.next(p);
        look_up(i + kPagedStages < count);
      }
      cp_async_commit();
      if (fresh) {
        const T* qb = static_cast<const T*>(p.q) + (long long)cur.b * p.q_sb + (long long)cur.h * p.G * p.q_sh;
        load_a_frags_global<T, D / 16>(qf, [&](int r) { return r < p.G ? qb + (long long)r * p.q_sh : (const T*)nullptr; });
#pragma unroll
        for (int j = 0; j < D / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
        m[0] = m[1] = -INFINITY;
        l[0] = l[1] = 0.f;
        seg_t0 = cur.t;
        fresh = false;
      }
      cp_async_wait<kPagedStages - 1>();
      __syncwarp();
      const int s = i % kPagedStages;
      const uint32_t ks = smem_u32(ring + s * 2 * kPagedTileBytes), vs = ks + kPagedTileBytes;
      float x[NT][4];
#pragma unroll
      for (int j = 0; j < NT; ++j) x[j][0] = x[j][1] = x[j][2] = x[j][3] = 0.f;
      mma_nk<T, NT, D / 16, ROWS>(x, qf, ks, 0, 0);
      // ---- running maximum and sum; masked logits take no part ----
      const int c0 = (lane & 3) * 2;
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const unsigned see = seen_sm[s * RPL + j / 4] >> ((j & 3) * 8 + c0);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[j][e] = (see >> (e & 1)) & 1u ? x[j][e] * p.scale2 : -INFINITY;
          mx[e >> 1] = fmaxf(mx[e >> 1], x[j][e]);
        }
      }
      if (p.logits) {
        const long long pair = (long long)cur.b * p.Hkv + cur.h;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int g = (lane >> 2) + half * 8;
          if (g < p.G) {
            float* dst = p.logits + (pair * p.G + g) * p.cap + cur.t * ROWS;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              const int u = cur.t * ROWS + j * 8 + c0;
              if (u < cur.rows.n) dst[j * 8 + c0] = x[j][2 * half];
              if (u + 1 < cur.rows.n) dst[j * 8 + c0 + 1] = x[j][2 * half + 1];
            }
          }
        }
      }
      float base[2], corr[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float top = fmaxf(m[r], quad_max(mx[r]));
        base[r] = top == -INFINITY ? 0.f : top;
        corr[r] = fast_exp2(m[r] - base[r]);
        m[r] = top;
      }
      float sum[2] = {0.f, 0.f};
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[j][e] = fast_exp2(x[j][e] - base[e >> 1]);
          sum[e >> 1] += x[j][e];
        }
      l[0] = l[0] * corr[0] + quad_sum(sum[0]);
      l[1] = l[1] * corr[1] + quad_sum(sum[1]);
#pragma unroll
      for (int j = 0; j < D / 8; ++j) {
        o[j][0] *= corr[0];
        o[j][1] *= corr[0];
        o[j][2] *= corr[1];
        o[j][3] *= corr[1];
      }
      uint32_t hi[NT / 2][4], lo[NT / 2][4];
#pragma unroll
      for (int kk = 0; kk < NT / 2; ++kk)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float a = x[2 * kk + (e >> 1)][(e & 1) * 2], b = x[2 * kk + (e >> 1)][(e & 1) * 2 + 1];
          hi[kk][e] = DT<T>::pack(a, b);
          const float2 r = DT<T>::unpack(hi[kk][e]);
          lo[kk][e] = DT<T>::pack(a - r.x, b - r.y);
        }
      // o += (hi + lo) v
      {
        const int row_in = (lane & 7) + (((lane >> 3) & 1) << 3), ch_in = lane >> 4;
#pragma unroll
        for (int kk = 0; kk < NT / 2; ++kk)
#pragma unroll
          for (int jp = 0; jp < D / 16; ++jp) {
            uint32_t b[4];
            ldmatrix_x4_trans(b, swz_addr<ROWS>(vs, kk * 16 + row_in, 2 * jp + ch_in));
            DT<T>::mma(o[2 * jp], hi[kk], b[0], b[1]);
            DT<T>::mma(o[2 * jp + 1], hi[kk], b[2], b[3]);
            DT<T>::mma(o[2 * jp], lo[kk], b[0], b[1]);
            DT<T>::mma(o[2 * jp + 1], lo[kk], b[2], b[3]);
          }
      }
      __syncwarp();  // the stage has been read
      // ---- the end of the pair or of the run ----
      const bool pair_ends = cur.t + 1 == cur.ntiles;
      if (pair_ends || i + 1 == count) {
        const int pair = cur.b * p.Hkv + cur.h;
        const int r0 = lane >> 2;
        if (pair_ends && seg_t0 == 0) {
          T* ob = static_cast<T*>(p.o) + (long long)cur.b * p.o_sb + (long long)cur.h * p.G * p.o_sh;
          const float inv[2] = {l[0] > 0.f ? 1.f / l[0] : 0.f, l[1] > 0.f ? 1.f / l[1] : 0.f};
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int g = r0 + half * 8;
            if (g < p.G) {
              T* row = ob + (long long)g * p.o_sh + c0;
#pragma unroll
              for (int j = 0; j < D / 8; ++j)
                *reinterpret_cast<uint32_t*>(row + j * 8) = DT<T>::pack(o[j][2 * half] * inv[half], o[j][2 * half + 1] * inv[half]);
              if (p.lse && (lane & 3) == 0) p.lse[(long long)pair * p.G + g] = l[half] > 0.f ? m[half] + log2f(l[half]) : -INFINITY;
            }
          }
        } else {
          const bool tail = !first_seg;  // the run's last part, and its ring is empty
          if (tail) {
            cp_async_wait<0>();
            __syncwarp();
          }
          Part<D>* dst = tail ? tail_part : head_part;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int g = r0 + half * 8;
#pragma unroll
            for (int j = 0; j < D / 8; ++j) *reinterpret_cast<float2*>(&dst->o[g][j * 8 + c0]) = make_float2(o[j][2 * half], o[j][2 * half + 1]);
            if ((lane & 3) == 0) {
              dst->m[g] = m[half];
              dst->l[g] = l[half];
            }
          }
          if (lane == 0) part_pair[2 * warp + tail] = pair;
        }
        first_seg = false;
        fresh = true;
      }
      cur.next(p);
    }
    cp_async_wait<0>();
  }
  __syncthreads();

  // ---- join the parts: first the CTA's, in order, then those of other CTAs ----
  auto part_at = [&](int i) -> Part<D>* {
    return (i & 1) ? reinterpret_cast<Part<D>*>(smem + (i >> 1) * (kPagedStages * 2 * kPagedTileBytes))
                   : reinterpret_cast<Part<D>*>(smem + kPagedWarps * kPagedStages * 2 * kPagedTileBytes) + (i >> 1);
  };
  auto write_row = [&](int pair, int g, int col, float val, float mm, float ll) {
    const int b = pair / p.Hkv, h = pair - b * p.Hkv;
    T* ob = static_cast<T*>(p.o) + (long long)b * p.o_sb + (long long)(h * p.G + g) * p.o_sh;
    ob[col] = DT<T>::from_float(ll > 0.f ? val / ll : 0.f);
    if (p.lse && col == 0) p.lse[(long long)pair * p.G + g] = ll > 0.f ? mm + log2f(ll) : -INFINITY;
  };
  constexpr int PART_FLOATS = 16 * (D + 2);
  for (int i = 0; i < 2 * kPagedWarps;) {
    const int pair = part_pair[i];
    if (pair < 0) {
      ++i;
      continue;
    }
    int e = i + 1;  // parts [i, e) of the pair
    while (e < 2 * kPagedWarps && (part_pair[e] == pair || part_pair[e] < 0)) ++e;
    // where the pair's tiles lie in the list
    TileCursor<ROWS> at;
    long long start = 0;
    {
      const int b = pair / p.Hkv;
      for (int x = lane; x < b; x += 32) start += tiles_of<ROWS>(p, x);
#pragma unroll
      for (int s = 16; s; s >>= 1) start += __shfl_xor_sync(0xffffffffu, start, s);
      at.b = b;
      at.load(p);
      start = start * p.Hkv + (long long)(pair - b * p.Hkv) * at.ntiles;
    }
    const long long stop = start + at.ntiles;
    const bool whole = start >= c_begin && stop <= c_end;
    float* mine = p.part + ((long long)cta * 2 + (start < c_begin ? 0 : 1)) * PART_FLOATS;
    for (int f = threadIdx.x; f < p.G * D; f += kPagedWarps * 32) {
      const int g = f / D, col = f % D;
      float mm = -INFINITY;
      for (int x = i; x < e; ++x)
        if (part_pair[x] == pair) mm = fmaxf(mm, part_at(x)->m[g]);
      const float base = mm == -INFINITY ? 0.f : mm;
      float val = 0.f, ll = 0.f;
      for (int x = i; x < e; ++x)
        if (part_pair[x] == pair) {
          const float w = fast_exp2(part_at(x)->m[g] - base);
          val += w * part_at(x)->o[g][col];
          ll += w * part_at(x)->l[g];
        }
      if (whole) {
        write_row(pair, g, col, val, mm, ll);
      } else {
        mine[g * D + col] = val;
        if (col == 0) {
          mine[16 * D + g] = mm;
          mine[16 * D + 16 + g] = ll;
        }
      }
    }
    if (!whole) {
      const int first = (int)(((start + 1) * nc - 1) / total), last = (int)((stop * nc - 1) / total);  // CTAs that hold some of it
      __threadfence();
      __syncthreads();
      if (threadIdx.x == 0) s_last = atomicInc(p.ctrl + first, (unsigned)(last - first)) == (unsigned)(last - first);
      __syncthreads();
      if (s_last) {
        __threadfence();
        for (int f = threadIdx.x; f < p.G * D; f += kPagedWarps * 32) {
          const int g = f / D, col = f % D;
          auto of = [&](int c) { return p.part + ((long long)c * 2 + (c == first ? 1 : 0)) * PART_FLOATS; };
          float mm = -INFINITY;
          for (int c = first; c <= last; ++c) mm = fmaxf(mm, __ldcg(of(c) + 16 * D + g));
          const float base = mm == -INFINITY ? 0.f : mm;
          float val = 0.f, ll = 0.f;
          for (int c = first; c <= last; ++c) {
            const float w = fast_exp2(__ldcg(of(c) + 16 * D + g) - base);
            val += w * __ldcg(of(c) + g * D + col);
            ll += w * __ldcg(of(c) + 16 * D + 16 + g);
          }
          write_row(pair, g, col, val, mm, ll);
        }
      }
      __syncthreads();
    }
    i = e;
  }
}

// weights[b][h][j] += sum over the G heads of 2^(x_j - lse), row by row of the logits the attention kernel left.
__global__ void __launch_bounds__(256) paged_weights_kernel(PagedDecodeParams p, float* weights, long long w_sb, long long w_sh) {
  const int b = blockIdx.x / p.Hkv, h = blockIdx.x % p.Hkv;
  const Rows rows = visible_rows(__ldg(p.seqlens + b), p.window, p.sinks, p.cap);
  const int u = blockIdx.y * 256 + threadIdx.x;
  if (u >= rows.n) return;
  const float* x = p.logits + (long long)blockIdx.x * p.G * p.cap + u;
  const float* lse = p.lse + (long long)blockIdx.x * p.G;
  float sum = 0.f;
  for (int g = 0; g < p.G; ++g) {
    const float ls = __ldg(lse + g);
    sum += ls == -INFINITY ? 0.f : fast_exp2(__ldg(x + (long long)g * p.cap) - ls);
  }
  const int j = u < rows.gap_at ? u : u + rows.gap;
  weights[b * w_sb + h * w_sh + j] += sum;
}

// One float of control per CTA, rounded up to whole lines; the parts behind them; with weights the logits and log-sum-exps.
static long long paged_ctrl_floats() { return (num_sms() + 63) / 64 * 64; }
static long long paged_part_floats(int D) { return (long long)num_sms() * 2 * 16 * (D + 2); }

template <typename T, int D>
static int launch_paged_decode(PagedDecodeParams p, float* weights, long long w_sb, long long w_sh, cudaStream_t stream) {
  constexpr int ROWS = kPagedTileBytes / (D * 2);
  const size_t smem = kPagedWarps * (kPagedStages * 2 * kPagedTileBytes + sizeof(Part<D>)) + kPagedWarps * kPagedStages * (ROWS / 32) * 4 +
                      2 * kPagedWarps * sizeof(int);
  auto kern = paged_decode_kernel<T, D>;
  cudaError_t e = allow_smem(kern, smem);
  if (e != cudaSuccess) return cuda_rc(e);
  const long long most = (long long)p.B * p.Hkv * std::max(1, (p.cap + ROWS - 1) / ROWS);
  const int grid = (int)std::min<long long>(num_sms(), (most + kPagedWarps - 1) / kPagedWarps);
  { LaunchScope ls_("paged_decode", stream); kern<<<grid, kPagedWarps * 32, smem, stream>>>(p); }
  e = cudaGetLastError();
  if (e != cudaSuccess || !weights) return cuda_rc(e);
  { LaunchScope ls_("paged_weights", stream); paged_weights_kernel<<<dim3(p.B * p.Hkv, (p.cap + 255) / 256), 256, 0, stream>>>(p, weights, w_sb, w_sh); }
  return cuda_rc(cudaGetLastError());
}

}  // namespace nsa

extern "C" long long nsa_paged_decode_control_words(void) { return nsa::paged_ctrl_floats(); }

extern "C" long long nsa_paged_decode_scratch_floats(int batch, int num_q_heads, int head_dim, int capacity, int with_weights) {
  return nsa::paged_ctrl_floats() + nsa::paged_part_floats(head_dim) + (with_weights ? (long long)batch * num_q_heads * (capacity + 1ll) : 0);
}

extern "C" int nsa_paged_attn_decode(const void* q, const void* k_pages, const void* v_pages, const int* block_table, const int* seqlens, void* o,
                                     float* weights, float* scratch, long long scratch_floats, int batch, int num_q_heads, int num_kv_heads,
                                     int head_dim, int num_pages, int page_size, int max_pages, int window_left, int num_sinks,
                                     const long long* strides, float sm_scale, int dtype, void* stream) {
  using namespace nsa;
  if (!q || !k_pages || !v_pages || !block_table || !seqlens || !o || !scratch || !strides) return kInvalid;
  if (batch <= 0 || num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads) return kInvalid;
  if (num_pages <= 0 || page_size <= 0 || max_pages <= 0 || num_sinks < 0) return kInvalid;
  const long long cap = (long long)page_size * max_pages;
  if (cap > (1ll << 30) || (long long)batch * num_kv_heads > (1ll << 30)) return kUnsupported;
  if (num_q_heads / num_kv_heads > 16) return kUnsupported;
  if (weights && cap > 65535 * 256) return kUnsupported;
  // strides: q_b q_h  k_page k_slot k_h  v_page v_slot v_h  o_b o_h  table_b  weights_b weights_h
  for (int i = 0; i < 10; ++i)
    if (strides[i] % 8) return kInvalid;
  if (!aligned16(q) || !aligned16(k_pages) || !aligned16(v_pages) || !aligned16(o)) return kInvalid;
  if (scratch_floats < nsa_paged_decode_scratch_floats(batch, num_q_heads, head_dim, (int)cap, weights != nullptr)) return kWorkspace;
  PagedDecodeParams p;
  p.q = q; p.k = k_pages; p.v = v_pages; p.o = o; p.table = block_table; p.seqlens = seqlens;
  p.ctrl = reinterpret_cast<unsigned*>(scratch);
  p.part = scratch + paged_ctrl_floats();
  p.lse = weights ? p.part + paged_part_floats(head_dim) : nullptr;
  p.logits = weights ? p.lse + (long long)batch * num_q_heads : nullptr;
  p.q_sb = strides[0]; p.q_sh = strides[1];
  p.k_sp = strides[2]; p.k_ss = strides[3]; p.k_sh = strides[4];
  p.v_sp = strides[5]; p.v_ss = strides[6]; p.v_sh = strides[7];
  p.o_sb = strides[8]; p.o_sh = strides[9]; p.t_sb = strides[10];
  p.B = batch; p.Hkv = num_kv_heads; p.G = num_q_heads / num_kv_heads;
  p.page = page_size; p.max_pages = max_pages; p.num_pages = num_pages; p.cap = (int)cap;
  p.window = window_left; p.sinks = num_sinks;
  p.scale2 = sm_scale * kLog2e;
  p.st.word = status_word();
  return NSA_DISPATCH_T_D(dtype, head_dim, launch_paged_decode, p, weights, strides[11], strides[12], static_cast<cudaStream_t>(stream));
}
