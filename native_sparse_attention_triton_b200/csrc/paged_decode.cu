// Attention of one new token per sequence over a paged key-value cache, all of it or a sliding window and sinks.
//
// With L = seqlens[b] rows in the cache of sequence b (the new token's own row among them) row j is visible iff
//     j < L  and  (no window, or j >= L - 1 - window, or j < sinks),
// which is what the query at position L - 1 sees in the varlen form (sink_window_attention).  For every query head
//     o = sum_j p_j v_j,   p_j = 2^(x_j - m) / l,   x_j = scale log2(e) <q, k_j>,   m = max x_j,   l = sum_j 2^(x_j - m).
// Row j lies in page table[b][j / page], slot j % page.
//
// What bounds it is HBM: 4 D bytes of K and V per visible row and KV head against 4 D G flops, which 16 x 8 x 16 products of one warp
// (rows = the G query heads of a KV head) take with room to spare.  76 sequences of 1 to 8192 tokens, 32q/4kv, d = 128: 137 us, 5.4 TB/s (tiles
// with cp.async instead of TMA boxes: 182); one of 517 rows 13.4 us (12.8 without a look at whether what is written is finite), of 20 000 clocks 5000 until its tile is there, 6000 for it and the join in the
// CTA, 8500 for the join between CTAs.
//
// A sequence's rows are cut into tiles of 32; those with a visible row, of all (sequence, KV head) pairs, form one list, which is
// cut evenly over the CTAs and their warps whatever the lengths are: a warp walks a run of tiles that may end one pair and begin others.
// It fetches them into a ring of its own, keeps a running maximum and sum and writes a pair that lies in its run whole.  Parts of a pair
// are joined in the order of the list, within a CTA through shared memory and between CTAs through scratch, by the CTA that finishes
// last: the result does not depend on which one that is.
//
// The probabilities are rounded to 16 bits twice, p = hi + lo, for two products instead of one: their rounding (2^-9 in bf16, as much as
// the output's own) then costs nothing that can be seen, and the products are not what bounds the kernel.
#include "attn_tile.cuh"
#include "dispatch.h"
#include "host_util.h"
#include "nsa_b200.h"
#include "sink_exact.cuh"

#include <algorithm>
#include <cfloat>
#include <type_traits>

namespace nsa {

namespace {
constexpr int kPagedRows = 32;  // of a tile: one a lane
constexpr int kPagedStages = 3;
// Warps and shared memory of a CTA, one an SM: 192 KB of rings either way.
template <int D>
struct PagedShape {
  static constexpr int kWarps = D == 128 ? 4 : 8;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kTileBytes = kPagedRows * D * 2;           // of K, and of V
  static constexpr int kRing = kPagedStages * 2 * kTileBytes;     // of a warp
};
}  // namespace

struct PagedDecodeParams {
  const void* q;
  const void* k;
  const void* v;
  void* o;
  const int* table;
  const int* seqlens;
  float* logits;  // [pairs][G][logit_row] base-2 logits of a sequence's tiles, or nullptr
  float* lse;     // [pairs][G], with logits
  unsigned* ctrl;
  float* part;    // [CTAs][2][16][D + 2]
  long long q_sb, q_sh, k_sp, k_ss, k_sh, v_sp, v_ss, v_sh, o_sb, o_sh, t_sb;
  int B, Hkv, G, page, max_pages, num_pages, cap;
  int logit_row;      // rows of the tiles that a sequence may have
  int box;            // rows of a TMA box: they divide a page and a tile
  int window, sinks;  // window < 0: every row
  float scale2;
  Status st;
};

// Visible rows of a sequence, [0, head) and [first, len); its tiles, [0, gap_at) and [gap_at + gap, gap_at + gap + ...), n of them.
struct Rows {
  int len, head, first, n, gap_at, gap;
};
__device__ __forceinline__ Rows visible_rows(const PagedDecodeParams& p, int b) {
  constexpr int R = kPagedRows;
  Rows r;
  r.len = max(0, min(load_fresh(p.seqlens + b), p.cap));
  r.first = p.window < 0 ? 0 : max(0, r.len - 1 - p.window);
  r.head = min(p.sinks, r.first);
  r.gap_at = min((r.head + R - 1) / R, r.first / R);
  r.gap = r.first / R - r.gap_at;
  r.n = max(1, (r.len + R - 1) / R - r.gap);  // a sequence without rows has a tile of which none is visible
  return r;
}

// A position in the list of tiles.
struct TileCursor {
  int b, h, t;
  Rows rows;
  __device__ __forceinline__ int row0() const { return (t < rows.gap_at ? t : t + rows.gap) * kPagedRows; }
  __device__ __forceinline__ void next(const PagedDecodeParams& p) {
    if (++t < rows.n) return;
    t = 0;
    if (++h < p.Hkv) return;
    h = 0;
    if (++b < p.B) rows = visible_rows(p, b);
  }
};

// The tiles in front of every THREADS-th part of the batch, in `before`; returns those of the whole list.  The whole CTA.
template <int THREADS>
__device__ __forceinline__ unsigned count_tiles(const PagedDecodeParams& p, unsigned* before, unsigned* warp_sums) {
  const int per = (p.B + THREADS - 1) / THREADS, b0 = min(p.B, (int)threadIdx.x * per), b1 = min(p.B, b0 + per);
  unsigned sum = 0;
  for (int b = b0; b < b1; ++b) {
    sum += visible_rows(p, b).n;
    if (blockIdx.x == 0 && load_fresh(p.seqlens + b) > p.cap) p.st.raise(kErrBadIndex);  // more rows than its pages hold
  }
  sum *= p.Hkv;
  unsigned upto = sum;
#pragma unroll
  for (int s = 1; s < 32; s <<= 1) {
    const unsigned y = __shfl_up_sync(0xffffffffu, upto, s);
    if (lane_id() >= s) upto += y;
  }
  if (lane_id() == 31) warp_sums[threadIdx.x >> 5] = upto;
  __syncthreads();
  unsigned total = 0, front = upto - sum;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    const unsigned x = warp_sums[w];
    front += w < (int)(threadIdx.x >> 5) ? x : 0;
    total += x;
  }
  before[threadIdx.x] = front;
  __syncthreads();
  return total;
}

// The cursor of tile number x.  A whole warp.
template <int THREADS>
__device__ __forceinline__ TileCursor find_tile(const PagedDecodeParams& p, const unsigned* before, unsigned x) {
  const int per = (p.B + THREADS - 1) / THREADS, lane = lane_id();
  int part = -1;
#pragma unroll
  for (int k = 0; k < THREADS / 32; ++k) part += __popc(__ballot_sync(0xffffffffu, before[k * 32 + lane] <= x));
  TileCursor c;
  unsigned at = x - before[part];
  const int end = min(p.B, (part + 1) * per);
  for (int b0 = part * per;; b0 += 32) {
    const int b = b0 + lane;
    const unsigned mine = b < end ? visible_rows(p, b).n * p.Hkv : 0;
    unsigned upto = mine;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      const unsigned y = __shfl_up_sync(0xffffffffu, upto, s);
      if (lane >= s) upto += y;
    }
    const unsigned past = __ballot_sync(0xffffffffu, upto > at);
    if (past || b0 + 32 >= end) {
      const int src = past ? __ffs(past) - 1 : 31;
      at -= __shfl_sync(0xffffffffu, upto - mine, src);
      c.b = min(b0 + src, p.B - 1);
      c.rows = visible_rows(p, c.b);
      c.h = at / (unsigned)c.rows.n;
      c.t = at - (unsigned)c.h * c.rows.n;
      return c;
    }
    at -= __shfl_sync(0xffffffffu, upto, 31);
  }
}

// The list over n CTAs: the first `rest` take one tile more than the others.
struct Shares {
  unsigned each;
  int rest, n;
  __device__ __forceinline__ Shares(unsigned total, int n) : n(n) {
    each = total / (unsigned)n;
    rest = (int)(total - each * n);
  }
  __device__ __forceinline__ unsigned begin(int c) const { return c * each + min(c, rest); }
  // the CTA that has tile x; a whole warp
  __device__ __forceinline__ int owner(unsigned x) const {
    int c = -1;
    for (int k = lane_id(); k - lane_id() < n; k += 32) c += __popc(__ballot_sync(0xffffffffu, k < n && begin(k) <= x));
    return c;
  }
};

// A part of a pair's result: rows of [D] with their running maximum and sum.
template <int D>
struct Part {
  float o[16][D];
  float m[16], l[16];
};

// A pair and its tiles' place in the list.
struct PairSpan {
  int pair;  // -1: none
  unsigned start, stop;
};

// Output of query head h * G + g of sequence b by 32-bit probabilities over the rows it sees, from its maximum m and sum l; a warp.  A row whose
// tiles gave it a value that is not finite is computed again here: hi * inf + lo * inf is no number where lo is zero or below, nor is the product
// of infinity and a probability that 16 or 32 bits round to zero (row_probability: none is zero).  Some 100 clocks a
// row of the cache, which only those that hold such values pay.
template <typename T, int D>
__device__ __noinline__ void exact_decode_row(const PagedDecodeParams* p, int b, int h, int g, float m, float l) {
  const Rows rows = visible_rows(*p, b);
  const int head = h * p->G + g, lane = lane_id();
  float q[4], k[4], v[4], acc[4] = {0.f, 0.f, 0.f, 0.f};
  lane_elements<T, D>(q, p->q, (long long)b * p->q_sb + (long long)head * p->q_sh);
  for (int t = 0; t < rows.n; ++t) {
    const int j = (t < rows.gap_at ? t : t + rows.gap) * kPagedRows + lane;
    const bool in = j < rows.len && (j >= rows.first || j < rows.head);
    const int page = in ? load_fresh(p->table + (long long)b * p->t_sb + j / p->page) : -1;
    for (unsigned see = __ballot_sync(0xffffffffu, (unsigned)page < (unsigned)p->num_pages); see; see &= see - 1) {
      const int src = __ffs(see) - 1;
      const long long pg = __shfl_sync(0xffffffffu, page, src), slot = __shfl_sync(0xffffffffu, j % p->page, src);
      lane_elements<T, D>(k, p->k, pg * p->k_sp + slot * p->k_ss + (long long)h * p->k_sh);
      lane_elements<T, D>(v, p->v, pg * p->v_sp + slot * p->v_ss + (long long)h * p->v_sh);
      const float w = row_probability(warp_dot(q, k) * p->scale2 - m);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] = fmaf(w, v[e], acc[e]);
    }
  }
  const float inv = 1.f / l;
  __syncwarp();  // what the tiles gave has been written
  store_lane_elements<T, D>(static_cast<T*>(p->o) + (long long)b * p->o_sb + (long long)head * p->o_sh,
                            make_float4(acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv));
}

// 1 / sum and log-sum-exp of a row.  A sum of zero is one over nothing (its maximum is -infinity; outputs are zero), or over logits that are all
// -infinity (its maximum is kNothingYet): no number then, as where the sum itself is none.
constexpr float kNothingYet = -FLT_MAX;
__device__ __forceinline__ float inverse_sum(float m, float l) { return l != 0.f ? 1.f / l : m == -INFINITY ? 0.f : NAN; }
__device__ __forceinline__ float log_sum(float m, float l) { return l != 0.f ? m + log2f(l) : m == -INFINITY ? -INFINITY : NAN; }

// TMA: tiles come as boxes of p.box rows; else row by row with cp.async (pages whose size has no factor of 8).
template <typename T, int D, bool TMA>
__global__ void __launch_bounds__(PagedShape<D>::kThreads, 1)
paged_decode_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                    const __grid_constant__ PagedDecodeParams p) {
  constexpr int ROWS = kPagedRows, NT = ROWS / 8, CH = D / 8;  // 16-byte chunks of a row
  constexpr int WARPS = PagedShape<D>::kWarps, THREADS = WARPS * 32, TILE = PagedShape<D>::kTileBytes, RING = PagedShape<D>::kRing;
  extern __shared__ __align__(1024) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* ring = smem + warp * RING;
  Part<D>* head_parts = reinterpret_cast<Part<D>*>(smem + WARPS * RING);
  Part<D>* tail_part = reinterpret_cast<Part<D>*>(ring);  // once the ring is empty
  __shared__ uint64_t full_bars[WARPS * kPagedStages];
  __shared__ unsigned seen[WARPS * kPagedStages];
  __shared__ unsigned before[THREADS];
  __shared__ unsigned warp_sums[WARPS];
  __shared__ PairSpan parts[2 * WARPS];  // of each warp's first and of its last part
  __shared__ PairSpan open[2];           // the CTA's first and last part
  __shared__ int last_of[2], first_of[2];
  uint64_t* full = full_bars + warp * kPagedStages;
  unsigned* seen_sm = seen + warp * kPagedStages;

  wait_for_launch_before();
  // ---- this CTA's and this warp's run of tiles ----
  const unsigned total = count_tiles<THREADS>(p, before, warp_sums);
  const int nc = (int)min(gridDim.x, (total + WARPS - 1) / WARPS);  // CTAs with work
  const int cta = blockIdx.x;
  if (cta >= nc) return;
  const Shares shares(total, nc);
  const unsigned c_begin = shares.begin(cta), c_end = shares.begin(cta + 1);
  const int c_count = (int)(c_end - c_begin);
  const int w_begin = (int)((long long)warp * c_count / WARPS);
  const int count = (int)((warp + 1ll) * c_count / WARPS) - w_begin;
  if (smem_u32(smem) & 1023u) {  // the swizzled tiles need a 1024-byte aligned base
    if (threadIdx.x == 0) p.st.raise(kErrSmemLayout);
    return;
  }
  if (lane == 0) {
    parts[2 * warp].pair = parts[2 * warp + 1].pair = -1;
    if (TMA) {
      for (int s = 0; s < kPagedStages; ++s) mbar_init(full + s, 1);
      fence_barrier_init();
    }
  }
  if (threadIdx.x < 2) open[threadIdx.x].pair = -1;
  __syncwarp();
  if (count > 0) {
    TileCursor cur = find_tile<THREADS>(p, before, c_begin + w_begin), ld = cur;
    // pages of the tile that is loaded next, looked up a tile ahead
    int page_id, slot;
    bool in;
    auto look_up = [&](bool more) {
      const int j = ld.row0() + lane;
      in = more && j < ld.rows.len && (j >= ld.rows.first || j < ld.rows.head);
      const int pg = in ? j / p.page : 0;
      slot = j - pg * p.page;
      page_id = in ? load_fresh(p.table + (long long)ld.b * p.t_sb + pg) : -1;
    };
    auto fetch = [&](int i) {  // tile number i of the run into its stage
      const int s = i % kPagedStages;
      if (ld.t == 0 && lane * 64 < p.G * D) {  // a pair begins: its queries towards this SM
        const T* qb = static_cast<const T*>(p.q) + (long long)ld.b * p.q_sb + ((long long)ld.h * p.G + lane * 64 / D) * p.q_sh + lane * 64 % D;
        asm volatile("prefetch.global.L1 [%0];\n" ::"l"(qb));
      }
      uint8_t* ks = ring + s * 2 * TILE;
      const bool good = in && (unsigned)page_id < (unsigned)p.num_pages;
      if (in && !good) p.st.raise(kErrBadIndex);
      const unsigned see = __ballot_sync(0xffffffffu, good);
      if (lane == 0) seen_sm[s] = see;
      if (!good) page_id = -1;
      if constexpr (TMA) {
        // the lane at the first row of a box issues it, where any of its rows is visible (which says the page)
        const int at = lane & (p.box - 1);
        const unsigned mine = see >> (lane - at) & (0xffffffffu >> (32 - p.box));
        const int src = lane - at + (mine ? __ffs(mine) - 1 : 0);
        const int pg = __shfl_sync(0xffffffffu, page_id, src), sl = __shfl_sync(0xffffffffu, slot, src) - (src & (p.box - 1));
        const unsigned boxes = __ballot_sync(0xffffffffu, at == 0 && mine);
        if (lane == 0) {
          if (boxes) mbar_expect_tx(full + s, __popc(boxes) * p.box * D * 2 * 2);
          else mbar_arrive(full + s);
        }
        __syncwarp();
        if (at == 0 && mine) {
#pragma unroll
          for (int pn = 0; pn < D / 64; ++pn) {
            uint8_t* dst = ks + pn * ROWS * 128 + lane * 128;
            tma_load_4d(dst, &tmK, full + s, pn * 64, ld.h, sl, pg);
            tma_load_4d(dst + TILE, &tmV, full + s, pn * 64, ld.h, sl, pg);
          }
        }
      } else {
        const uint32_t kb_sm = smem_u32(ks), vb_sm = kb_sm + TILE;
        const T* kb = static_cast<const T*>(p.k) + (long long)ld.h * p.k_sh;
        const T* vb = static_cast<const T*>(p.v) + (long long)ld.h * p.v_sh;
#pragma unroll
        for (int c = 0; c < ROWS * CH / 32; ++c) {
          const int flat = c * 32 + lane;
          const int row = flat / CH, chunk = flat % CH;
          const int pg = __shfl_sync(0xffffffffu, page_id, row), sl = __shfl_sync(0xffffffffu, slot, row);
          const bool good = pg >= 0;
          const uint32_t off = swz_addr<ROWS>(0, row, chunk);
          cp_async16(kb_sm + off, good ? kb + (long long)pg * p.k_sp + (long long)sl * p.k_ss + chunk * 8 : kb, good);
          cp_async16(vb_sm + off, good ? vb + (long long)pg * p.v_sp + (long long)sl * p.v_ss + chunk * 8 : vb, good);
        }
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
      if (!TMA) cp_async_commit();
    }

    uint32_t qf[D / 16][4];
    float o[D / 8][4], m[2], l[2];
    bool fresh = true, first_seg = true;
    int seg_t0 = 0;  // first tile of the present pair in this run
    for (int i = 0; i < count; ++i) {
      if (i + kPagedStages - 1 < count) {
        fetch(i + kPagedStages - 1);
        ld.next(p);
        look_up(i + kPagedStages < count);
      }
      if (!TMA) cp_async_commit();
      if (fresh) {
        const T* qb = static_cast<const T*>(p.q) + (long long)cur.b * p.q_sb + (long long)cur.h * p.G * p.q_sh;
        load_a_frags_global<T, D / 16, /*FRESH=*/true>(qf, [&](int r) { return r < p.G ? qb + (long long)r * p.q_sh : (const T*)nullptr; });
#pragma unroll
        for (int j = 0; j < D / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
        m[0] = m[1] = -INFINITY;
        l[0] = l[1] = 0.f;
        seg_t0 = cur.t;
        fresh = false;
      }
      const int s = i % kPagedStages;
      if (TMA) mbar_wait(full + s, (i / kPagedStages) & 1, p.st);
      else cp_async_wait<kPagedStages - 1>();
      __syncwarp();
      const uint32_t ks = smem_u32(ring + s * 2 * TILE), vs = ks + TILE;
      const unsigned see = seen_sm[s];
      if (TMA && see != 0xffffffffu) {
        // rows that are not visible may hold anything, and 0 times that is not 0 where it is not finite
        if (!(see >> lane & 1u))
#pragma unroll
          for (int c = 0; c < CH; ++c)
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};\n" ::"r"(swz_addr<ROWS>(vs, lane, c)), "r"(0) : "memory");
        fence_proxy_async();  // TMA writes there again
        __syncwarp();
      }
      float x[NT][4];
#pragma unroll
      for (int j = 0; j < NT; ++j) x[j][0] = x[j][1] = x[j][2] = x[j][3] = 0.f;
      mma_nk<T, NT, D / 16, ROWS>(x, qf, ks, 0, 0);
      // ---- running maximum and sum; masked logits take no part ----
      const int c0 = (lane & 3) * 2;
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const unsigned bits = see >> (j * 8 + c0);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[j][e] = (bits >> (e & 1)) & 1u ? x[j][e] * p.scale2 : -INFINITY;
          mx[e >> 1] = fmaxf(mx[e >> 1], x[j][e]);
        }
      }
      if (p.logits) {
        const long long pair = (long long)cur.b * p.Hkv + cur.h;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int g = (lane >> 2) + half * 8;
          if (g < p.G) {
            float* dst = p.logits + (pair * p.G + g) * p.logit_row + cur.t * kPagedRows + c0;
#pragma unroll
            for (int j = 0; j < NT; ++j) *reinterpret_cast<float2*>(dst + j * 8) = make_float2(x[j][2 * half], x[j][2 * half + 1]);
          }
        }
      }
      float base[2], corr[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float top = fmaxf(fmaxf(m[r], see ? kNothingYet : -INFINITY), quad_max(mx[r]));
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
      l[0] = l[0] * corr[0] + sum[0];  // of this lane's columns
      l[1] = l[1] * corr[1] + sum[1];
      if (__any_sync(0xffffffffu, corr[0] != 1.f || corr[1] != 1.f)) {
#pragma unroll
        for (int j = 0; j < D / 8; ++j) {
          o[j][0] *= corr[0];
          o[j][1] *= corr[0];
          o[j][2] *= corr[1];
          o[j][3] *= corr[1];
        }
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
      const bool pair_ends = cur.t + 1 == cur.rows.n;
      if (pair_ends || i + 1 == count) {
        l[0] = quad_sum(l[0]);
        l[1] = quad_sum(l[1]);
        const int pair = cur.b * p.Hkv + cur.h;
        const int r0 = lane >> 2;
        if (pair_ends && seg_t0 == 0) {
          T* ob = static_cast<T*>(p.o) + (long long)cur.b * p.o_sb + (long long)cur.h * p.G * p.o_sh;
          const float inv[2] = {inverse_sum(m[0], l[0]), inverse_sum(m[1], l[1])};
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int g = r0 + half * 8;
            float zero = 0.f;  // 0 times each value
            if (g < p.G) {
              T* row = ob + (long long)g * p.o_sh + c0;
#pragma unroll
              for (int j = 0; j < D / 8; ++j) {
                zero = fmaf(o[j][2 * half + 1], 0.f, fmaf(o[j][2 * half], 0.f, zero));
                *reinterpret_cast<uint32_t*>(row + j * 8) = DT<T>::pack(o[j][2 * half] * inv[half], o[j][2 * half + 1] * inv[half]);
              }
              if (p.lse && (lane & 3) == 0) p.lse[(long long)pair * p.G + g] = log_sum(m[half], l[half]);
            }
            for (unsigned redo = __ballot_sync(0xffffffffu, l[half] > 0.f && zero != 0.f); redo;) {
              const int src = (__ffs(redo) - 1) & ~3;  // a row is four lanes'
              redo &= ~(15u << src);
              exact_decode_row<T, D>(&p, cur.b, cur.h, (src >> 2) + half * 8, __shfl_sync(0xffffffffu, m[half], src), __shfl_sync(0xffffffffu, l[half], src));
            }
          }
        } else {
          const bool tail = !first_seg;  // the run's last part: nothing is on its way into the ring
          Part<D>* dst = tail ? tail_part : head_parts + warp;
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
          if (lane == 0) {
            const unsigned start = c_begin + w_begin + i - cur.t;
            parts[2 * warp + tail] = PairSpan{pair, start, start + cur.rows.n};
          }
        }
        first_seg = false;
        fresh = true;
      }
      cur.next(p);
    }
    if (!TMA) cp_async_wait<0>();
  }
  __syncthreads();

  // ---- join the CTA's parts of each pair in order: a warp a pair, or a part of its rows where there are fewer pairs than warps ----
  constexpr int PART_FLOATS = 16 * (D + 2), EPL = D / 32, RY = 16 / WARPS;  // columns of a lane, rows at a time
  typedef typename std::conditional<EPL == 4, float4, float2>::type Cols;
  auto fma_cols = [](float (&a)[EPL], float w, Cols x) {
    const float* e = reinterpret_cast<const float*>(&x);
#pragma unroll
    for (int c = 0; c < EPL; ++c) a[c] = fmaf(w, e[c], a[c]);
  };
  auto write_row = [&](int pair, int g, const float (&val)[EPL], float mm, float ll) {
    const int b = pair / p.Hkv, h = pair - b * p.Hkv;
    const float inv = inverse_sum(mm, ll);
    uint32_t* row = reinterpret_cast<uint32_t*>(static_cast<T*>(p.o) + (long long)b * p.o_sb + (long long)(h * p.G + g) * p.o_sh + lane * EPL);
#pragma unroll
    for (int c = 0; c < EPL; c += 2) row[c / 2] = DT<T>::pack(val[c] * inv, val[c + 1] * inv);
    if (p.lse && lane == 0) p.lse[(long long)pair * p.G + g] = log_sum(mm, ll);
    float zero = 0.f;  // 0 times each value
#pragma unroll
    for (int c = 0; c < EPL; ++c) zero = fmaf(val[c], 0.f, zero);
    if (__any_sync(0xffffffffu, ll > 0.f && zero != 0.f)) exact_decode_row<T, D>(&p, b, h, g, mm, ll);
  };
  {
    auto part_at = [&](int i) { return (i & 1) ? reinterpret_cast<const Part<D>*>(smem + (i >> 1) * RING) : head_parts + (i >> 1); };
    const PairSpan mine = lane < 2 * WARPS ? parts[lane] : PairSpan{-1, 0, 0};
    const unsigned present = __ballot_sync(0xffffffffu, mine.pair >= 0), below = present & ((1u << lane) - 1u);
    const int prev = __shfl_sync(0xffffffffu, mine.pair, below ? 31 - __clz(below) : 0);
    const unsigned starts = __ballot_sync(0xffffffffu, mine.pair >= 0 && (!below || prev != mine.pair));
    const int pairs = __popc(starts);
    int slices = 1;
    if (pairs > 0)
      while (2 * slices * pairs <= WARPS) slices *= 2;
    const int per = (p.G + slices - 1) / slices;  // rows of a slice
    for (int item = warp; item < pairs * slices; item += WARPS) {
      unsigned from = starts;
      for (int k = item / slices; k; --k) from &= from - 1;
      const int a = __ffs(from) - 1;
      const unsigned later = from & (from - 1);
      const unsigned members = present & (0xffffffffu << a) & (later ? (later & -later) - 1u : 0xffffffffu);
      const PairSpan w{__shfl_sync(0xffffffffu, mine.pair, a), __shfl_sync(0xffffffffu, mine.start, a), __shfl_sync(0xffffffffu, mine.stop, a)};
      const bool whole = w.start >= c_begin && w.stop <= c_end;
      const int which = w.start < c_begin ? 0 : 1, slice = item % slices;
      float* out = p.part + ((long long)cta * 2 + which) * PART_FLOATS;
      // factors and sums of RY rows at a time, a lane a part and row; then their columns
      const int x = lane % (2 * WARPS);
      const bool has = members >> x & 1u;
      const Part<D>* own = part_at(has ? x : a);
      for (int g0 = slice * per; g0 < min(p.G, (slice + 1) * per); g0 += RY) {
        const int g = min(g0 + lane / (2 * WARPS), 15);
        const float pm = has ? own->m[g] : -INFINITY, pl = has ? own->l[g] : 0.f;
        float mm = pm;
#pragma unroll
        for (int s = WARPS; s; s >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, s));
        const float f = fast_exp2(pm - (mm == -INFINITY ? 0.f : mm));
        float ll = f * pl;
#pragma unroll
        for (int s = WARPS; s; s >>= 1) ll += __shfl_xor_sync(0xffffffffu, ll, s);
        alignas(16) float val[RY][EPL] = {};
        for (unsigned rem = members; rem; rem &= rem - 1) {
          const int y = __ffs(rem) - 1;
          const float* src = &part_at(y)->o[0][lane * EPL];
#pragma unroll
          for (int r = 0; r < RY; ++r)
            fma_cols(val[r], __shfl_sync(0xffffffffu, f, r * 2 * WARPS + y), *reinterpret_cast<const Cols*>(src + min(g0 + r, 15) * D));
        }
#pragma unroll
        for (int r = 0; r < RY; ++r) {
          const float m1 = __shfl_sync(0xffffffffu, mm, r * 2 * WARPS), l1 = __shfl_sync(0xffffffffu, ll, r * 2 * WARPS);
          if (g0 + r >= min(p.G, (slice + 1) * per)) continue;
          if (whole) {
            write_row(w.pair, g0 + r, val[r], m1, l1);
          } else {
            *reinterpret_cast<Cols*>(out + (g0 + r) * D + lane * EPL) = *reinterpret_cast<const Cols*>(val[r]);
            if (lane == 0) *reinterpret_cast<float2*>(out + 16 * D + 2 * (g0 + r)) = make_float2(m1, l1);
          }
        }
      }
      if (!whole && slice == 0 && lane == 0) open[which] = w;
    }
  }
  __syncthreads();

  // ---- what other CTAs have parts of: the last of them joins, 16 / WARPS rows a warp ----
  if (warp < 2) {
    const PairSpan w = open[warp];
    if (w.pair >= 0) {
      const int first = shares.owner(w.start), n = shares.owner(w.stop - 1) - first + 1;
      if (lane == 0) {  // (released and acquired by one thread: the CTA's barriers stand on either side)
        unsigned came;
        asm volatile("atom.acq_rel.gpu.global.inc.u32 %0, [%1], %2;\n" : "=r"(came) : "l"(p.ctrl + first), "r"((unsigned)(n - 1)) : "memory");
        last_of[warp] = came == (unsigned)(n - 1) ? n : 0;
        first_of[warp] = first;
      }
    } else if (lane == 0) {
      last_of[warp] = 0;
    }
  }
  __syncthreads();
  for (int x = 0; x < 2; ++x) {
    const int n = last_of[x];
    if (n == 0) continue;
    const int pair = open[x].pair, first = first_of[x];
    auto of = [&](int c) { return p.part + ((long long)(first + c) * 2 + (c == 0 ? 1 : 0)) * PART_FLOATS; };
    // four parts of RY rows on their way at a time
    float mm[RY], ll[RY], val[RY][EPL] = {};
#pragma unroll
    for (int r = 0; r < RY; ++r) mm[r] = -INFINITY, ll[r] = 0.f;
    for (int c0 = 0; c0 < n; c0 += 4) {
      float2 ml[4][RY];
      Cols o[4][RY];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float* src = of(min(c0 + c, n - 1));
#pragma unroll
        for (int r = 0; r < RY; ++r) {
          const int g = min(warp * RY + r, p.G - 1);
          ml[c][r] = load_fresh<kShared>(reinterpret_cast<const float2*>(src + 16 * D + 2 * g));
          o[c][r] = load_fresh<kShared>(reinterpret_cast<const Cols*>(src + g * D + lane * EPL));
        }
      }
#pragma unroll
      for (int r = 0; r < RY; ++r) {
        float now = mm[r];
#pragma unroll
        for (int c = 0; c < 4; ++c) now = fmaxf(now, ml[c][r].x);
        const float base = now == -INFINITY ? 0.f : now, old = fast_exp2(mm[r] - base);
        mm[r] = now;
        ll[r] *= old;
#pragma unroll
        for (int e = 0; e < EPL; ++e) val[r][e] *= old;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float f = c0 + c < n ? fast_exp2(ml[c][r].x - base) : 0.f;
          ll[r] = fmaf(f, ml[c][r].y, ll[r]);
          fma_cols(val[r], f, o[c][r]);
        }
      }
    }
#pragma unroll
    for (int r = 0; r < RY; ++r)
      if (warp * RY + r < p.G) write_row(pair, warp * RY + r, val[r], mm[r], ll[r]);
  }
}

constexpr int kWeightRows = 2;  // of a thread
// weights[b][h][j] += sum over the G heads of 2^(x_j - lse), row by row of the logits the attention kernel left: place u of a sequence's tiles.
__global__ void __launch_bounds__(256) paged_weights_kernel(PagedDecodeParams p, float* weights, long long w_sb, long long w_sh) {
  wait_for_launch_before();
  const int b = blockIdx.x / p.Hkv, h = blockIdx.x % p.Hkv;
  const Rows rows = visible_rows(p, b);
  if ((int)blockIdx.y * 256 * kWeightRows >= rows.n * kPagedRows) return;
  float* out = weights + b * w_sb + h * w_sh;
  const float* lse = p.lse + (long long)blockIdx.x * p.G;
  const int u0 = blockIdx.y * (256 * kWeightRows) + threadIdx.x;
  float sum[kWeightRows], old[kWeightRows];
  int at[kWeightRows];
  bool in[kWeightRows];
#pragma unroll
  for (int y = 0; y < kWeightRows; ++y) {
    const int u = u0 + y * 256, j = at[y] = u + (u / kPagedRows < rows.gap_at ? 0 : rows.gap * kPagedRows);
    in[y] = j < rows.len && (j < rows.head || j >= rows.first);
    old[y] = in[y] ? out[j] : 0.f;
    sum[y] = 0.f;
  }
  // The loads of four heads in front of their first use, of places that stand for no row too: no branch between them, and nothing is made of those.
  const float* logits = p.logits + (long long)blockIdx.x * p.G * p.logit_row;
  for (int g0 = 0; g0 < p.G; g0 += 4) {
    float ls[4], x[4][kWeightRows];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int head = min(g0 + g, p.G - 1);
      ls[g] = load_fresh(lse + head);
      if (g0 + g >= p.G) ls[g] = -INFINITY;
#pragma unroll
      for (int y = 0; y < kWeightRows; ++y) x[g][y] = load_fresh(logits + (long long)head * p.logit_row + min(u0 + y * 256, p.logit_row - 1));
    }
#pragma unroll
    for (int g = 0; g < 4; ++g)
#pragma unroll
      for (int y = 0; y < kWeightRows; ++y) sum[y] += ls[g] == -INFINITY ? 0.f : fast_exp2(x[g][y] - ls[g]);
  }
#pragma unroll
  for (int y = 0; y < kWeightRows; ++y)
    if (in[y]) out[at[y]] = old[y] + sum[y];
}

// Rows of the tiles that a sequence may have: those of its pages, and with a window no more than the window and the sinks reach into.
static long long most_logits(long long capacity, long long window, long long sinks) {
  const long long all = (capacity + kPagedRows - 1) / kPagedRows;
  // the window's rows begin anywhere in a tile
  const long long seen = window < 0 ? all : (window + 1 + kPagedRows - 1) / kPagedRows + 1 + (sinks + kPagedRows - 1) / kPagedRows;
  return std::max(1ll, std::min(all, seen)) * kPagedRows;
}

// One float of control per CTA, rounded up to whole lines; the parts behind them; with weights the logits and log-sum-exps.
static long long paged_ctrl_floats() { return (num_sms() + 63) / 64 * 64; }
static long long paged_part_floats(int D) { return (long long)num_sms() * 2 * 16 * (D + 2); }

template <typename T, int D>
static int launch_paged_decode(PagedDecodeParams p, float* weights, long long w_sb, long long w_sh, cudaStream_t stream) {
  constexpr int WARPS = PagedShape<D>::kWarps;
  const size_t smem = WARPS * (PagedShape<D>::kRing + sizeof(Part<D>));
  // the largest power of two that divides a page, at most 32
  p.box = std::min(32, p.page & -p.page);
  const bool tma = p.box >= 8;
  CUtensorMap tmK{}, tmV{};
  if (tma) {
    int rc = make_tmap_4d(&tmK, DT<T>::kTmapType, p.k, D, p.Hkv, p.page, p.num_pages, p.k_sh, p.k_ss, p.k_sp, 64, p.box, 1);
    if (!rc) rc = make_tmap_4d(&tmV, DT<T>::kTmapType, p.v, D, p.Hkv, p.page, p.num_pages, p.v_sh, p.v_ss, p.v_sp, 64, p.box, 1);
    if (rc) return rc;
  }
  auto kern = tma ? paged_decode_kernel<T, D, true> : paged_decode_kernel<T, D, false>;
  cudaError_t e = allow_smem(kern, smem);
  if (e != cudaSuccess) return cuda_rc(e);
  const long long most = (long long)p.B * p.Hkv * ((p.cap + kPagedRows - 1) / kPagedRows);
  const int grid = (int)std::min<long long>(num_sms(), (most + WARPS - 1) / WARPS);
  {
    LaunchScope ls_("paged_decode", stream);
    e = launch_early(kern, grid, WARPS * 32, smem, stream, tmK, tmV, p);
  }
  if (e != cudaSuccess || !weights) return cuda_rc(e);
  LaunchScope ls_("paged_weights", stream);
  return cuda_rc(launch_early(paged_weights_kernel, dim3(p.B * p.Hkv, (p.logit_row + 256 * kWeightRows - 1) / (256 * kWeightRows)), 256, 0, stream, p, weights, w_sb, w_sh));
}

}  // namespace nsa

extern "C" long long nsa_paged_decode_control_words(void) { return nsa::paged_ctrl_floats(); }

extern "C" long long nsa_paged_decode_window_scratch_floats(int batch, int num_q_heads, int head_dim, int capacity, int with_weights, int window_left,
                                                            int num_sinks) {
  const long long rows = with_weights ? nsa::most_logits(capacity, window_left, num_sinks) : 0;
  return nsa::paged_ctrl_floats() + nsa::paged_part_floats(head_dim) + (with_weights ? (long long)batch * num_q_heads * (rows + 1) + 64 : 0);
}

extern "C" long long nsa_paged_decode_scratch_floats(int batch, int num_q_heads, int head_dim, int capacity, int with_weights) {
  return nsa_paged_decode_window_scratch_floats(batch, num_q_heads, head_dim, capacity, with_weights, -1, 0);
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
  // tiles are counted in 32 bits
  if (cap > (1ll << 30) || (long long)batch * num_kv_heads > (1ll << 30) || (double)batch * num_kv_heads * (cap + 31) >= 0x1p36) return kUnsupported;
  if (num_q_heads / num_kv_heads > 16) return kUnsupported;
  const long long logit_row = most_logits(cap, window_left, num_sinks);
  if (weights && logit_row > 65535ll * 256 * kWeightRows) return kUnsupported;
  // strides: q_b q_h  k_page k_slot k_h  v_page v_slot v_h  o_b o_h  table_b  weights_b weights_h
  for (int i = 0; i < 10; ++i)
    if (strides[i] % 8) return kInvalid;
  if (!aligned16(q) || !aligned16(k_pages) || !aligned16(v_pages) || !aligned16(o)) return kInvalid;
  if (scratch_floats < nsa_paged_decode_window_scratch_floats(batch, num_q_heads, head_dim, (int)cap, weights != nullptr, window_left, num_sinks))
    return kWorkspace;
  PagedDecodeParams p;
  p.q = q; p.k = k_pages; p.v = v_pages; p.o = o; p.table = block_table; p.seqlens = seqlens;
  p.ctrl = reinterpret_cast<unsigned*>(scratch);
  p.part = scratch + paged_ctrl_floats();
  p.lse = weights ? p.part + paged_part_floats(head_dim) : nullptr;
  p.logits = weights ? p.lse + ((long long)batch * num_q_heads + 31) / 32 * 32 : nullptr;
  p.logit_row = (int)logit_row;
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
