// The paged key-value cache's own kernels: rows written behind those that a sequence holds, and a sequence cut down to the rows that
// attention has used most.
//
// Row j of sequence b is slot j % page of page table[b][j / page]; a page holds the rows of all KV heads.  Both operators move bytes and
// are bound by HBM (long inputs) or by one chain of dependent loads (length, page, row).  16 384 rows of 8 heads, d = 128: append 22.9 us, 5.9 TB/s.
//
// Eviction, for every (sequence, KV head) with L > budget rows: kept are the first `sinks` rows, the last `recent` ones, and of those
// between the r = budget - sinks - recent with the largest weights, equal ones by the lower row; a weight that is no number counts as
// the smallest.  The kept rows go, in their order, to the first `budget` rows of other pages.  `evict_select` finds the r-th largest
// weight by a radix selection on the bits of the weights, eleven at a time, then numbers the kept rows; `evict_move` copies them.  32 sequences of 1100 to 4107 rows
// cut to 1024, 8 heads: 16 and 44 us; one of 4160 rows to 4096: 16 us for both.
#include "dispatch.h"
#include "host_util.h"
#include "nsa_b200.h"

#include "common.cuh"

#include <algorithm>

namespace nsa {

struct PagedAppendParams {
  const void* k;
  const void* v;
  void* kp;
  void* vp;
  const int* table;
  const int* held;
  const int* cu;  // nullptr: one row per sequence
  int* after;
  long long k_sn, k_sh, v_sn, v_sh, kp_sp, kp_ss, kp_sh, vp_sp, vp_ss, vp_sh, t_sb;
  int N, B, Hkv, page, cap, num_pages;
  Status st;
};

// A warp per row: its sequence, page and slot once, then 16 bytes of K and of V a lane and step.
template <int D>
__global__ void __launch_bounds__(256) paged_append_kernel(PagedAppendParams p) {
  constexpr int CH = D / 8;
  const int lane = lane_id();
  wait_for_launch_before();
  for (int b = blockIdx.x * 256 + threadIdx.x; b < p.B; b += gridDim.x * 256)
    p.after[b] = (int)min((long long)p.cap, (long long)load_fresh(p.held + b) + (p.cu ? (long long)load_fresh(p.cu + b + 1) - load_fresh(p.cu + b) : 1));
  const int n = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (n >= (p.cu ? min(p.N, load_fresh(p.cu + p.B)) : p.N)) return;  // rows behind the last sequence are nobody's
  const int b = p.cu ? find_sequence(p.cu, p.B, n) : n;
  const long long at = (long long)load_fresh(p.held + b) + (p.cu ? n - load_fresh(p.cu + b) : 0);
  const int pos = at >= 0 && at < p.cap ? (int)at : -1;
  const int pg = pos >= 0 ? load_fresh(p.table + b * p.t_sb + pos / p.page) : -1;
  if ((unsigned)pg >= (unsigned)p.num_pages) {
    if (lane == 0) p.st.raise(kErrBadIndex);
    return;
  }
  const int slot = pos % p.page;
  typedef const unsigned short* Src;  // 16-bit elements of either type
  typedef unsigned short* Dst;
  const Src k = static_cast<Src>(p.k) + n * p.k_sn, v = static_cast<Src>(p.v) + n * p.v_sn;
  const Dst kp = static_cast<Dst>(p.kp) + pg * p.kp_sp + slot * p.kp_ss, vp = static_cast<Dst>(p.vp) + pg * p.vp_sp + slot * p.vp_ss;
  const int chunks = p.Hkv * CH;
  for (int c0 = lane; c0 < chunks; c0 += 4 * 32) {
    uint4 kr[4], vr[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int c = c0 + 32 * x, h = c / CH, e = c % CH * 8;
      if (c < chunks) {
        kr[x] = load_fresh(reinterpret_cast<const uint4*>(k + h * p.k_sh + e));
        vr[x] = load_fresh(reinterpret_cast<const uint4*>(v + h * p.v_sh + e));
      }
    }
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int c = c0 + 32 * x, h = c / CH, e = c % CH * 8;
      if (c < chunks) {
        *reinterpret_cast<uint4*>(kp + h * p.kp_sh + e) = kr[x];
        *reinterpret_cast<uint4*>(vp + h * p.vp_sh + e) = vr[x];
      }
    }
  }
}

struct PagedEvictParams {
  const float* w;   // [B][Hkv][...]
  float* w_out;     // [B][Hkv][w_cols], contiguous
  int* kept;        // [B][Hkv][budget], contiguous
  int* after;       // [B]
  void* kp;
  void* vp;
  const int* table;
  const int* target;
  const int* seqlens;
  long long w_sb, w_sh, kp_sp, kp_ss, kp_sh, vp_sp, vp_ss, vp_sh, t_sb, n_sb;
  int B, Hkv, page, cap, num_pages, w_cols, budget, sinks, recent;
  Status st;
};

constexpr int kSelectThreads = 512;
constexpr int kSelectItems = 16;  // rows a thread holds in registers
constexpr int kBins = 2048;

// Larger weights have larger keys; both zeros the same one.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(w + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Exclusive sum over the block's threads; `total` gets the sum of all.  `sums`: a word a warp, free again after the next barrier.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* sums, uint32_t& total) {
  const int lane = lane_id(), warp = threadIdx.x >> 5;
  uint32_t up = v;
#pragma unroll
  for (int s = 1; s < 32; s <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, up, s);
    if (lane >= s) up += y;
  }
  if (lane == 31) sums[warp] = up;
  __syncthreads();
  uint32_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kSelectThreads / 32; ++w) {
    const uint32_t x = sums[w];
    before += w < warp ? x : 0;
    total += x;
  }
  return before + up - v;
}

// A CTA per (sequence, KV head).  A warp holds neighbouring rows, 32 at a time, so that votes and one scan over the warps number them and what is
// written lies together; up to 8192 rows stay in registers, longer sequences are read again for every pass, 8192 rows at a time.  Digits of
// 11, 11 and 10 bits: the first (sign, exponent and two bits) spreads weights over enough bins that the atomics on shared memory do not queue.
// What bounds it is the chain of its passes.
__global__ void __launch_bounds__(kSelectThreads) evict_select_kernel(PagedEvictParams p) {
  __shared__ unsigned hist[kBins];
  __shared__ uint32_t sums[4][kSelectThreads / 32];
  __shared__ uint32_t s_digit, s_rank;
  const int b = blockIdx.x / p.Hkv, h = blockIdx.x % p.Hkv, tid = threadIdx.x;
  wait_for_launch_before();
  const int len = load_fresh(p.seqlens + b), L = max(0, min(len, p.cap)), m = min(L, p.budget);
  if (len > p.cap && tid == 0) p.st.raise(kErrBadIndex);
  const float* w = p.w + b * p.w_sb + h * p.w_sh;
  float* w_out = p.w_out + (long long)blockIdx.x * p.w_cols;
  int* kept = p.kept + (long long)blockIdx.x * p.budget;
  if (h == 0 && tid == 0) p.after[b] = m;
  for (int i = m + tid; i < p.w_cols; i += kSelectThreads) w_out[i] = 0.f;
  for (int i = m + tid; i < p.budget; i += kSelectThreads) kept[i] = -1;
  if (L <= p.budget) {
    for (int i = tid; i < m; i += kSelectThreads) {
      kept[i] = i;
      w_out[i] = load_fresh(w + i);
    }
    return;
  }
  // this thread's rows of a span: base + first + 32 j for j < per
  constexpr int kSpan = kSelectThreads * kSelectItems;
  const int per = min(kSelectItems, (L + kSelectThreads - 1) / kSelectThreads), span = per * kSelectThreads;
  const int lane = lane_id(), warp = tid >> 5, first = warp * per * 32 + lane;
  const int lo = p.sinks, hi = L - p.recent;
  float x[kSelectItems];
  uint32_t within, between;  // which of them are rows, and which of those are neither sinks nor recent
  auto load = [&](int base) {
    within = between = 0;
#pragma unroll
    for (int j = 0; j < kSelectItems; ++j) {
      const int i = base + first + 32 * j;
      const bool in = j < per && i < L;
      x[j] = in ? load_fresh(w + i) : 0.f;
      within |= (in ? 1u : 0u) << j;
      between |= (in && i >= lo && i < hi ? 1u : 0u) << j;
    }
  };
  load(0);
  // ---- the key of the r-th largest weight between the sinks and the recent rows, and how many of its equals are kept ----
  int rank = p.budget - p.sinks - p.recent;  // below the number of rows between
  uint32_t found = 0xffffffffu;              // above every key
  if (rank > 0) {
    found = 0;
    uint32_t mask = 0;
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
      const uint32_t digit = pass == 2 ? 1023u : 2047u;
      for (int i = tid; i < kBins; i += kSelectThreads) hist[i] = 0;
      __syncthreads();
      for (int base = 0; base < L; base += span) {
        if (L > kSpan) load(base);
#pragma unroll
        for (int j = 0; j < kSelectItems; ++j) {
          if (j >= per) break;
          const uint32_t key = weight_key(x[j]);
          if ((between >> j & 1u) && (key & mask) == found) atomicAdd(hist + (key >> shift & digit), 1u);
        }
      }
      __syncthreads();
      // the digit at which the counts from the top pass the rank; a thread has four neighbouring ones, the largest first
      uint32_t own = 0, total;
#pragma unroll
      for (int y = 0; y < kBins / kSelectThreads; ++y) own += hist[kBins - 1 - tid * (kBins / kSelectThreads) - y];
      const uint32_t front = block_scan(own, sums[pass], total);
      if (front < (uint32_t)rank && front + own >= (uint32_t)rank) {
        uint32_t left = rank - front;
        int at = kBins - 1 - tid * (kBins / kSelectThreads);
        while (hist[at] < left) left -= hist[at--];
        s_digit = at;
        s_rank = left;
      }
      __syncthreads();
      found |= s_digit << shift;
      mask |= digit << shift;
      rank = s_rank;
    }
  }
  // ---- the kept rows in their order: the sure ones, and of the last key's equals those within the rank ----
  int taken = 0, equals = 0;
  for (int base = 0; base < L; base += span) {
    if (L > kSpan) load(base);
    uint32_t sure = 0, equal = 0;
#pragma unroll
    for (int j = 0; j < kSelectItems; ++j) {
      const uint32_t key = weight_key(x[j]), bit = 1u << j;
      if ((within & bit) && (!(between & bit) || key > found)) sure |= bit;
      if ((between & bit) && key == found && rank > 0) equal |= bit;
    }
    // of the warps in front: sure ones, and equals in the upper half (at most 8192 each)
    uint32_t total;
    const uint32_t counts = __reduce_add_sync(0xffffffffu, __popc(sure) | __popc(equal) << 16);
    const uint32_t front = __shfl_sync(0xffffffffu, block_scan(lane == 0 ? counts : 0u, sums[3], total), 0);
    int eq = equals + (int)(front >> 16);
    int to = taken + (int)(front & 0xffffu) + min(eq, rank) - min(equals, rank);
    const uint32_t below = (1u << lane) - 1u;
#pragma unroll
    for (int j = 0; j < kSelectItems; ++j) {
      if (j >= per) break;
      const uint32_t eqs = __ballot_sync(0xffffffffu, equal >> j & 1u);
      const bool keep = (sure >> j & 1u) || ((equal >> j & 1u) && eq + __popc(eqs & below) < rank);
      const uint32_t keeps = __ballot_sync(0xffffffffu, keep);
      if (keep) {
        const int at = to + __popc(keeps & below);
        kept[at] = base + first + 32 * j;
        w_out[at] = x[j];
      }
      eq += __popc(eqs);
      to += __popc(keeps);
    }
    taken += (int)(total & 0xffffu) + min(equals + (int)(total >> 16), rank) - min(equals, rank);
    equals += (int)(total >> 16);
    __syncthreads();
  }
}

// A warp copies 16 kept rows: a lane looks up the pages of one, then all lanes copy 16 bytes each of its K and V.
template <int D>
__global__ void __launch_bounds__(256) evict_move_kernel(PagedEvictParams p) {
  constexpr int CH = D / 8, AT_ONCE = 32 / (2 * CH);  // rows copied by one step
  wait_for_launch_before();
  const int b = blockIdx.x / p.Hkv, h = blockIdx.x % p.Hkv, lane = lane_id();
  const int m = min(max(0, min(load_fresh(p.seqlens + b), p.cap)), p.budget);
  const int i0 = (blockIdx.y * 8 + (threadIdx.x >> 5)) * 16;
  if (i0 >= m) return;
  int from = -1, to = -1, from_slot = 0, to_slot = 0;
  if (lane < 16 && i0 + lane < m) {
    const int i = i0 + lane, j = load_fresh(p.kept + (long long)blockIdx.x * p.budget + i);
    from = load_fresh(p.table + b * p.t_sb + j / p.page);
    to = load_fresh(p.target + b * p.n_sb + i / p.page);
    from_slot = j % p.page;
    to_slot = i % p.page;
    if ((unsigned)from >= (unsigned)p.num_pages || (unsigned)to >= (unsigned)p.num_pages) {
      p.st.raise(kErrBadIndex);
      from = to = -1;
    }
  }
  const bool is_v = lane / CH & 1;
  const int e = lane % CH * 8, sub = lane / (2 * CH);
  unsigned short* base = static_cast<unsigned short*>(is_v ? p.vp : p.kp) + h * (is_v ? p.vp_sh : p.kp_sh) + e;
  const long long sp = is_v ? p.vp_sp : p.kp_sp, ss = is_v ? p.vp_ss : p.kp_ss;
  constexpr int STEPS = 16 / AT_ONCE;
#pragma unroll
  for (int s0 = 0; s0 < STEPS; s0 += 8) {
    uint4 r[8];
    long long dst[8];
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      const int row = (s0 + x) * AT_ONCE + sub;
      const int f = __shfl_sync(0xffffffffu, from, row), fs = __shfl_sync(0xffffffffu, from_slot, row);
      const int t = __shfl_sync(0xffffffffu, to, row), ts = __shfl_sync(0xffffffffu, to_slot, row);
      dst[x] = t < 0 ? -1 : t * sp + ts * ss;
      if (t >= 0) r[x] = load_fresh<kOnce>(reinterpret_cast<const uint4*>(base + f * sp + fs * ss));
    }
#pragma unroll
    for (int x = 0; x < 8; ++x)
      if (dst[x] >= 0) *reinterpret_cast<uint4*>(base + dst[x]) = r[x];
  }
}

}  // namespace nsa

extern "C" int nsa_paged_kv_append(void* k_pages, void* v_pages, const int* block_table, const int* seqlens, const void* k, const void* v,
                                   const int* cu_seqlens, int* seqlens_after, int total_len, int batch, int num_kv_heads, int head_dim,
                                   int num_pages, int page_size, int max_pages, const long long* strides, void* stream) {
  using namespace nsa;
  if (!k_pages || !v_pages || !block_table || !seqlens || !seqlens_after || !strides) return kInvalid;
  if (total_len < 0 || (total_len > 0 && (!k || !v))) return kInvalid;
  if (batch <= 0 || num_kv_heads <= 0 || num_pages <= 0 || page_size <= 0 || max_pages <= 0) return kInvalid;
  if (!cu_seqlens && total_len != batch) return kInvalid;
  if (head_dim != 64 && head_dim != 128) return kUnsupported;
  const long long cap = (long long)page_size * max_pages;
  if (cap > (1ll << 30)) return kUnsupported;
  // strides: k_n k_h  v_n v_h  kpage_p kpage_s kpage_h  vpage_p vpage_s vpage_h  table_b
  for (int i = 0; i < 10; ++i)
    if (strides[i] % 8) return kInvalid;
  if (!aligned16(k_pages) || !aligned16(v_pages) || !aligned16(k) || !aligned16(v)) return kInvalid;
  PagedAppendParams p;
  p.k = k; p.v = v; p.kp = k_pages; p.vp = v_pages; p.table = block_table; p.held = seqlens; p.cu = cu_seqlens; p.after = seqlens_after;
  p.k_sn = strides[0]; p.k_sh = strides[1]; p.v_sn = strides[2]; p.v_sh = strides[3];
  p.kp_sp = strides[4]; p.kp_ss = strides[5]; p.kp_sh = strides[6];
  p.vp_sp = strides[7]; p.vp_ss = strides[8]; p.vp_sh = strides[9]; p.t_sb = strides[10];
  p.N = total_len; p.B = batch; p.Hkv = num_kv_heads; p.page = page_size; p.cap = (int)cap; p.num_pages = num_pages;
  p.st.word = status_word();
  const int grid = std::max(1, (total_len + 7) / 8);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  LaunchScope ls_("paged_append", s);
  return cuda_rc(launch_early(head_dim == 128 ? paged_append_kernel<128> : paged_append_kernel<64>, dim3(grid), 256, 0, s, p));
}

extern "C" int nsa_paged_kv_evict(void* k_pages, void* v_pages, const int* block_table, const int* seqlens, const float* weights,
                                  const int* new_block_table, int* seqlens_after, float* weights_after, int* kept, int batch, int num_kv_heads,
                                  int head_dim, int num_pages, int page_size, int max_pages, int max_new_pages, int weight_columns, int budget,
                                  int num_sinks, int num_recent, const long long* strides, void* stream) {
  using namespace nsa;
  if (!k_pages || !v_pages || !block_table || !seqlens || !weights || !new_block_table || !seqlens_after || !weights_after || !kept || !strides)
    return kInvalid;
  if (batch <= 0 || num_kv_heads <= 0 || num_pages <= 0 || page_size <= 0 || max_pages <= 0 || max_new_pages <= 0) return kInvalid;
  if (budget <= 0 || num_sinks < 0 || num_recent < 0 || (long long)num_sinks + num_recent > budget) return kInvalid;
  if (head_dim != 64 && head_dim != 128) return kUnsupported;
  const long long cap = (long long)page_size * max_pages, room = (long long)page_size * max_new_pages;
  if (cap > (1ll << 30) || room > (1ll << 30) || (long long)batch * num_kv_heads > (1ll << 30)) return kUnsupported;
  if (weight_columns < cap || room < std::min<long long>(budget, cap)) return kInvalid;
  const long long most = std::min<long long>(budget, cap);
  if ((most + 127) / 128 > 65535) return kUnsupported;
  // strides: weights_b weights_h  kpage_p kpage_s kpage_h  vpage_p vpage_s vpage_h  table_b new_table_b
  for (int i = 2; i < 8; ++i)
    if (strides[i] % 8) return kInvalid;
  if (!aligned16(k_pages) || !aligned16(v_pages)) return kInvalid;
  PagedEvictParams p;
  p.w = weights; p.w_out = weights_after; p.kept = kept; p.after = seqlens_after; p.kp = k_pages; p.vp = v_pages;
  p.table = block_table; p.target = new_block_table; p.seqlens = seqlens;
  p.w_sb = strides[0]; p.w_sh = strides[1];
  p.kp_sp = strides[2]; p.kp_ss = strides[3]; p.kp_sh = strides[4];
  p.vp_sp = strides[5]; p.vp_ss = strides[6]; p.vp_sh = strides[7]; p.t_sb = strides[8]; p.n_sb = strides[9];
  p.B = batch; p.Hkv = num_kv_heads; p.page = page_size; p.cap = (int)cap; p.num_pages = num_pages; p.w_cols = weight_columns;
  p.budget = budget; p.sinks = num_sinks; p.recent = num_recent;
  p.st.word = status_word();
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  {
    LaunchScope ls_("evict_select", s);
    e = launch_early(evict_select_kernel, dim3(batch * num_kv_heads), kSelectThreads, 0, s, p);
  }
  if (e != cudaSuccess) return cuda_rc(e);
  const dim3 grid(batch * num_kv_heads, (unsigned)((most + 127) / 128));
  LaunchScope ls_("evict_move", s);
  return cuda_rc(launch_early(head_dim == 128 ? evict_move_kernel<128> : evict_move_kernel<64>, grid, 256, 0, s, p));
}
