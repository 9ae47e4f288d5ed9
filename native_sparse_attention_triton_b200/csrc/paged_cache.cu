// The paged key-value cache's own kernels: rows written behind those that a sequence holds, and a sequence cut down to the rows that
// attention has used most.
//
// Row j of sequence b is slot j % page of page table[b][j / page]; a page holds the rows of all KV heads.  Both operators move bytes and
// are bound by HBM (long inputs) or by one chain of dependent loads (length, page, row).
//
// Eviction, for every (sequence, KV head) with L > budget rows: kept are the first `sinks` rows, the last `recent` ones, and of those
// between the r = budget - sinks - recent with the largest weights, equal ones by the lower row; a weight that is no number counts as
// the smallest.  The kept rows go, in their order, to the first `budget` rows of other pages.  `evict_select` finds the r-th largest
// weight by a radix selection on the bits of the weights, eight at a time, then numbers the kept rows; `evict_move` copies them.
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
  for (int b = blockIdx.x * 256 + threadIdx.x; b < p.B; b += gridDim.x * 256)
    p.after[b] = min(p.cap, __ldg(p.held + b) + (p.cu ? __ldg(p.cu + b + 1) - __ldg(p.cu + b) : 1));
  const int n = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (n >= (p.cu ? min(p.N, __ldg(p.cu + p.B)) : p.N)) return;  // rows behind the last sequence are nobody's
  const int b = p.cu ? find_sequence(p.cu, p.B, n) : n;
  const int pos = __ldg(p.held + b) + (p.cu ? n - __ldg(p.cu + b) : 0);
  const int pg = pos >= 0 && pos < p.cap ? __ldg(p.table + b * p.t_sb + pos / p.page) : -1;
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
        kr[x] = __ldg(reinterpret_cast<const uint4*>(k + h * p.k_sh + e));
        vr[x] = __ldg(reinterpret_cast<const uint4*>(v + h * p.v_sh + e));
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

// Larger weights have larger keys; both zeros the same one.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(w + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Exclusive sum over the block's threads of two counts below 65536 each, packed in one word; `total` gets the sum of all.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* warp_sums, uint32_t& total) {
  const int lane = lane_id(), warp = threadIdx.x >> 5;
  uint32_t up = v;
#pragma unroll
  for (int s = 1; s < 32; s <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, up, s);
    if (lane >= s) up += y;
  }
  __syncthreads();
  if (lane == 31) warp_sums[warp] = up;
  __syncthreads();
  uint32_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kSelectThreads / 32; ++w) {
    const uint32_t x = warp_sums[w];
    before += w < warp ? x : 0;
    total += x;
  }
  return before + up - v;
}

__global__ void __launch_bounds__(kSelectThreads) evict_select_kernel(PagedEvictParams p) {
  __shared__ unsigned hist[256];
  __shared__ uint32_t warp_sums[kSelectThreads / 32];
  __shared__ uint32_t s_digit, s_rank;
  const int b = blockIdx.x / p.Hkv, h = blockIdx.x % p.Hkv, tid = threadIdx.x;
  const int len = __ldg(p.seqlens + b), L = max(0, min(len, p.cap)), m = min(L, p.budget);
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
      w_out[i] = __ldg(w + i);
    }
    return;
  }
  // ---- the key of the r-th largest weight between the sinks and the recent rows, and how many of its equals are kept ----
  const int lo = p.sinks, hi = L - p.recent;
  int rank = p.budget - p.sinks - p.recent;  // below the number of rows between
  uint32_t found = 0, mask = 0;
  if (rank > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += kSelectThreads) hist[i] = 0;
      __syncthreads();
      for (int i = lo + tid; i < hi; i += kSelectThreads) {
        const uint32_t key = weight_key(__ldg(w + i));
        if ((key & mask) == found) atomicAdd(hist + (key >> shift & 255u), 1u);
      }
      __syncthreads();
      if (tid < 32) {  // the digit at which the counts from the top pass the rank; eight digits a lane, the largest first
        unsigned own = 0;
#pragma unroll
        for (int x = 0; x < 8; ++x) own += hist[255 - tid * 8 - x];
        unsigned upto = own;
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
          const unsigned y = __shfl_up_sync(0xffffffffu, upto, s);
          if (tid >= s) upto += y;
        }
        const unsigned before = upto - own;
        if (before < (unsigned)rank && upto >= (unsigned)rank) {
          unsigned left = rank - before;
          int x = 0;
          while (hist[255 - tid * 8 - x] < left) left -= hist[255 - tid * 8 - x++];
          s_digit = 255 - tid * 8 - x;
          s_rank = left;
        }
      }
      __syncthreads();
      found |= s_digit << shift;
      mask |= 255u << shift;
      rank = s_rank;
      __syncthreads();
    }
  } else {
    found = 0xffffffffu;  // above every key
  }
  // ---- the kept rows in their order ----
  int taken = 0, equals = 0;
  for (int i0 = 0; i0 < L; i0 += kSelectThreads) {
    const int i = i0 + tid;
    float x = 0.f;
    bool sure = false, equal = false;
    if (i < L) {
      x = __ldg(w + i);
      const bool between = i >= lo && i < hi;
      const uint32_t key = weight_key(x);
      sure = !between || key > found;
      equal = between && key == found && rank > 0;
    }
    uint32_t all;
    const uint32_t at = block_scan((sure ? 1u : 0u) | (equal ? 0x10000u : 0u), warp_sums, all);
    const int eq = equals + (int)(at >> 16);
    const bool keep = sure || (equal && eq < rank);
    // rows kept before this one: the sure ones, and of its equals those that are still within the rank
    const int to = taken + (int)(at & 0xffffu) + min(eq, rank) - min(equals, rank);
    if (keep) {
      kept[to] = i;
      w_out[to] = x;
    }
    taken += (int)(all & 0xffffu) + min(equals + (int)(all >> 16), rank) - min(equals, rank);
    equals += (int)(all >> 16);
  }
}

// A warp copies 16 kept rows: a lane looks up the pages of one, then all lanes copy 16 bytes each of its K and V.
template <int D>
__global__ void __launch_bounds__(256) evict_move_kernel(PagedEvictParams p) {
  constexpr int CH = D / 8, AT_ONCE = 32 / (2 * CH);  // rows copied by one step
  const int b = blockIdx.x / p.Hkv, h = blockIdx.x % p.Hkv, lane = lane_id();
  const int m = min(max(0, min(__ldg(p.seqlens + b), p.cap)), p.budget);
  const int i0 = (blockIdx.y * 8 + (threadIdx.x >> 5)) * 16;
  if (i0 >= m) return;
  int from = -1, to = -1, from_slot = 0, to_slot = 0;
  if (lane < 16 && i0 + lane < m) {
    const int i = i0 + lane, j = __ldg(p.kept + (long long)blockIdx.x * p.budget + i);
    from = __ldg(p.table + b * p.t_sb + j / p.page);
    to = __ldg(p.target + b * p.n_sb + i / p.page);
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
      if (t >= 0) r[x] = __ldcs(reinterpret_cast<const uint4*>(base + f * sp + fs * ss));
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
  if (head_dim == 128) paged_append_kernel<128><<<grid, 256, 0, s>>>(p);
  else paged_append_kernel<64><<<grid, 256, 0, s>>>(p);
  return cuda_rc(cudaGetLastError());
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
  { LaunchScope ls_("evict_select", s); evict_select_kernel<<<batch * num_kv_heads, kSelectThreads, 0, s>>>(p); }
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_rc(e);
  const dim3 grid(batch * num_kv_heads, (unsigned)((most + 127) / 128));
  {
    LaunchScope ls_("evict_move", s);
    if (head_dim == 128) evict_move_kernel<128><<<grid, 256, 0, s>>>(p);
    else evict_move_kernel<64><<<grid, 256, 0, s>>>(p);
  }
  return cuda_rc(cudaGetLastError());
}
