// Forward of the sliding window with sinks on the 5th-generation tensor cores.
//
// CTA = 128 rows = (128/G consecutive tokens) x (G heads of one KV head) against the tiles of 64 keys of its rows' list (sink_keys.cuh):
//     S  = Q K^T    [128 x 64]   A = Q (SMEM, K-major),   B = K tile (SMEM, K-major)      TMEM [0,64) and [64,128) in turn
//     O += P V      [128 x D]    A = P (TMEM, 16-bit),    B = V tile (SMEM, MN-major)     TMEM [128,128+D)
//   warps 0..3 : softmax, one thread per row (TMEM lane).  The 64 logits of a tile stay in registers between maximum and exponentials; P
//                goes back into tensor memory over the logits.  A lazily updated reference maximum is kept: O and the sums are rescaled
//                only when the row maximum grows by more than 2^8.  At the end the threads normalise O and write it to the Q tile,
//                from where TMA stores take it (row by row to memory in the last CTA of a sequence)
//   warp 4     : TMA producer (Q, K ring of two, V ring of two);   warp 5 : TMEM allocation and MMA issue (one thread)
//
// A row tile sees few keys (9 tiles of 64 at a window of 512), so what bounds the pass is a CTA's beginning and end and the chain of a tile's softmax.
// Hence 96 KB of shared memory and 256 columns of tensor memory, so that two CTAs share an SM and one works while the other loads, waits or
// stores; and two logit buffers, so that the products of a tile run under the softmax of the one before it.  64q/4kv, window 512, 4 sinks, 32 768
// tokens: 775 us alone, 1050 in front of a backward pass (REST below).  Of the 22 600 clocks of a CTA that wrote o's rest with one part of P (895 us) 4000
// passed until its first logits, 900 and a hand-over of 300 a tile of 64 (2200 the first, 1700 the last, which are masked), 4900 from the last P to the
// end.  Against that variant two threads per row made a tile's softmax no shorter (920 us: the exponential unit then serves four warps); the dense
// forward's organisation (two row tiles in one CTA, tiles of 128 keys, one logit buffer each, persistent) took 911 us without the rest and 1074 with it.
#include <type_traits>

#include "attn_tile.cuh"
#include "dispatch.h"
#include "host_util.h"
#include "nsa_b200.h"
#include "sink_exact.cuh"
#include "sink_keys.cuh"
#include "tc5.cuh"
#include "work_steal.cuh"

#include <algorithm>

namespace nsa {

namespace {
constexpr int kKeys = 64;      // of a tile
constexpr int kStages = 2;     // K tiles, and V tiles, in flight
constexpr int kPolyEvery = 3;  // one pair of exponentials in kPolyEvery is evaluated as a polynomial
constexpr int kThreads = 192;
}  // namespace

struct SinkFwdParams {
  void* o;
  uint4* rest;  // what o's rounding took away (rest_chunk), or nullptr
  float* lse;   // [rows, Hq]
  const int* cu;
  long long o_sn, o_sh;
  int rows, B, Hq, Hkv, G, logG, left, sinks;
  float scale2;
  Status st;
};

// REST: for a backward pass.  The probabilities are then two 16-bit parts, p = hi + lo, and P V two products: the backward pass needs sum_d o dO
// next to single dO v, and one part's rounding in o (2^-9 of each p in bf16) would add to dS, which is rounded itself, more than half as much
// again.  Packed 32 K tokens: 915 us with o's rest and one part, 1085 with two; errors against 64 bits, in
// units of the final rounding: o 1.36 -> 1.00, dQ 1.50 -> 1.43, dK 1.46 -> 1.41 (1.41 is what rounding dS alone leaves).
template <typename T, int D, bool REST>
__global__ void __launch_bounds__(kThreads, 2)
sink_fwd_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                   const __grid_constant__ CUtensorMap tmO, SinkFwdParams p, const __grid_constant__ SinkMaps split) {
  constexpr int PANELS = D / 64;
  constexpr int ROW_PANEL = 128 * 128, ROW_BYTES = PANELS * ROW_PANEL;    // Q: [128][D]
  constexpr int KEY_PANEL = kKeys * 128, KEY_BYTES = PANELS * KEY_PANEL;  // K, V tile: [64][D]
  constexpr uint32_t kO = 128;                                            // TMEM columns of O
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* q_sm = smem;  // at the end the output tile
  uint8_t* k_sm = q_sm + ROW_BYTES;
  uint8_t* v_sm = k_sm + kStages * KEY_BYTES;
  uint64_t* q_full = reinterpret_cast<uint64_t*>(v_sm + kStages * KEY_BYTES);
  uint64_t* k_full = q_full + 1;
  uint64_t* k_empty = k_full + kStages;
  uint64_t* v_full = k_empty + kStages;
  uint64_t* v_empty = v_full + kStages;
  uint64_t* s_full = v_empty + kStages;  // [2] per logit buffer
  uint64_t* p_full = s_full + 2;         // [2] likewise: a warp may be a tile ahead of another
  uint64_t* pv_done = p_full + 2;
  uint64_t* all_done = pv_done + 1;  // (at the end the last but one P V may be on its way too: pv_done's parity would not tell)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(all_done + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (smem_u32(smem) & 1023u) {  // the swizzled operand tiles need a 1024-byte aligned base
    if (threadIdx.x == 0) p.st.raise(kErrSmemLayout);
    return;
  }
  const int QT = 128 >> p.logG, h = blockIdx.y;
  wait_for_launch_before();
  int b, qs, Lq, qt;
  const bool work = find_tile_of_rows(p.cu, p.B, p.rows, 7 - p.logG, gridDim.x - 1 - blockIdx.x, p.st, b, qs, Lq, qt);  // long rows first
  if (warp == 0)
    zero_rows_behind<T, D>(p.o, p.o_sn, p.o_sh, end_of_rows(p.cu, p.B, p.rows, p.st), p.rows, blockIdx.x, gridDim.x, h * p.G, p.G);
  if (!work) return;
  const int q0 = qt * QT;
  const int room = sink_room(p.sinks), shift = sink_shift(q0, p.left, room);
  const int columns = min(q0 + QT, Lq) - shift;  // of the list of keys
  const int ntiles = (columns + kKeys - 1) / kKeys;

  if (warp == 4 && lane == 0) {
    mbar_init(q_full, 1);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(k_full + s, 1);
      mbar_init(k_empty + s, 1);
      mbar_init(v_full + s, 1);
      mbar_init(v_empty + s, 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(s_full + s, 1);
      mbar_init(p_full + s, 4);
    }
    mbar_init(pv_done, 1);
    mbar_init(all_done, 1);
    fence_barrier_init();
    mbar_expect_tx(q_full, ROW_BYTES);  // on its way while the tensor memory is allocated
#pragma unroll
    for (int pn = 0; pn < PANELS; ++pn) tma_load_3d(q_sm + pn * ROW_PANEL, &tmQ, q_full, pn * 64, h * p.G, qs + q0);
    mbar_expect_tx(k_full, KEY_BYTES);
    load_key_tile<kKeys, PANELS>(k_sm, &tmK, split.k, k_full, h, qs, 0, room, shift);
  }
  if (warp == 5) {
    tmem_alloc(tmem_slot, 256);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(tmem_slot);

  if (warp == 4) {
    // ===================== TMA producer =====================
    if (lane == 0) {
      for (int i = 0; i < ntiles; ++i) {
        const int s = i % kStages, n = i + 1, sn = n % kStages;
        if (n < ntiles) {
          if (n >= kStages) mbar_wait(k_empty + sn, ((n / kStages) - 1) & 1, p.st);
          mbar_expect_tx(k_full + sn, KEY_BYTES);
          load_key_tile<kKeys, PANELS>(k_sm + sn * KEY_BYTES, &tmK, split.k, k_full + sn, h, qs, n, room, shift);
        }
        if (i >= kStages) mbar_wait(v_empty + s, ((i / kStages) - 1) & 1, p.st);
        mbar_expect_tx(v_full + s, KEY_BYTES);
        load_key_tile<kKeys, PANELS>(v_sm + s * KEY_BYTES, &tmV, split.v, v_full + s, h, qs, i, room, shift);
      }
    }
  } else if (warp == 5) {
    // ===================== MMA issuer =====================
    // The whole warp runs the control flow converged; one elected lane issues (see tc5.cuh on why).
    const uint32_t idesc_s = umma_idesc<T>(128, kKeys, false, false);
    const uint32_t idesc_o = umma_idesc<T>(128, D, false, true);
    const uint32_t q_addr = smem_u32(q_sm), k_base = smem_u32(k_sm), v_base = smem_u32(v_sm);
    // S(i) takes the buffer of P(i - 2), whose product has been issued: the pipe executes in issue order
    auto issue_s = [&](int i) {
      const int s = i % kStages;
      mbar_wait(k_full + s, (i / kStages) & 1, p.st);
      tc_fence_after_sync();
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          umma_ss(tmem + (i & 1) * kKeys, umma_desc_kmajor(q_addr + (kk >> 2) * ROW_PANEL + (kk & 3) * 32),
                  umma_desc_kmajor(k_base + s * KEY_BYTES + (kk >> 2) * KEY_PANEL + (kk & 3) * 32), idesc_s, kk > 0);
        umma_commit(s_full + (i & 1));
        umma_commit(k_empty + s);
      }
      __syncwarp();
    };
    mbar_wait(q_full, 0, p.st);
    issue_s(0);
    for (int i = 0; i < ntiles; ++i) {
      const int s = i % kStages;
      if (i + 1 < ntiles) issue_s(i + 1);
      mbar_wait(v_full + s, (i / kStages) & 1, p.st);
      clean_key_tile<kKeys, PANELS>(v_base + s * KEY_BYTES, i, columns);
      mbar_wait(p_full + (i & 1), (i >> 1) & 1, p.st);
      tc_fence_after_sync();
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < kKeys / 16; ++kk)
          umma_ts(tmem + kO, tmem + (i & 1) * kKeys + kk * 8, umma_desc_mnmajor(v_base + s * KEY_BYTES + kk * 2048, KEY_PANEL), idesc_o, i > 0 || kk > 0);
        if (REST) {
#pragma unroll
          for (int kk = 0; kk < kKeys / 16; ++kk)
            umma_ts(tmem + kO, tmem + (i & 1) * kKeys + 32 + kk * 8, umma_desc_mnmajor(v_base + s * KEY_BYTES + kk * 2048, KEY_PANEL), idesc_o, true);
        }
        umma_commit(v_empty + s);
        umma_commit(pv_done);
      }
      __syncwarp();
    }
    if (elect_one()) umma_commit(all_done);
    __syncwarp();
  } else {
    // ===================== softmax: one thread per row =====================
    const int row = warp * 32 + lane;
    const int tpos = q0 + (row >> p.logG);
    const int head = h * p.G + (row & (p.G - 1));
    const bool valid = tpos < Lq;
    const uint32_t lane_base = tmem + ((uint32_t)(warp * 32) << 16);
    // columns that all rows of the tile see, if all of them are rows
    const int inner0 = q0 + QT - 1 - p.left - shift, inner1 = q0 + QT <= Lq ? q0 + 1 - shift : -1;
    // With one part the output is divided by the sum of the ROUNDED probabilities of tiles that a row does not see in full: where it sees few keys,
    // one of nearly all the weight then leaves no rounding in o.  Log-sum-exp has the exact sum.
    float m_ref = -INFINITY, l = 0.f, l_rounded = 0.f;
    for (int i = 0; i < ntiles; ++i) {
      const uint32_t s_base = lane_base + (i & 1) * kKeys;
      const int u0 = i * kKeys;
      const bool all = u0 >= inner0 && u0 + kKeys <= inner1;
      mbar_wait(s_full + (i & 1), (i >> 1) & 1, p.st);
      tc_fence_after_sync();
      uint32_t su[2][32];
      tmem_ld32(s_base, su[0]);
      tmem_ld32(s_base + 32, su[1]);
      tmem_ld_wait();
      if (!all) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          auto below = [&](int x) { return __funnelshift_lc(0xffffffffu, 0u, min(32, max(0, x - u0 - c * 32))); };
          const uint32_t see = valid ? (below(tpos + 1 - shift) & ~below(tpos - p.left - shift)) | below(min(p.sinks, tpos + 1)) : 0u;
#pragma unroll
          for (int j = 0; j < 32; ++j) su[c][j] = see >> j & 1u ? su[c][j] : __float_as_uint(-INFINITY);
        }
      }
      float t4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int j = 0; j < 64; j += 2) t4[j >> 1 & 3] = fmax3(t4[j >> 1 & 3], __uint_as_float(su[j >> 5][j & 31]), __uint_as_float(su[j >> 5][(j & 31) + 1]));
      const float top = fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3])) * p.scale2;  // (the scale is positive)
      const bool need = top > m_ref + 8.f;
      if (__any_sync(0xffffffffu, need)) {
        float factor = 1.f;
        if (need) {
          factor = m_ref == -INFINITY ? 0.f : fast_exp2(m_ref - top);
          m_ref = top;
          l *= factor;
          l_rounded *= factor;
        }
        if (i > 0) {
          mbar_wait(pv_done, (i - 1) & 1, p.st);  // P V of the tile before is complete (that of the one before it is since S): O is stable
          tc_fence_after_sync();
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t r[32];
            tmem_ld32(lane_base + kO + c * 32, r);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
              const float2 y = fmul2(make_float2(__uint_as_float(r[j]), __uint_as_float(r[j + 1])), make_float2(factor, factor));
              r[j] = __float_as_uint(y.x);
              r[j + 1] = __float_as_uint(y.y);
            }
            tmem_st32(lane_base + kO + c * 32, r);
          }
          tmem_st_wait();
        }
      }
      const float nm = m_ref == -INFINITY ? 0.f : -m_ref;
      float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
      uint32_t pk[32], lo[32];
      auto exps = [&](auto full_tag) {
        constexpr bool FULL = decltype(full_tag)::value;
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          const float2 x = ffma2(make_float2(__uint_as_float(su[j >> 4][2 * j & 31]), __uint_as_float(su[j >> 4][(2 * j & 31) + 1])),
                                 make_float2(p.scale2, p.scale2), make_float2(nm, nm));
          const float2 e = FULL && j % kPolyEvery == kPolyEvery - 1 ? exp2_poly2(x) : make_float2(fast_exp2(x.x), fast_exp2(x.y));
          sum[j & 1] = fadd2(sum[j & 1], e);
          pk[j] = DT<T>::pack(e.x, e.y);
          if (REST) {
            const float2 r = DT<T>::unpack(pk[j]);
            lo[j] = DT<T>::pack(e.x - r.x, e.y - r.y);
          }
        }
      };
      if (all) exps(std::true_type{});
      else exps(std::false_type{});
      tmem_st32(s_base, pk);
      if (REST) tmem_st32(s_base + 32, lo);
      const float more = (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
      l += more;
      if (REST || all) {
        l_rounded += more;
      } else {
        float2 r[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int j = 0; j < 32; ++j) r[j & 1] = fadd2(r[j & 1], DT<T>::unpack(pk[j]));
        l_rounded += (r[0].x + r[0].y) + (r[1].x + r[1].y);
      }
      tmem_st_wait();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full + (i & 1));
    }
    // ---- epilogue: O / sum, 64 columns at a time ----
    // A query sees itself at least: its sum is zero where all its logits are minus infinity, and neither output nor log-sum-exp is a number then.
    // (With minus infinity the backward pass would give its keys infinities, as for a sum that is none.)
    const float inv = valid ? 1.f / l_rounded : 0.f, lse = l == 0.f ? NAN : m_ref + log2f(l);
    if (valid) p.lse[(long long)(qs + tpos) * p.Hq + head] = lse;
    // A row tile whose tokens all belong to the sequence leaves through the Q tile (free since the last S product, in the swizzled
    // panel layout) and one TMA store per panel; otherwise row by row.
    const bool staged = q0 + QT <= Lq;
    T* orow = static_cast<T*>(p.o) + (long long)(qs + tpos) * p.o_sn + (long long)head * p.o_sh;
    const long long rest_step = rest_chunk(1, 0, p.Hkv, p.rows, 0, p.G, 0);
    uint4* rest = p.rest + rest_chunk(0, h, p.Hkv, p.rows, qs + tpos, p.G, row & (p.G - 1));
    float2 zero = make_float2(0.f, 0.f);  // 0 times each value
    mbar_wait(all_done, 0, p.st);
    tc_fence_after_sync();
#pragma unroll 1
    for (int c = 0; c < D / 64; ++c) {
      uint32_t r[2][32];
      tmem_ld32(lane_base + kO + c * 64, r[0]);
      tmem_ld32(lane_base + kO + c * 64 + 32, r[1]);
      tmem_ld_wait();
#pragma unroll
      for (int q8 = 0; q8 < 8; ++q8) {  // 16-byte chunk c * 8 + q8 of the row
        const uint32_t* x8 = r[q8 >> 2] + (q8 & 3) * 8;
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 x = fmul2(make_float2(__uint_as_float(x8[2 * e]), __uint_as_float(x8[2 * e + 1])), make_float2(inv, inv));
          zero = ffma2(x, make_float2(0.f, 0.f), zero);
          hi[e] = DT<T>::pack(x.x, x.y);
          const float2 h2 = DT<T>::unpack(hi[e]);
          lo[e] = DT<T>::pack(x.x - h2.x, x.y - h2.y);
        }
        if (REST && valid) rest[q8 * rest_step] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        if (staged)
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(smem_u32(q_sm) + c * ROW_PANEL + row * 128 + ((q8 ^ (row & 7)) << 4)),
                       "r"(hi[0]), "r"(hi[1]), "r"(hi[2]), "r"(hi[3]) : "memory");
        else if (valid)
          *reinterpret_cast<uint4*>(orow + c * 64 + q8 * 8) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
      }
      rest += 8 * rest_step;
    }
    // rows with a value that is not finite, one by one (0 times infinity is no number)
    __syncwarp();
    for (unsigned redo = __ballot_sync(0xffffffffu, valid && zero.x + zero.y != 0.f); redo; redo &= redo - 1) {
      const int src = __ffs(redo) - 1;
      const int t = __shfl_sync(0xffffffffu, tpos, src), hd = __shfl_sync(0xffffffffu, head, src), rw = __shfl_sync(0xffffffffu, row, src);
      const float4 x = exact_query_row<T, D, false>(&split, qs, t, hd, h, p.left, p.sinks, p.scale2, 0.f, __shfl_sync(0xffffffffu, lse, src), 0.f);
      if (staged) store_lane_elements_swizzled<T, D, ROW_PANEL>(q_sm, rw, x);
      else store_lane_elements<T, D>(static_cast<T*>(p.o) + (long long)(qs + t) * p.o_sn + (long long)hd * p.o_sh, x);
      if (REST) {
        const int at = lane * (D / 32);  // element; a chunk has eight
        T* chunk = reinterpret_cast<T*>(p.rest + rest_chunk(at / 8, h, p.Hkv, p.rows, qs + t, p.G, hd - h * p.G));
        const float2 a = DT<T>::unpack(DT<T>::pack(x.x, x.y)), c = DT<T>::unpack(DT<T>::pack(x.z, x.w));
        const auto lost = [](float exact, float rounded) { return isinf(exact) ? 0.f : exact - rounded; };  // (an infinity loses nothing)
        uint32_t* dst = reinterpret_cast<uint32_t*>(chunk + at % 8);
        dst[0] = DT<T>::pack(lost(x.x, a.x), lost(x.y, a.y));
        if constexpr (D == 128) dst[1] = DT<T>::pack(lost(x.z, c.x), lost(x.w, c.y));
      }
    }
    if (staged) {
      fence_proxy_async();  // the TMA engine reads the tile through the async proxy
      asm volatile("bar.sync 1, 128;\n" ::: "memory");
      if (threadIdx.x == 0) {
#pragma unroll
        for (int pn = 0; pn < PANELS; ++pn) tma_store_3d(&tmO, q_sm + pn * ROW_PANEL, pn * 64, h * p.G, qs + q0);
        tma_store_commit();
        tma_store_wait_read();
      }
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 5) tmem_dealloc(tmem, 256);
}

int make_sink_maps(SinkMaps& m, CUtensorMapDataType dt, const void* q, const void* k, const void* v, const void* dout, const long long* S, int D,
                   int Hkv, int rows, int sinks, int tile) {
  sink_inputs(m, q, k, v, dout, S);
  const int first = sink_room(sinks) % tile;
  for (int x = 0; x < 2; ++x) {
    const int height = first == 0 ? tile : x ? tile - first : first;
    int rc = make_tmap_3d(&m.k[x], dt, k, D, Hkv, rows, S[3], S[2], 64, 1, height);
    if (!rc) rc = make_tmap_3d(&m.v[x], dt, v, D, Hkv, rows, S[5], S[4], 64, 1, height);
    if (rc) return rc;
  }
  return kOk;
}

template <typename T, int D>
static int launch_sink_fwd(const void* q, const void* k, const void* v, const long long* S, SinkFwdParams p, cudaStream_t stream) {
  // S: q_n q_h k_n k_h v_n v_h o_n o_h
  CUtensorMap tmQ, tmK, tmV, tmO;
  SinkMaps split;
  const int QT = 128 / p.G;
  int rc = make_tmap_3d(&tmQ, DT<T>::kTmapType, q, D, p.Hq, p.rows, S[1], S[0], 64, p.G, QT);
  if (!rc) rc = make_tmap_3d(&tmK, DT<T>::kTmapType, k, D, p.Hkv, p.rows, S[3], S[2], 64, 1, kKeys);
  if (!rc) rc = make_tmap_3d(&tmV, DT<T>::kTmapType, v, D, p.Hkv, p.rows, S[5], S[4], 64, 1, kKeys);
  if (!rc) rc = make_tmap_3d(&tmO, DT<T>::kTmapType, p.o, D, p.Hq, p.rows, p.o_sh, p.o_sn, 64, p.G, QT);
  if (!rc) rc = make_sink_maps(split, DT<T>::kTmapType, q, k, v, nullptr, S, D, p.Hkv, p.rows, p.sinks, kKeys);
  if (rc) return rc;
  const size_t smem = (size_t)(128 + 2 * kStages * kKeys) * D * 2 + 18 * sizeof(uint64_t);
  auto kern = p.rest ? sink_fwd_tc_kernel<T, D, true> : sink_fwd_tc_kernel<T, D, false>;
  cudaError_t e = allow_smem(kern, smem, /*shared_sm=*/true);
  if (e != cudaSuccess) return cuda_rc(e);
  const dim3 grid((unsigned)row_tile_slots(p.rows, p.B, 7 - p.logG), p.Hkv);
  LaunchScope ls_("sink_fwd_tc", stream);
  return cuda_rc(launch_early(kern, grid, kThreads, smem, stream, tmQ, tmK, tmV, tmO, p, split));
}

}  // namespace nsa

extern "C" int nsa_sink_window_attn_fwd(const void* q, const void* k, const void* v, const int* cu_seqlens, void* o, void* o_rest, float* lse,
                                        int total_len, int batch, int num_q_heads, int num_kv_heads, int head_dim, int window_left,
                                        int num_sinks, const long long* strides, float sm_scale, int dtype, void* stream) {
  using namespace nsa;
  if (!q || !k || !v || !cu_seqlens || !o || !lse || !strides) return kInvalid;
  if (total_len <= 0 || batch <= 0 || num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads) return kInvalid;
  if (window_left < 0 || num_sinks < 0) return kInvalid;
  const int G = num_q_heads / num_kv_heads;
  if (G > 16 || (G & (G - 1)) || num_kv_heads > 65535) return kUnsupported;
  for (int i = 0; i < 8; ++i)
    if (strides[i] % 8) return kInvalid;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(o) || !aligned16(o_rest)) return kInvalid;
  SinkFwdParams p;
  p.o = o; p.rest = static_cast<uint4*>(o_rest); p.lse = lse; p.cu = cu_seqlens;
  p.o_sn = strides[6]; p.o_sh = strides[7];
  p.rows = total_len; p.B = batch; p.Hq = num_q_heads; p.Hkv = num_kv_heads; p.G = G;
  p.logG = 0;
  while ((1 << p.logG) < G) ++p.logG;
  // no query is further from a key than the batch is long
  p.left = std::min(window_left, total_len);
  p.sinks = std::min(num_sinks, total_len);
  p.scale2 = sm_scale * kLog2e;
  p.st.word = status_word();
  return NSA_DISPATCH_T_D(dtype, head_dim, launch_sink_fwd, q, k, v, strides, p, static_cast<cudaStream_t>(stream));
}
