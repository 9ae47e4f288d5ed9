// dQ pass of the sliding window with sinks on the 5th-generation tensor cores.
//
// CTA = 128 rows = (128/G tokens) x (G heads of one KV head) against the tiles of 64 keys of its rows' list (sink_keys.cuh):
//     S  = Q  K^T   [128 x 64]   A = Q  (SMEM, K-major), B = K tile (SMEM, K-major)       TMEM [0,64)
//     dP = dO V^T   [128 x 64]   A = dO (SMEM, K-major), B = V tile (SMEM, K-major)       TMEM [64,128)
//     dQ += dS K    [128 x D]    A = dS (TMEM, 16-bit),  B = K tile (SMEM, MN-major)      TMEM [128,128+D)
// with P = exp2(S scale - lse), dS = P (dP - delta) scale, delta = sum_d o dO, which it also publishes with lse for the dK/dV pass.
//
// A row tile sees few key tiles (9 of 64 at a window of 512), so what bounds the pass is not its products but a CTA's beginning and end and
// the chain S -> P -> dP -> dS -> dQ of each tile.  Hence tiles of 64 keys instead of the dense pass's 128: with 112 KB of shared memory and
// 256 columns of tensor memory two CTAs share an SM and each works while the other waits, and less of the last tile is empty.  64q/4kv, window 512, 4 sinks, 32 768 tokens: 1390 us against 1650 with
// tiles of 128 and one CTA; of a CTA's 36 000 clocks 9000 pass before its first dS (dO, o and its rest come from memory), 2500 a tile of 64.
//   warps 0..7 : two threads per row (32 key columns each)
//   warp 8     : TMA producer (Q, dO; K ring of two, V ring of one);   warp 9 : TMEM allocation and MMA issue (one thread)
#include "attn_bwd.h"
#include "attn_tile.cuh"
#include "dispatch.h"
#include "host_util.h"
#include "sink_exact.cuh"
#include "sink_keys.cuh"
#include "tc5.cuh"
#include "work_steal.cuh"

namespace nsa {

namespace {
constexpr int kKeys = 64;     // of a tile
constexpr int kKStages = 2;
}  // namespace

template <typename T, int D>
__global__ void __launch_bounds__(320, 2)
sink_dq_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmDO, const __grid_constant__ CUtensorMap tmK,
                  const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmDQ, DenseBwdParams p,
                  const __grid_constant__ SinkMaps split) {
  constexpr int PANELS = D / 64;
  constexpr int ROW_PANEL = 128 * 128, ROW_BYTES = PANELS * ROW_PANEL;     // Q, dO: [128][D]
  constexpr int KEY_PANEL = kKeys * 128, KEY_BYTES = PANELS * KEY_PANEL;   // K, V tile: [64][D]
  constexpr uint32_t kDP = 64, kDQ = 128;                                  // TMEM columns
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* q_sm = smem;
  uint8_t* do_sm = q_sm + ROW_BYTES;
  uint8_t* k_sm = do_sm + ROW_BYTES;                 // ring of kKStages; at the end the dQ tile
  uint8_t* v_sm = k_sm + kKStages * KEY_BYTES;
  float* row_sh = reinterpret_cast<float*>(v_sm + KEY_BYTES);  // [128]
  uint64_t* bars = reinterpret_cast<uint64_t*>(row_sh + 128);
  uint64_t* q_full = bars;
  uint64_t* do_full = bars + 1;
  uint64_t* k_full = bars + 2;
  uint64_t* k_empty = k_full + kKStages;
  uint64_t* v_full = k_empty + kKStages;
  uint64_t* v_empty = v_full + 1;
  uint64_t* s_full = v_empty + 1;
  uint64_t* s_empty = s_full + 1;
  uint64_t* dp_full = s_empty + 1;
  uint64_t* ds_full = dp_full + 1;
  uint64_t* all_done = ds_full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(all_done + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (smem_u32(smem) & 1023u) {  // the swizzled operand tiles need a 1024-byte aligned base
    if (threadIdx.x == 0) p.st.raise(kErrSmemLayout);
    return;
  }
  const int QT = 128 >> p.logG, h = blockIdx.y;
  wait_for_launch_before();
  int b, qs, Lq, qt;
  const bool work = find_tile_of_rows(p.cu_q, p.B, p.rows, 7 - p.logG, gridDim.x - 1 - blockIdx.x, p.st, b, qs, Lq, qt);
  if (warp == 0)
    zero_rows_behind<T, D>(p.dq, p.dq_sn, p.dq_sh, end_of_rows(p.cu_q, p.B, p.rows, p.st), p.rows, blockIdx.x, gridDim.x, h * p.G, p.G);
  if (warp < 8) {  // a warp a row
    for (long long x = (long long)blockIdx.x * 8 + warp; x < p.summed.count(); x += gridDim.x * 8ll) {
      int n;
      if (!p.summed.row(x, n)) continue;
      const long long at = ((long long)n * p.Hkv + h) * D + lane * (D / 32);
#pragma unroll
      for (int c = 0; c < D / 32; ++c) p.dk32[at + c] = p.dv32[at + c] = 0.f;
    }
  }
  if (!work) return;
  const int q0 = qt * QT;
  const int room = sink_room(p.sinks), shift = sink_shift(q0, p.left, room);
  const int columns = min(q0 + QT, Lq) - shift;  // of the list of keys
  const int ntiles = (columns + kKeys - 1) / kKeys;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(do_full, 1);
    for (int s = 0; s < kKStages; ++s) {
      mbar_init(k_full + s, 1);
      mbar_init(k_empty + s, 1);
    }
    mbar_init(v_full, 1);
    mbar_init(v_empty, 1);
    mbar_init(s_full, 1);
    mbar_init(s_empty, 8);
    mbar_init(dp_full, 1);
    mbar_init(ds_full, 8);
    mbar_init(all_done, 1);
    fence_barrier_init();
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, 256);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(tmem_slot);

  if (warp == 8) {
    // ===================== TMA producer =====================
    if (lane == 0) {
      mbar_expect_tx(q_full, ROW_BYTES);
#pragma unroll
      for (int pn = 0; pn < PANELS; ++pn) tma_load_3d(q_sm + pn * ROW_PANEL, &tmQ, q_full, pn * 64, h * p.G, qs + q0);
      for (int i = 0; i < ntiles; ++i) {
        const int sk = i % kKStages;
        if (i >= kKStages) mbar_wait(k_empty + sk, ((i / kKStages) - 1) & 1, p.st);
        mbar_expect_tx(k_full + sk, KEY_BYTES);
        load_key_tile<kKeys, PANELS>(k_sm + sk * KEY_BYTES, &tmK, split.k, k_full + sk, h, qs, i, room, shift);
        if (i == 0) {
          mbar_expect_tx(do_full, ROW_BYTES);
#pragma unroll
          for (int pn = 0; pn < PANELS; ++pn) tma_load_3d(do_sm + pn * ROW_PANEL, &tmDO, do_full, pn * 64, h * p.G, qs + q0);
        } else {
          mbar_wait(v_empty, (i - 1) & 1, p.st);
        }
        mbar_expect_tx(v_full, KEY_BYTES);
        load_key_tile<kKeys, PANELS>(v_sm, &tmV, split.v, v_full, h, qs, i, room, shift);
      }
    }
  } else if (warp == 9) {
    // ===================== MMA issuer =====================
    // The whole warp runs the control flow converged; one elected lane issues (see tc5.cuh on why).
    const uint32_t idesc_s = umma_idesc<T>(128, kKeys, false, false);
    const uint32_t idesc_q = umma_idesc<T>(128, D, false, true);
    const uint32_t q_addr = smem_u32(q_sm), do_addr = smem_u32(do_sm), k_base = smem_u32(k_sm), v_addr = smem_u32(v_sm);
    // logits of a row tile and a key tile, whose panels differ in height
    auto issue_logits = [&](uint32_t d_tmem, uint32_t a_addr, uint32_t b_addr) {
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk)
        umma_ss(d_tmem, umma_desc_kmajor(a_addr + (kk >> 2) * ROW_PANEL + (kk & 3) * 32), umma_desc_kmajor(b_addr + (kk >> 2) * KEY_PANEL + (kk & 3) * 32),
                idesc_s, kk > 0);
    };
    mbar_wait(q_full, 0, p.st);
    // S(i) may start once the softmax threads have read S(i-1); dP(i) once dQ(i-1) has been issued (it overwrites
    // dS(i-1); the pipe executes in issue order); dQ(i) needs dS(i).
    int ns = 0, np = 0, nq = 0;
    long long t0 = 0;
    int idle = 0;
    while (nq < ntiles) {
      bool progressed = false;
      if (ns < ntiles && mbar_test(k_full + (ns % kKStages), (ns / kKStages) & 1) && (ns < 1 || mbar_test(s_empty, (ns - 1) & 1))) {
        clean_key_tile<kKeys, PANELS>(k_base + (ns % kKStages) * KEY_BYTES, ns, columns);
        tc_fence_after_sync();
        if (elect_one()) {
          issue_logits(tmem, q_addr, k_base + (ns % kKStages) * KEY_BYTES);
          umma_commit(s_full);
        }
        __syncwarp();
        ++ns;
        progressed = true;
      }
      if (nq < np && mbar_test(ds_full, nq & 1)) {
        tc_fence_after_sync();
        const int sk = nq % kKStages;
        if (elect_one()) {
          // dS as the two threads of a row left it: 16 columns of pairs at 0 and at 32
#pragma unroll
          for (int kk = 0; kk < kKeys / 16; ++kk)
            umma_ts(tmem + kDQ, tmem + kDP + 32 * (kk >> 1) + 8 * (kk & 1), umma_desc_mnmajor(k_base + sk * KEY_BYTES + kk * 2048, KEY_PANEL), idesc_q,
                    nq > 0 || kk > 0);
          umma_commit(k_empty + sk);
        }
        __syncwarp();
        ++nq;
        progressed = true;
      }
      if (np < ntiles && np == nq && np < ns && mbar_test(v_full, np & 1) && (np > 0 || mbar_test(do_full, 0))) {
        clean_key_tile<kKeys, PANELS>(v_addr, np, columns);
        tc_fence_after_sync();
        if (elect_one()) {
          issue_logits(tmem + kDP, do_addr, v_addr);
          umma_commit(v_empty);
          umma_commit(dp_full);
        }
        __syncwarp();
        ++np;
        progressed = true;
      }
      if (progressed) {
        idle = 0;
      } else if (((++idle) & 1023) == 0) {
        // bounded: every 1024 idle polls look at the clock and at the grid-wide abort flag
        if (idle == 1024) t0 = clock64();
        if (clock64() - t0 > (1ll << 30) || (p.st.word && (*reinterpret_cast<volatile int*>(p.st.word) & kErrWaitTimeout))) {
          p.st.raise(kErrWaitTimeout);
          break;
        }
      }
    }
    if (elect_one()) umma_commit(all_done);
    __syncwarp();
  } else {
    // ===================== softmax / dS: two threads per row =====================
    const int half = warp >> 2;
    const int row = (warp & 3) * 32 + lane;
    const int tpos = q0 + (row >> p.logG);
    const int head = h * p.G + (row & (p.G - 1));
    const bool valid = tpos < Lq;
    const uint32_t lane_base = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    // ---- delta = sum_d o dO of this row, o with what its rounding took away; each of the two threads sums half of the row ----
    const float lse2 = valid ? load_fresh(p.lse + (long long)(qs + tpos) * p.Hq + head) : INFINITY;
    float part = 0.f;
    {
      const uint4* orow = reinterpret_cast<const uint4*>(static_cast<const T*>(p.o) + (long long)(qs + tpos) * p.o_sn + (long long)head * p.o_sh);
      uint4 hi[D / 16], lo[D / 16];
#pragma unroll
      for (int c = 0; c < D / 16; ++c) {
        const int ci = half * (D / 16) + c;  // 16-byte chunk of the row
        hi[c] = valid ? load_fresh(orow + ci) : make_uint4(0, 0, 0, 0);
        lo[c] = valid && p.rest ? load_fresh<kOnce>(p.rest + rest_chunk(ci, h, p.Hkv, p.rows, qs + tpos, p.G, row & (p.G - 1))) : make_uint4(0, 0, 0, 0);
      }
      mbar_wait(do_full, 0, p.st);
      const uint32_t d_addr = smem_u32(do_sm) + row * 128;
#pragma unroll
      for (int c = 0; c < D / 16; ++c) {
        const int ci = half * (D / 16) + c;
        uint32_t du[4];
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];\n" : "=r"(du[0]), "=r"(du[1]), "=r"(du[2]), "=r"(du[3])
                     : "r"(d_addr + (ci >> 3) * ROW_PANEL + (((ci & 7) ^ (row & 7)) << 4)));
        const uint32_t hw[4] = {hi[c].x, hi[c].y, hi[c].z, hi[c].w}, lw[4] = {lo[c].x, lo[c].y, lo[c].z, lo[c].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 a = DT<T>::unpack(hw[e]), r = DT<T>::unpack(lw[e]), g = DT<T>::unpack(du[e]);
          part = fmaf(a.x + r.x, g.x, part);
          part = fmaf(a.y + r.y, g.y, part);
        }
      }
    }
    if (!valid) part = 0.f;
    if (half) row_sh[row] = part;
    asm volatile("bar.sync 1, 256;\n" ::: "memory");
    if (!half) row_sh[row] = part += row_sh[row];
    asm volatile("bar.sync 1, 256;\n" ::: "memory");
    const float delta = row_sh[row];
    if (valid && half == 0) p.ld[(long long)(qs + tpos) * p.Hq + head] = make_float2(lse2, delta);
    const float nlse = -lse2;
    const float ndsc = -delta * p.sm_scale;

    for (int i = 0; i < ntiles; ++i) {
      // the columns this thread's row sees of its 32
      const int u0 = i * kKeys + half * 32;
      auto below = [&](int x) { return __funnelshift_lc(0xffffffffu, 0u, min(32, max(0, x - u0))); };
      const uint32_t see = valid ? (below(tpos + 1 - shift) & ~below(tpos - p.left - shift)) | below(min(p.sinks, tpos + 1)) : 0u;
      const bool any = __any_sync(0xffffffffu, see != 0u), all = __all_sync(0xffffffffu, see == 0xffffffffu);
      // ---- P phase ----
      mbar_wait(s_full, i & 1, p.st);
      tc_fence_after_sync();
      float pf[32];
      if (any) {
        uint32_t su[32];
        tmem_ld32(lane_base + half * 32, su);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
          const float2 x = ffma2(make_float2(__uint_as_float(su[j]), __uint_as_float(su[j + 1])), make_float2(p.scale2, p.scale2), make_float2(nlse, nlse));
          pf[j] = fast_exp2(x.x);
          pf[j + 1] = fast_exp2(x.y);
        }
        if (!all) {
#pragma unroll
          for (int j = 0; j < 32; ++j) pf[j] = see >> j & 1u ? pf[j] : 0.f;
        }
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(s_empty);
      // ---- dS phase ----
      mbar_wait(dp_full, i & 1, p.st);
      tc_fence_after_sync();
      uint32_t dw[16];
      if (any) {
        uint32_t du[32];
        tmem_ld32(lane_base + kDP + half * 32, du);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
          const float2 t2 = ffma2(make_float2(__uint_as_float(du[j]), __uint_as_float(du[j + 1])), make_float2(p.sm_scale, p.sm_scale),
                                  make_float2(ndsc, ndsc));
          const float2 d2 = fmul2(make_float2(pf[j], pf[j + 1]), t2);
          dw[j >> 1] = DT<T>::pack(d2.x, d2.y);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) dw[j] = 0u;
      }
      tmem_st16(lane_base + kDP + half * 32, dw);  // over this thread's own dP logits
      tmem_st_wait();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(ds_full);
    }
    // ---- epilogue: dQ row (this thread stores D/2 of its D values) ----
    mbar_wait(all_done, 0, p.st);
    tc_fence_after_sync();
    // A CTA whose rows all belong to its sequence stages the tile in the K ring, in the swizzled panel layout, and writes it with one TMA
    // store per panel; the last of a sequence stores row by row.
    const bool staged = q0 + QT <= Lq;
    float2 zero = make_float2(0.f, 0.f);  // 0 times each value
    T* dqrow = static_cast<T*>(p.dq) + (long long)(qs + tpos) * p.dq_sn + (long long)head * p.dq_sh + half * (D / 2);
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
      uint32_t r[32];
      tmem_ld32(lane_base + kDQ + half * (D / 2) + c * 32, r);
      tmem_ld_wait();
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) {
        const uint32_t* x = r + q4 * 8;
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          zero = ffma2(make_float2(__uint_as_float(x[2 * e]), __uint_as_float(x[2 * e + 1])), make_float2(0.f, 0.f), zero);
          w[e] = DT<T>::pack(__uint_as_float(x[2 * e]), __uint_as_float(x[2 * e + 1]));
        }
        const int ci = (half * (D / 2) + c * 32) / 8 + q4;  // 16-byte chunk of the row
        if (staged)
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(smem_u32(k_sm) + (ci >> 3) * ROW_PANEL + row * 128 +
                                                                         (((ci & 7) ^ (row & 7)) << 4)),
                       "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
        else if (valid)
          *reinterpret_cast<uint4*>(dqrow + c * 32 + q4 * 8) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
    // rows with a value that is not finite, one by one; a row is two threads', of warps four apart
    const bool fine = !valid || zero.x + zero.y == 0.f;
    asm volatile("bar.sync 1, 256;\n" ::: "memory");
    if (half) row_sh[row] = fine ? 0.f : 1.f;
    asm volatile("bar.sync 1, 256;\n" ::: "memory");
    for (unsigned redo = __ballot_sync(0xffffffffu, !half && (!fine || row_sh[row] != 0.f)); redo; redo &= redo - 1) {
      const int src = __ffs(redo) - 1;
      const int t = __shfl_sync(0xffffffffu, tpos, src), hd = __shfl_sync(0xffffffffu, head, src), rw = __shfl_sync(0xffffffffu, row, src);
      const float4 x = exact_query_row<T, D, true>(&split, qs, t, hd, h, p.left, p.sinks, p.scale2, p.sm_scale, __shfl_sync(0xffffffffu, lse2, src),
                                                   __shfl_sync(0xffffffffu, delta, src));
      if (staged) store_lane_elements_swizzled<T, D, ROW_PANEL>(k_sm, rw, x);
      else store_lane_elements<T, D>(static_cast<T*>(p.dq) + (long long)(qs + t) * p.dq_sn + (long long)hd * p.dq_sh, x);
    }
    if (staged) {
      fence_proxy_async();  // the TMA engine reads the tile through the async proxy
      asm volatile("bar.sync 1, 256;\n" ::: "memory");
      if (threadIdx.x == 0) {
#pragma unroll
        for (int pn = 0; pn < PANELS; ++pn) tma_store_3d(&tmDQ, k_sm + pn * ROW_PANEL, pn * 64, h * p.G, qs + q0);
        tma_store_commit();
        tma_store_wait_read();
      }
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 9) tmem_dealloc(tmem, 256);
}

template <typename T, int D>
static int launch_sink_dq(const void* k, const void* v, const long long* S, int total, DenseBwdParams p, cudaStream_t stream) {
  CUtensorMap tmQ, tmDO, tmK, tmV, tmDQ;
  const int QT = 128 / p.G;
  int rc = make_tmap_3d(&tmQ, DT<T>::kTmapType, p.q, D, p.Hq, total, p.q_sh, p.q_sn, 64, p.G, QT);
  if (!rc) rc = make_tmap_3d(&tmDO, DT<T>::kTmapType, p.dout, D, p.Hq, total, p.do_sh, p.do_sn, 64, p.G, QT);
  if (!rc) rc = make_tmap_3d(&tmK, DT<T>::kTmapType, k, D, p.Hkv, total, S[3], S[2], 64, 1, kKeys);
  if (!rc) rc = make_tmap_3d(&tmV, DT<T>::kTmapType, v, D, p.Hkv, total, S[5], S[4], 64, 1, kKeys);
  if (!rc) rc = make_tmap_3d(&tmDQ, DT<T>::kTmapType, p.dq, D, p.Hq, total, p.dq_sh, p.dq_sn, 64, p.G, QT);
  SinkMaps split;
  if (!rc) rc = make_sink_maps(split, DT<T>::kTmapType, p.q, k, v, p.dout, S, D, p.Hkv, total, p.sinks, kKeys);
  if (rc) return rc;
  p.rows = total;
  const size_t smem = (size_t)(2 * 128 + (kKStages + 1) * kKeys) * D * 2 + 128 * sizeof(float) + 16 * sizeof(uint64_t) + 16;
  auto kern = sink_dq_tc_kernel<T, D>;
  cudaError_t e = allow_smem(kern, smem, /*shared_sm=*/true);
  if (e != cudaSuccess) return cuda_rc(e);
  const dim3 grid((unsigned)row_tile_slots(total, p.B, 7 - p.logG), p.Hkv);
  LaunchScope ls_("sink_dq_tc", stream);
  return cuda_rc(launch_early(kern, grid, 320, smem, stream, tmQ, tmDO, tmK, tmV, tmDQ, p, split));
}

int sink_dq_tc(const void* k, const void* v, const long long* strides, int total, int head_dim, int dtype, DenseBwdParams p, cudaStream_t stream) {
  return NSA_DISPATCH_T_D(dtype, head_dim, launch_sink_dq, k, v, strides, total, p, stream);
}

}  // namespace nsa
