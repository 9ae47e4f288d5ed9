// Rows and keys of a sliding window with sinks one by one, on values of their own alone.
//
// In a tile's products a masked probability is 0, and 0 times a value that is not finite is not 0.  The tensor-core kernels therefore
// look at their results, and what is not finite is computed again here, over the keys (or queries) that the mask lets through and no
// others: a value that is not finite reaches exactly the results that depend on it.  A warp does one row; a row costs it some 60 clocks a key,
// which only batches pay that hold such values.
#pragma once
#include "common.cuh"
#include "sink_keys.cuh"

#include <cfloat>

namespace nsa {

// Elements lane * EPL .. of a row of D.
template <typename T, int D>
__device__ __forceinline__ void lane_elements(float (&x)[4], const void* base, long long offset) {
  const T* p = static_cast<const T*>(base) + offset;
  if constexpr (D == 128) {
    const uint2 u = *reinterpret_cast<const uint2*>(p + lane_id() * 4);
    const float2 a = DT<T>::unpack(u.x), b = DT<T>::unpack(u.y);
    x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y;
  } else {
    const float2 a = DT<T>::unpack(*reinterpret_cast<const uint32_t*>(p + lane_id() * 2));
    x[0] = a.x; x[1] = a.y; x[2] = x[3] = 0.f;
  }
}
__device__ __forceinline__ float warp_dot(const float (&a)[4], const float (&b)[4]) {
  float s = fmaf(a[3], b[3], fmaf(a[2], b[2], fmaf(a[1], b[1], a[0] * b[0])));
#pragma unroll
  for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
  return s;
}

// 2^x.  No probability is zero where its logit is above minus infinity, however far below the smallest float: infinity times it is infinity.  (Nothing
// finite shows the least normal number, which stands for it.)
__device__ __forceinline__ float row_probability(float x) {
  const float w = fast_exp2(x);
  return w == 0.f && x > -INFINITY ? FLT_MIN : w;
}

// Output of query t (GRAD: its dQ) of query head `head`, key head `kvh`; the sequence starts at row `row0`.  lse in base 2.
template <typename T, int D, bool GRAD>
__device__ __noinline__ float4 exact_query_row(const SinkMaps* m, int row0, int t, int head, int kvh, int left, int sinks, float scale2,
                                               float sm_scale, float lse, float delta) {
  float q[4], g[4], k[4], v[4], acc[4] = {0.f, 0.f, 0.f, 0.f};
  lane_elements<T, D>(q, m->q, (long long)(row0 + t) * m->q_sn + head * m->q_sh);
  if constexpr (GRAD) lane_elements<T, D>(g, m->dout, (long long)(row0 + t) * m->do_sn + head * m->do_sh);
  const int first = max(0, t - left), gap_at = min(sinks, first);
  for (int j = gap_at > 0 ? 0 : first; j <= t; j = j + 1 == gap_at ? first : j + 1) {
    lane_elements<T, D>(k, m->keys, (long long)(row0 + j) * m->k_sn + kvh * m->k_sh);
    lane_elements<T, D>(v, m->values, (long long)(row0 + j) * m->v_sn + kvh * m->v_sh);
    float w = row_probability(fmaf(warp_dot(q, k), scale2, -lse));
    if constexpr (GRAD) w *= (warp_dot(g, v) - delta) * sm_scale;
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = fmaf(w, GRAD ? k[e] : v[e], acc[e]);
  }
  return make_float4(acc[0], acc[1], acc[2], acc[3]);
}

// dK and dV of key j of key head `kvh` (its heads are kvh * G ..), a sequence of L rows; ld = (lse, delta) by [row][query head].
template <typename T, int D>
__device__ __noinline__ void exact_key_row(float4& dk, float4& dv, const SinkMaps* m, const float2* ld, int Hq, int row0, int L, int j, int kvh, int G,
                                           int left, int sinks, float scale2, float sm_scale) {
  float q[4], g[4], k[4], v[4], ak[4] = {0.f, 0.f, 0.f, 0.f}, av[4] = {0.f, 0.f, 0.f, 0.f};
  lane_elements<T, D>(k, m->keys, (long long)(row0 + j) * m->k_sn + kvh * m->k_sh);
  lane_elements<T, D>(v, m->values, (long long)(row0 + j) * m->v_sn + kvh * m->v_sh);
  const int last = j < sinks ? L - 1 : (int)min((long long)L - 1, (long long)j + left);
  for (int t = j; t <= last; ++t)
    for (int x = 0; x < G; ++x) {
      const int head = kvh * G + x;
      lane_elements<T, D>(q, m->q, (long long)(row0 + t) * m->q_sn + head * m->q_sh);
      lane_elements<T, D>(g, m->dout, (long long)(row0 + t) * m->do_sn + head * m->do_sh);
      const float2 s = load_fresh(ld + (long long)(row0 + t) * Hq + head);
      const float p = row_probability(fmaf(warp_dot(q, k), scale2, -s.x)), ds = p * (warp_dot(g, v) - s.y) * sm_scale;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        ak[e] = fmaf(ds, q[e], ak[e]);
        av[e] = fmaf(p, g[e], av[e]);
      }
    }
  dk = make_float4(ak[0], ak[1], ak[2], ak[3]);
  dv = make_float4(av[0], av[1], av[2], av[3]);
}

// A lane's share of such a row as 16-bit values.
template <typename T, int D>
__device__ __forceinline__ void store_lane_elements(T* row, float4 x) {
  if constexpr (D == 128)
    *reinterpret_cast<uint2*>(row + lane_id() * 4) = make_uint2(DT<T>::pack(x.x, x.y), DT<T>::pack(x.z, x.w));
  else
    *reinterpret_cast<uint32_t*>(row + lane_id() * 2) = DT<T>::pack(x.x, x.y);
}
// The same into row `row` of a swizzled tile in shared memory, PANEL bytes a panel.
template <typename T, int D, int PANEL>
__device__ __forceinline__ void store_lane_elements_swizzled(uint8_t* tile, int row, float4 x) {
  const int byte = lane_id() * (D / 32) * 2, ci = byte >> 4;
  T* at = reinterpret_cast<T*>(tile + (ci >> 3) * PANEL + row * 128 + (((ci & 7) ^ (row & 7)) << 4) + (byte & 15));
  if constexpr (D == 128)
    *reinterpret_cast<uint2*>(at) = make_uint2(DT<T>::pack(x.x, x.y), DT<T>::pack(x.z, x.w));
  else
    *reinterpret_cast<uint32_t*>(at) = DT<T>::pack(x.x, x.y);
}

}  // namespace nsa
