// attention.cu — attention over a paged KV pool whose requests share a prefix.
//
// Query token j of request i (n_i new tokens) sees the P prefix keys and its
// own keys 0 .. lens_i - n_i + j, so with s = q.k * scale
//   lse = log sum exp(s),   o = sum exp(s - lse) v
// over those; a row that sees nothing is o = 0, lse = -inf.
#include <climits>

#include "attention.cuh"
#include "kvpool.cuh"

namespace gsec {

static __device__ unsigned g_attn_status;

namespace {

// Slot of key x of request r (prefix first), or -1 (flagged) for a page outside the pool.
__device__ __forceinline__ int64_t key_slot(const AttnArgs& a, int r, int32_t x) {
  const int32_t own = x - a.prefix_len;
  const uint32_t y = own < 0 ? (uint32_t)x : (uint32_t)own;
  const uint32_t pi = a.page_div.div(y);
  const int32_t page = own < 0 ? __ldg(a.prefix + pi) : __ldg(a.table + r * a.table_pitch + pi);
  const int64_t slot = (int64_t)page * a.page + (y - pi * a.page);
  if (page < 0 || slot >= a.pool_rows) {
    atomicOr(&g_attn_status, 1u);
    return -1;
  }
  return slot;
}

// ------------------------------------------------------ one row per CTA -------
// One query row per CTA. The keys are dealt out to lane groups (a group holds
// one key's vector per step), each with its own running maximum m, sum l and
// accumulator; they meet at the end by
//   m = max m_g, l = sum l_g 2^(m_g - m), o = sum o_g 2^(m_g - m) / l.
constexpr int kRowThreads = 256;

template <typename T, int NC>
__global__ void __launch_bounds__(kRowThreads) attend_row_kernel(const AttnArgs a, int L) {
  using V = Vec16<T>;
  constexpr int E = V::N * NC;
  extern __shared__ float sm[];  // [groups][dim + 2]
  grid_dep_wait();
  grid_dep_launch();
  const int64_t t = blockIdx.x / a.hq;
  const int h = (int)(blockIdx.x - t * a.hq), kh = (int)a.group_div.div(h);
  const int total = a.cu[a.batch] < a.tokens ? a.cu[a.batch] : (int)a.tokens;
  if (t >= total) return;  // rows behind the last request stay as they are
  // the request of token t: the last r with cu[r] <= t
  int r = 0, hi = a.batch;
  while (hi - r > 1) {
    const int mid = (r + hi) >> 1;
    if (a.cu[mid] <= t)
      r = mid;
    else
      hi = mid;
  }
  const int64_t room = (int64_t)a.width * a.page;
  const int64_t len = a.lens[r] < room ? a.lens[r] : room;
  if (threadIdx.x == 0 && a.lens[r] > room) atomicOr(&g_attn_status, 1u);
  const int64_t n = a.cu[r + 1] - a.cu[r], j = t - a.cu[r];
  int64_t own = len - n + j + 1;
  own = own < 0 ? 0 : (own > len ? len : own);
  const int32_t keys = (int32_t)(a.prefix_len + own);

  const int lane = threadIdx.x % L, grp = threadIdx.x / L, ngrp = kRowThreads / L;
  const int vecs = a.dim / V::N;
  const float scale = a.scale * 1.4426950408889634f;
  float q[E], o[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int v = lane + c * L;
    uint4 w = vzero();
    if (v < vecs) w = *reinterpret_cast<const uint4*>(a.q + t * a.q_pitch + h * a.q_head + v * 16);
    V::unpack(w, q + c * V::N);
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] *= scale;
    o[e] = 0.f;
  }
  const int rounds = (keys + ngrp - 1) / ngrp;
  for (int it = 0; it < rounds; ++it) {
    const int32_t x = it * ngrp + grp;
    const int64_t slot = x < keys ? key_slot(a, r, x) : -1;
    const char* rec = a.pool + slot * a.pitch + (int64_t)kh * a.dim * sizeof(T);
    float k[E], v[E], s = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int i = lane + c * L;
      uint4 kw = vzero(), vw = vzero();
      if (slot >= 0 && i < vecs) {
        kw = __ldg(reinterpret_cast<const uint4*>(rec) + i);
        vw = __ldg(reinterpret_cast<const uint4*>(rec + a.plane) + i);
      }
      V::unpack(kw, k + c * V::N);
      V::unpack(vw, v + c * V::N);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) s += q[e] * k[e];
    for (int d = L >> 1; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    if (x < keys) {
      const float top = fmaxf(m, s);
      const float old = top == -INFINITY ? 1.f : exp2f(m - top);  // both empty: nothing to scale
      const float p = top == -INFINITY ? 0.f : exp2f(s - top);
      l = l * old + p;
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = o[e] * old + p * v[e];
      m = top;
    }
  }
  // the groups meet in shared memory
  float* mine = sm + grp * (a.dim + 2);
  if (lane == 0) {
    mine[a.dim] = m;
    mine[a.dim + 1] = l;
  }
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int e = 0; e < V::N; ++e)
      if (lane + c * L < vecs) mine[(lane + c * L) * V::N + e] = o[c * V::N + e];
  __syncthreads();
  float top = -INFINITY, sum = 0.f;
  for (int g = 0; g < ngrp; ++g) top = fmaxf(top, sm[g * (a.dim + 2) + a.dim]);
  for (int g = 0; g < ngrp; ++g)
    if (sm[g * (a.dim + 2) + a.dim] > -INFINITY)
      sum += sm[g * (a.dim + 2) + a.dim + 1] * exp2f(sm[g * (a.dim + 2) + a.dim] - top);
  for (int d = threadIdx.x; d < a.dim; d += kRowThreads) {
    float x = 0.f;
    for (int g = 0; g < ngrp; ++g)
      if (sm[g * (a.dim + 2) + a.dim] > -INFINITY)
        x += sm[g * (a.dim + 2) + d] * exp2f(sm[g * (a.dim + 2) + a.dim] - top);
    reinterpret_cast<T*>(a.out)[(t * a.hq + h) * a.dim + d] = (T)(sum == 0.f ? 0.f : x / sum);
  }
  if (threadIdx.x == 0 && a.lse) a.lse[t * a.hq + h] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
}

template <typename T, int NC>
int launch_rows(const AttnArgs& a, int L, cudaStream_t s) {
  const size_t smem = (size_t)(kRowThreads / L) * (a.dim + 2) * sizeof(float);
  if (launch_cache().blocks_per_sm(attend_row_kernel<T, NC>, kRowThreads, smem) < 0)
    return check_launch("attend_row launch shape");
  return launch_rc(launch_pdl(attend_row_kernel<T, NC>, dim3((unsigned)(a.tokens * a.hq)), dim3(kRowThreads), smem, s,
                              a, L),
                   "prefix_attention");
}

template <typename T>
int attend_rows(const AttnArgs& a, cudaStream_t s) {
  const int vecs = a.dim / Vec16<T>::N;
  int L = 1;
  while (L < vecs && L < 32) L <<= 1;
  return vecs > 32 ? launch_rows<T, 2>(a, L, s) : launch_rows<T, 1>(a, L, s);
}

}  // namespace

int64_t attention_workspace(const AttnArgs&, int) { return 0; }

int attention(const AttnArgs& a, int dtype, cudaStream_t s) {
  if (a.tokens == 0) return GSEC_OK;
  switch (dtype) {
    case GSEC_BF16:
      return attend_rows<__nv_bfloat16>(a, s);
    case GSEC_F16:
      return attend_rows<__half>(a, s);
    default:
      return attend_rows<float>(a, s);
  }
}

unsigned attention_device_status(bool clear) {
  unsigned v = 0;
  if (cudaMemcpyFromSymbol(&v, g_attn_status, sizeof(v)) != cudaSuccess) return 0xffffffffu;
  if (clear && v) {
    const unsigned z = 0;
    cudaMemcpyToSymbol(g_attn_status, &z, sizeof(z));
  }
  return v;
}

}  // namespace gsec
