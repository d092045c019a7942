// kvpool.cu — what a serving step does to a paged KV pool before attention:
// the slot plan of a ragged batch, and the norm, rotation and store of its
// queries and keys.
#include <climits>

#include "kvpool.cuh"

namespace gsec {

// Bit 0: a slot past the pool; bit 1: a plan short of pages, table width or
// capacity, or given a negative length; bit 2: a position outside the tables.
static __device__ unsigned g_kvpool_status;

namespace {

// ---------------------------------------------------------------- slot plan --
// Request i holds old_i tokens on the first have_i = ceil(old_i / page) pages
// of its table row and gets new_i more: need_i = ceil((old_i + new_i) / page) -
// have_i pages, taken in request order from the free list. Both the token and
// the page offsets are exclusive sums over the requests; everything else is
// elementwise over tokens or pages, found by a search in those sums. The sums
// are short (a few KB), so every CTA makes them for itself in shared memory and
// then fills its share of the outputs: one launch, no second pass over a
// workspace, no CTA waits on another.
constexpr int kPlanThreads = 512;

__device__ __forceinline__ int32_t clamp_i32(int64_t v) { return v > INT_MAX ? INT_MAX : (int32_t)v; }

// Last i in [0, n) with sum[i] <= x (sum[0] = 0).
__device__ __forceinline__ int last_le(const int32_t* sum, int n, int32_t x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (sum[mid] <= x)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kPlanThreads) slots_plan_kernel(const SlotPlanArgs a) {
  extern __shared__ int32_t sm[];
  int32_t* cu = sm;                   // [batch + 1]
  int32_t* pg = cu + a.batch + 1;     // [batch + 1]
  int32_t* old = pg + a.batch + 1;    // [batch]
  __shared__ int64_t wsum[2][kPlanThreads / 32];
  const int tid = threadIdx.x, B = a.batch;
  grid_dep_wait();
  grid_dep_launch();
  bool bad = false;
  for (int i = tid; i < B; i += kPlanThreads) {
    int32_t o = a.lens[i], n = a.fresh[i];
    bad |= o < 0 || n < 0;
    o = o < 0 ? 0 : o;
    n = n < 0 ? 0 : n;
    const uint32_t have = a.page_div.div((uint32_t)o + a.page - 1);
    uint32_t want = a.page_div.div((uint32_t)o + (uint32_t)n + a.page - 1);
    bad |= want > (uint32_t)a.width;
    want = want > (uint32_t)a.width ? (uint32_t)a.width : want;
    old[i] = o;
    cu[i] = n;
    pg[i] = want > have ? (int32_t)(want - have) : 0;
  }
  __syncthreads();
  // exclusive sums: each thread over a run of requests, then over the threads
  const int per = (B + kPlanThreads - 1) / kPlanThreads;
  const int i0 = tid * per < B ? tid * per : B, i1 = i0 + per < B ? i0 + per : B;
  int64_t st = 0, sp = 0;
  for (int i = i0; i < i1; ++i) {
    st += cu[i];
    sp += pg[i];
  }
  int64_t xt = st, xp = sp;  // inclusive over the warp
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t yt = __shfl_up_sync(0xffffffffu, xt, d), yp = __shfl_up_sync(0xffffffffu, xp, d);
    if ((tid & 31) >= d) {
      xt += yt;
      xp += yp;
    }
  }
  if ((tid & 31) == 31) {
    wsum[0][tid >> 5] = xt;
    wsum[1][tid >> 5] = xp;
  }
  __syncthreads();
  int64_t bt = xt - st, bp = xp - sp;
  for (int w = 0; w < (tid >> 5); ++w) {
    bt += wsum[0][w];
    bp += wsum[1][w];
  }
  for (int i = i0; i < i1; ++i) {
    const int32_t n = cu[i], q = pg[i];
    cu[i] = clamp_i32(bt);
    pg[i] = clamp_i32(bp);
    bt += n;
    bp += q;
  }
  if (tid == kPlanThreads - 1) {  // its run ends at B: the totals
    cu[B] = clamp_i32(bt);
    pg[B] = clamp_i32(bp);
  }
  __syncthreads();
  const int32_t total = cu[B], pages = pg[B];
  const int64_t cursor = a.cursor[0];
  const int64_t gid = (int64_t)blockIdx.x * kPlanThreads + tid, gsize = (int64_t)gridDim.x * kPlanThreads;
  bad |= total > a.capacity;
  const auto take = [&](int64_t k) -> int32_t {  // k-th page of this step
    const int64_t at = cursor + k;
    if (at >= 0 && at < a.nfree) return a.free_pages[at];
    bad = true;
    return -1;
  };
  for (int64_t i = gid; i <= B; i += gsize) {
    a.cu[i] = cu[i];
    if (i < B) a.lens_out[i] = old[i] + (cu[i + 1] - cu[i]);
  }
  if (gid == 0) a.cursor_out[0] = (int32_t)(cursor + pages);
  for (int64_t k = gid; k < pages; k += gsize) {
    const int r = last_le(pg, B + 1, (int32_t)k);
    const int64_t col = a.page_div.div((uint32_t)old[r] + a.page - 1) + (k - pg[r]);
    a.table[r * a.table_pitch + col] = take(k);
  }
  // four tokens per thread: one search, wide stores
  for (int64_t t0 = gid * 4; t0 < a.capacity; t0 += gsize * 4) {
    int64_t slot[4];
    int32_t pos[4];
    int r = t0 < total ? last_le(cu, B + 1, (int32_t)t0) : 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t t = t0 + j;
      slot[j] = -1;
      pos[j] = 0;
      if (t < total) {
        while (cu[r + 1] <= t) ++r;  // requests without new tokens are passed over
        const int32_t p = old[r] + (int32_t)(t - cu[r]);
        const uint32_t pi = a.page_div.div((uint32_t)p);
        const uint32_t have = a.page_div.div((uint32_t)old[r] + a.page - 1);
        int32_t page = -1;
        if (pi < (uint32_t)a.width)
          page = pi < have ? a.table[r * a.table_pitch + pi] : take((int64_t)pg[r] + (pi - have));
        bad |= page < 0;
        if (page >= 0) slot[j] = (int64_t)page * a.page + (p - (int32_t)(pi * a.page));
        pos[j] = a.base + p;
      }
    }
    if (t0 + 4 <= a.capacity) {
      *reinterpret_cast<longlong2*>(a.slots + t0) = make_longlong2(slot[0], slot[1]);
      *reinterpret_cast<longlong2*>(a.slots + t0 + 2) = make_longlong2(slot[2], slot[3]);
      *reinterpret_cast<int4*>(a.positions + t0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
    } else {
#pragma unroll
      for (int j = 0; j < 3; ++j)
        if (t0 + j < a.capacity) {
          a.slots[t0 + j] = slot[j];
          a.positions[t0 + j] = pos[j];
        }
    }
  }
  if (bad) atomicOr(&g_kvpool_status, 2u);
}

// ------------------------------------------- norm, rotation, store (q, k, v) --
// y = x * rsqrt(mean(x^2) + eps) * w per head (w given), then each pair (a, b)
// of the first `rot` values turns by its position's angle: (a c - b s,
// b c + a s). Pairs are (i, i + rot/2), or neighbours (interleaved). q goes to
// q_out, k and v to the pool record of the token's slot. All in 32 bits,
// rounded once at the store.
//
// A head is a group of G lanes (a power of two >= dim / vector), one 16-byte
// vector per lane: the sum of squares and the partner values of the rotation
// move by shuffles, and every load and store is one coalesced vector. A group
// takes H consecutive heads of one token, so that a token's cos and sin rows
// are read once per H heads and H loads are in flight per lane.
constexpr int kStoreThreads = 256;

template <typename T, typename SI, typename PI, int H>
__global__ void __launch_bounds__(kStoreThreads) qk_store_kernel(const QkStoreArgs a, int G) {
  using V = Vec16<T>;
  grid_dep_wait();
  grid_dep_launch();
  const int heads = a.hq + 2 * a.hk;
  const int parts = (heads + H - 1) / H;
  const int64_t groups = a.tokens * parts;
  const int lane = threadIdx.x % G;              // lane in its group
  const int vecs = a.dim / V::N, half = a.rot / 2;
  const bool live = lane < vecs;
  const bool turns = lane * V::N < a.rot;
  // partner lane of the split-half rotation; its sign
  const int hv = half / V::N;
  const int partner = a.interleaved || !turns ? lane : (lane < hv ? lane + hv : lane - hv);
  const float sign = lane < hv ? -1.f : 1.f;
  const int64_t step = (int64_t)gridDim.x * (kStoreThreads / G);
  const int64_t g0 = (int64_t)blockIdx.x * (kStoreThreads / G) + threadIdx.x / G;
  const int64_t rounds = (groups + step - 1) / step;  // the same for every lane: shuffles stay whole
  for (int64_t it = 0; it < rounds; ++it) {
    const int64_t g = g0 + it * step;
    const bool on = g < groups;
    const int64_t t = on ? g / parts : 0;
    const int h0 = on ? (int)(g - t * parts) * H : 0;
    const char* row = a.qkv + t * a.qkv_pitch + (int64_t)lane * 16;
    uint4 raw[H];
#pragma unroll
    for (int j = 0; j < H; ++j)
      if (on && live && h0 + j < heads)
        raw[j] = __ldg(reinterpret_cast<const uint4*>(row + (int64_t)(h0 + j) * a.dim * sizeof(T)));
      else
        raw[j] = vzero();
    float c[V::N], s[V::N];
    if (on && h0 < a.hq + a.hk) {
      const int64_t pos = (int64_t)static_cast<const PI*>(a.positions)[t];
      const bool in = pos >= 0 && pos < a.max_pos;
      if (!in && lane == 0) atomicOr(&g_kvpool_status, 4u);
      if (in && live && turns) {
        const float* cr = a.cos + pos * half;
        const float* sr = a.sin + pos * half;
        if (a.interleaved) {
#pragma unroll
          for (int e = 0; e < V::N; ++e) {
            c[e] = __ldg(cr + (lane * V::N + e) / 2);
            s[e] = __ldg(sr + (lane * V::N + e) / 2) * (e & 1 ? 1.f : -1.f);
          }
        } else {
          const int at = (lane < hv ? lane : lane - hv) * V::N;
#pragma unroll
          for (int e = 0; e < V::N; ++e) {
            c[e] = __ldg(cr + at + e);
            s[e] = __ldg(sr + at + e) * sign;
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < V::N; ++e) {
          c[e] = 1.f;
          s[e] = 0.f;
        }
      }
    }
    int64_t slot = -1;
    if (on && h0 + H > a.hq) {
      slot = (int64_t)static_cast<const SI*>(a.slots)[t];
      if (slot >= a.pool_rows) {
        if (lane == 0) atomicOr(&g_kvpool_status, 1u);
        slot = -1;
      }
    }
#pragma unroll
    for (int j = 0; j < H; ++j) {
      const int h = h0 + j;
      uint4 res = raw[j];
      const bool qk = on && h < a.hq + a.hk;
      float x[V::N];
      V::unpack(raw[j], x);
      const void* w = h < a.hq ? a.q_weight : a.k_weight;
      if (a.q_weight != nullptr || a.k_weight != nullptr) {  // the same for every lane
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < V::N; ++e) ss += x[e] * x[e];
        for (int d = G >> 1; d; d >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
        float down = 1.f;
        if (__any_sync(0xffffffffu, ss == INFINITY)) {  // squares past 32 bits: the same with x 2^-64
          float st = 0.f;
#pragma unroll
          for (int e = 0; e < V::N; ++e) st += (x[e] * 0x1p-64f) * (x[e] * 0x1p-64f);
          for (int d = G >> 1; d; d >>= 1) st += __shfl_xor_sync(0xffffffffu, st, d);
          if (ss == INFINITY) {
            ss = st;
            down = 0x1p-64f;
          }
        }
        if (qk && live && w != nullptr) {
          const float r = 1.f / sqrtf(ss / (float)a.dim + a.eps * down * down);
          float wf[V::N];
          V::unpack(__ldg(reinterpret_cast<const uint4*>(w) + lane), wf);
#pragma unroll
          for (int e = 0; e < V::N; ++e) x[e] = x[e] * down * r * wf[e];
        }
      }
      float y[V::N];
#pragma unroll
      for (int e = 0; e < V::N; ++e)
        y[e] = a.interleaved ? x[e ^ 1] : __shfl_sync(0xffffffffu, x[e], partner, G);
      if (qk && turns) {
#pragma unroll
        for (int e = 0; e < V::N; ++e) x[e] = x[e] * c[e] + y[e] * s[e];
      }
      if (qk) res = V::pack(x);
      if (!on || !live || h >= heads) continue;
      if (h < a.hq) {
        *reinterpret_cast<uint4*>(a.q_out + ((t * a.hq + h) * a.dim) * (int64_t)sizeof(T) + lane * 16) = res;
      } else if (slot >= 0) {
        const bool v = h >= a.hq + a.hk;
        const int kh = h - a.hq - (v ? a.hk : 0);
        *reinterpret_cast<uint4*>(a.pool + slot * a.pitch + (v ? a.plane : 0) +
                                  (int64_t)kh * a.dim * sizeof(T) + lane * 16) = res;
      }
    }
  }
}

template <typename T, typename SI, typename PI>
int launch_store(const QkStoreArgs& a, cudaStream_t s) {
  int G = 1;
  while (G * Vec16<T>::N < a.dim) G <<= 1;
  const int heads = a.hq + 2 * a.hk, per_cta = kStoreThreads / G;
  constexpr int H = 4;
  const int64_t groups = a.tokens * ((heads + H - 1) / H);
  int64_t grid = (groups + per_cta - 1) / per_cta;
  const int64_t most = (int64_t)sm_count() * 8;
  if (grid > most) grid = most;
  return launch_rc(launch_pdl(qk_store_kernel<T, SI, PI, H>, dim3((unsigned)grid), dim3(kStoreThreads), 0, s, a, G),
                   "qk_norm_rope_store");
}

template <typename T>
int launch_store_idx(const QkStoreArgs& a, int slot_bytes, int position_bytes, cudaStream_t s) {
  if (slot_bytes == 8)
    return position_bytes == 8 ? launch_store<T, int64_t, int64_t>(a, s) : launch_store<T, int64_t, int32_t>(a, s);
  return position_bytes == 8 ? launch_store<T, int32_t, int64_t>(a, s) : launch_store<T, int32_t, int32_t>(a, s);
}

}  // namespace

int slots_plan(const SlotPlanArgs& a, cudaStream_t s) {
  const size_t smem = (3 * (size_t)a.batch + 2) * sizeof(int32_t);
  const int per_sm = launch_cache().blocks_per_sm(slots_plan_kernel, kPlanThreads, smem);
  if (per_sm < 0) return check_launch("slots_plan launch shape");
  // every CTA pays for the sums: no more CTAs than the outputs keep busy
  int64_t grid = (a.capacity / 4 + kPlanThreads - 1) / kPlanThreads;
  if (grid < 1) grid = 1;
  if (grid > sm_count()) grid = sm_count();
  return launch_rc(launch_pdl(slots_plan_kernel, dim3((unsigned)grid), dim3(kPlanThreads), smem, s, a), "slots_plan");
}

int qk_norm_rope_store(const QkStoreArgs& a, int dtype, int slot_bytes, int position_bytes, cudaStream_t s) {
  if (a.tokens == 0) return GSEC_OK;
  switch (dtype) {
    case GSEC_BF16:
      return launch_store_idx<__nv_bfloat16>(a, slot_bytes, position_bytes, s);
    case GSEC_F16:
      return launch_store_idx<__half>(a, slot_bytes, position_bytes, s);
    default:
      return launch_store_idx<float>(a, slot_bytes, position_bytes, s);
  }
}

unsigned kvpool_device_status(bool clear) {
  unsigned v = 0;
  if (cudaMemcpyFromSymbol(&v, g_kvpool_status, sizeof(v)) != cudaSuccess) return 0xffffffffu;
  if (clear && v) {
    const unsigned z = 0;
    cudaMemcpyToSymbol(g_kvpool_status, &z, sizeof(z));
  }
  return v;
}

}  // namespace gsec
