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
// workspace, no CTA waits on another. Bound by the latency of lengths, sums, search
// and page lookup one after another, and by the call's host time: 64 decode requests
// 5.6 us a call, 3001 ragged ones 7.3, 16 prompts of 32768 tokens 8.0 (6.4 MB out).
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
  const int64_t cursor = a.cursor[0];
  bool bad = false;
  for (int i = tid; i < B; i += kPlanThreads) {
    int32_t o = a.lens[i], n = a.fresh[i];
    bad |= o < 0 || n < 0;
    o = o < 0 ? 0 : o;
    n = n < 0 ? 0 : n;
    // a length or a position past 32 bits does not exist
    const int32_t top = (a.base > 0 ? INT_MAX - a.base : INT_MAX) - o;
    if (n > 0 && n > top) {
      n = top < 0 ? 0 : top;
      bad = true;
    }
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
  // sums of the warps before this one: every warp adds them up for itself
  constexpr int kWarps = kPlanThreads / 32;
  const int lane = tid & 31, warp = tid >> 5;
  int64_t vt = lane < warp ? wsum[0][lane % kWarps] : 0, vp = lane < warp ? wsum[1][lane % kWarps] : 0;
#pragma unroll
  for (int d = kWarps >> 1; d; d >>= 1) {
    vt += __shfl_xor_sync(0xffffffffu, vt, d);
    vp += __shfl_xor_sync(0xffffffffu, vp, d);
  }
  int64_t bt = xt - st + __shfl_sync(0xffffffffu, vt, 0), bp = xp - sp + __shfl_sync(0xffffffffu, vp, 0);
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
// vector per lane: the sum of squares and the partner vectors of the rotation
// move by shuffles, and every load and store is one coalesced vector. A group
// takes up to H heads of one kind (query, key, value) of one token, so that a
// token's cos and sin rows are read once per H heads and H loads are in flight
// per lane. With the weights folded into cos and sin a head is
// r (x (w c) + y (w' s)), y the partner's values as they came: one shuffle per
// word of two values, before they are unpacked. Two values go to an instruction
// (f32x2) where they can.
//
// Instruction issue bounds it beside DRAM: about 160 instructions a vector of 8
// values. 16381 tokens of 48 heads, fp16: 81 us, 5.0 TB/s; 2048 in bf16: 12 us.
// Threads: 256 took 87 and 15 us, 64 82 and 14.7; heads: 2 took 98 and 18, 8 took 93
// and 16 (with 256 threads). What is read and written once streams past L2's other
// contents (ld.cs, st.cs): without either 82 and 14.2, loads alone 88 and 12.5.
constexpr int kStoreThreads = 128;
constexpr int kStoreHeads = 4;

__device__ __forceinline__ uint64_t two(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void apart(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// 16 bytes that are read once. Like every load of this file it stays behind
// grid_dep_wait(): the kernel before may still be writing them.
__device__ __forceinline__ uint4 load_once(const void* p) {
  uint4 v;
  asm volatile("ld.global.cs.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p)
               : "memory");
  return v;
}

// Four values of a cos or sin row (two for 32-bit pairs of neighbours).
template <int N>
__device__ __forceinline__ void load_angles(const float* at, float* f) {
  if (N == 2) {
    const float2 v = *reinterpret_cast<const float2*>(at);
    f[0] = v.x;
    f[1] = v.y;
  } else {
#pragma unroll
    for (int e = 0; e < N; e += 4) {
      const float4 v = *reinterpret_cast<const float4*>(at + e);
      f[e] = v.x;
      f[e + 1] = v.y;
      f[e + 2] = v.z;
      f[e + 3] = v.w;
    }
  }
}

__device__ __forceinline__ int64_t index_at(const void* p, int bytes, uint32_t i) {
  return bytes == 8 ? static_cast<const int64_t*>(p)[i] : (int64_t)static_cast<const int32_t*>(p)[i];
}

// G and the kind of pairs are compile-time: the shuffles of a loop whose length is
// not cost more than the arithmetic (290 instructions a vector).
template <typename T, int G, bool INTERLEAVED>
__global__ void __launch_bounds__(kStoreThreads) qk_store_kernel(const QkStoreArgs a) {
  using V = Vec16<T>;
  constexpr int N = V::N, H = kStoreHeads;
  grid_dep_wait();
  grid_dep_launch();
  const uint32_t g = blockIdx.x * (uint32_t)(kStoreThreads / G) + threadIdx.x / G;
  const uint32_t t = a.part_div.div(g);
  const int part = (int)(g - t * a.part_div.d);
  const int qp = (a.hq + H - 1) / H, kp = (a.hk + H - 1) / H;
  const int kind = part < qp ? 0 : (part < qp + kp ? 1 : 2);     // query, key, value
  const int h0 = (kind == 0 ? part : kind == 1 ? part - qp : part - qp - kp) * H;
  const int nh = t < a.tokens ? (kind ? a.hk : a.hq) - h0 : 0;   // heads from h0 on
  const int lane = threadIdx.x % G, vecs = a.dim / N, half = a.rot / 2;
  const bool live = lane < vecs;
  const int row_head = (kind == 0 ? 0 : kind == 1 ? a.hq : a.hq + a.hk) + h0;
  const char* row = a.qkv + (int64_t)t * a.qkv_pitch + (int64_t)row_head * (a.dim * (int)sizeof(T)) + lane * 16;
  uint4 raw[H];
#pragma unroll
  for (int j = 0; j < H; ++j)
    raw[j] = live && j < nh ? load_once(row + j * a.dim * (int)sizeof(T)) : vzero();
  int64_t slot = -1;
  if (kind && nh > 0) {
    slot = index_at(a.slots, a.slot_bytes, t);
    if (slot >= a.pool_rows) {
      if (lane == 0) atomicOr(&g_kvpool_status, 1u);
      slot = -1;
    }
  }
  // this lane's vector turns with its partner's: itself for pairs of neighbours
  const int hv = half / N;
  const bool turns = lane * N < a.rot;
  const int partner = INTERLEAVED || !turns ? lane : (lane < hv ? lane + hv : lane - hv);
  const void* w = kind ? a.k_weight : a.q_weight;
  float c[N], s[N];                                              // times x and times its partner
  bool rotates = false;
  if (kind < 2) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      c[e] = 1.f;
      s[e] = 0.f;
    }
    if (nh > 0) {
      const int64_t pos = index_at(a.positions, a.position_bytes, t);
      if (pos < 0 || pos >= a.max_pos) {
        if (lane == 0 && a.rot > 0) atomicOr(&g_kvpool_status, 4u);
      } else if (turns) {
        rotates = true;
        const float *cr = a.cos + pos * half, *sr = a.sin + pos * half;
        if (INTERLEAVED) {
          float cc[N / 2], ss[N / 2];
          load_angles<N / 2>(cr + lane * (N / 2), cc);
          load_angles<N / 2>(sr + lane * (N / 2), ss);
#pragma unroll
          for (int e = 0; e < N; ++e) {
            c[e] = cc[e / 2];
            s[e] = e & 1 ? ss[e / 2] : -ss[e / 2];
          }
        } else {
          const int at = (lane < hv ? lane : lane - hv) * N;
          load_angles<N>(cr + at, c);
          load_angles<N>(sr + at, s);
          if (lane < hv) {
#pragma unroll
            for (int e = 0; e < N; ++e) s[e] = -s[e];
          }
        }
      }
    }
    if (w != nullptr && live) {
      float wf[N], wp[N];
      V::unpack(reinterpret_cast<const uint4*>(w)[lane], wf);
      V::unpack(reinterpret_cast<const uint4*>(w)[partner], wp);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        c[e] *= wf[e];
        s[e] *= wp[INTERLEAVED ? e ^ 1 : e];
      }
    }
  }
  const int head = a.dim * (int)sizeof(T);
  char* dst = (kind == 0 ? a.q_out + ((int64_t)t * a.hq + h0) * head
                         : a.pool + slot * a.pitch + (kind == 2 ? a.plane : 0) + (int64_t)h0 * head) +
              lane * 16;
  const bool stores = live && (kind == 0 || slot >= 0);
  const bool norms = a.q_weight != nullptr || a.k_weight != nullptr;  // the same for every lane: shuffles stay whole
  const bool some = __any_sync(0xffffffffu, kind < 2);          // a warp of values alone has nothing to work out
#pragma unroll
  for (int j = 0; j < H; ++j) {
    float x[N], y[N], r = 1.f, down = 1.f;
    uint4 other = raw[j];
    if (!INTERLEAVED && some)
      other = make_uint4(__shfl_sync(0xffffffffu, other.x, partner, G), __shfl_sync(0xffffffffu, other.y, partner, G),
                         __shfl_sync(0xffffffffu, other.z, partner, G), __shfl_sync(0xffffffffu, other.w, partner, G));
    V::unpack(raw[j], x);
    if (norms && some) {
      uint64_t squares = two(0.f, 0.f);
#pragma unroll
      for (int e = 0; e < N; e += 2) squares = fma2(two(x[e], x[e + 1]), two(x[e], x[e + 1]), squares);
      float ss, odd;
      apart(squares, ss, odd);
      ss += odd;
#pragma unroll
      for (int d = G >> 1; d; d >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
      if (__any_sync(0xffffffffu, ss == INFINITY)) {  // squares past 32 bits: the same with x 2^-64
        float st = 0.f;
#pragma unroll
        for (int e = 0; e < N; ++e) st += (x[e] * 0x1p-64f) * (x[e] * 0x1p-64f);
#pragma unroll
        for (int d = G >> 1; d; d >>= 1) st += __shfl_xor_sync(0xffffffffu, st, d);
        if (ss == INFINITY) {
          ss = st;
          down = 0x1p-64f;
        }
      }
      r = rsqrtf(ss * a.inv_dim + a.eps * down * down);  // 2 ulp
    }
    if (!live || j >= nh) continue;
    uint4 res = raw[j];
    if (kind < 2 && (w != nullptr || rotates)) {
      if (w == nullptr) {
        down = 1.f;
      } else if (down != 1.f) {
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] *= down;
      }
#pragma unroll
      for (int e = 0; e < N; e += 2) apart(mul2(two(x[e], x[e + 1]), two(c[e], c[e + 1])), x[e], x[e + 1]);
      if (rotates) {
        V::unpack(other, y);
        if (down != 1.f) {
#pragma unroll
          for (int e = 0; e < N; ++e) y[e] *= down;
        }
#pragma unroll
        for (int e = 0; e < N; e += 2)
          apart(fma2(INTERLEAVED ? two(y[e + 1], y[e]) : two(y[e], y[e + 1]), two(s[e], s[e + 1]), two(x[e], x[e + 1])),
                x[e], x[e + 1]);
      }
      if (w != nullptr) {
#pragma unroll
        for (int e = 0; e < N; e += 2) apart(mul2(two(x[e], x[e + 1]), two(r, r)), x[e], x[e + 1]);
      }
      res = V::pack(x);
    }
    if (stores) __stcs(reinterpret_cast<uint4*>(dst + j * head), res);
  }
}

template <typename T, int G>
int launch_store(QkStoreArgs a, cudaStream_t s) {
  if constexpr (G > 1)
    if (G / 2 * Vec16<T>::N >= a.dim) return launch_store<T, G / 2>(a, s);
  const int qp = (a.hq + kStoreHeads - 1) / kStoreHeads, kp = (a.hk + kStoreHeads - 1) / kStoreHeads;
  a.part_div = FastDiv((uint32_t)(qp + 2 * kp));
  a.inv_dim = 1.f / (float)a.dim;
  const int64_t groups = a.tokens * (qp + 2 * kp), per_cta = kStoreThreads / G;
  GSEC_REQUIRE(groups < (1ll << 31), "qk_norm_rope_store: %lld tokens of %d heads are too many for one call",
               (long long)a.tokens, a.hq + 2 * a.hk);
  const dim3 grid((unsigned)((groups + per_cta - 1) / per_cta)), block(kStoreThreads);
  return launch_rc(a.interleaved ? launch_pdl(qk_store_kernel<T, G, true>, grid, block, 0, s, a)
                                 : launch_pdl(qk_store_kernel<T, G, false>, grid, block, 0, s, a),
                   "qk_norm_rope_store");
}

}  // namespace

int slots_plan(const SlotPlanArgs& a, cudaStream_t s) {
  const size_t smem = (3 * (size_t)a.batch + 2) * sizeof(int32_t);
  if (smem > 32 * 1024 && launch_cache().blocks_per_sm(slots_plan_kernel, kPlanThreads, smem) < 0)
    return check_launch("slots_plan launch shape");
  // every CTA pays for the sums: no more CTAs than the outputs keep busy
  int64_t grid = (a.capacity / 4 + kPlanThreads - 1) / kPlanThreads;
  if (grid < 1) grid = 1;
  if (grid > sm_count()) grid = sm_count();
  return launch_rc(launch_pdl(slots_plan_kernel, dim3((unsigned)grid), dim3(kPlanThreads), smem, s, a), "slots_plan");
}

int qk_norm_rope_store(const QkStoreArgs& a, int dtype, cudaStream_t s) {
  if (a.tokens == 0) return GSEC_OK;
  switch (dtype) {
    case GSEC_BF16:
      return launch_store<__nv_bfloat16, 32>(a, s);
    case GSEC_F16:
      return launch_store<__half, 32>(a, s);
    default:
      return launch_store<float, 32>(a, s);
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
