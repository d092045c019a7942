// attention.cu — attention over a paged KV pool whose requests share a prefix.
//
// Query token j of request i (n_i new tokens) sees the P prefix keys and its
// own keys 0 .. lens_i - n_i + j, so with s = q.k * scale
//   lse = log sum exp(s),   o = sum exp(s - lse) v
// over those; a row that sees nothing is o = 0, lse = -inf.
#include <climits>

#include "attention.cuh"
#include "kvpool.cuh"
#include "tc.cuh"

namespace gsec {

static __device__ unsigned g_attn_status;

namespace {

// Loads of what an earlier kernel may have written (lengths, pages, pool, partial
// results) take the ordinary path: a launch may begin while that kernel still writes,
// and a load through the read-only path promises that nobody does and is not held
// behind grid_dep_wait(). load() is an ordinary load that the compiler may still
// move past this kernel's own stores, which go elsewhere. (As plain dereferences: 256
// requests on one prefix 186 us instead of 181, three short ones 12.5 instead of 11.9.)
__device__ __forceinline__ int32_t load(const int32_t* p) {
  int32_t v;
  asm volatile("ld.global.b32 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}
__device__ __forceinline__ uint4 load(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ float load(const float* p) {
  return __int_as_float(load(reinterpret_cast<const int32_t*>(p)));
}
__device__ __forceinline__ float4 load(const float4* p) {
  float4 v;
  asm volatile("ld.global.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p));
  return v;
}

// Slot of key x of request r (prefix first), or -1 for a page outside the pool.
__device__ __forceinline__ int64_t key_slot(const AttnArgs& a, int r, int32_t x) {
  const int32_t own = x - a.prefix_len;
  const uint32_t y = own < 0 ? (uint32_t)x : (uint32_t)own;
  const uint32_t pi = a.page_div.div(y);
  const int32_t page = load(own < 0 ? a.prefix + pi : a.table + r * a.table_pitch + pi);
  const int64_t slot = (int64_t)page * a.page + (y - pi * a.page);
  return page < 0 || slot >= a.pool_rows ? -1 : slot;
}

// ---------------------------------------------------- a few rows per CTA -------
// What the tensor core does not take: G query heads of one token that share a KV
// head per CTA, so that a key is read once for them. The keys are dealt out to lane
// groups (a group holds one key's vector per step), each with its own running
// maximum m, sum l and accumulator per head; they meet at the end by
//   m = max m_g, l = sum l_g 2^(m_g - m), o = sum o_g 2^(m_g - m) / l.
// Bound by the latency of a step (lookup, loads, sum over the lanes), of which each
// has several keys: 16 requests of 32 fp32 heads on 8 KV heads of 128, behind 4096
// keys, 283 us; 256-wide bf16 heads 319. (G = 1: 418 and 508; G = 2: 392 and 326.)
// Not split over long keys: few rows behind a long cache leave SMs idle.
constexpr int kRowThreads = 256;

template <typename T, int NC, int G>
__global__ void __launch_bounds__(kRowThreads) attend_row_kernel(const AttnArgs a, int L) {
  using V = Vec16<T>;
  constexpr int E = V::N * NC;
  extern __shared__ float sm[];  // [lane groups][G][dim + 2]
  grid_dep_wait();
  grid_dep_launch();
  const int parts = (a.group + G - 1) / G;                // CTAs of a token and KV head
  const int64_t t = blockIdx.x / (unsigned)(a.hk * parts);
  const int rest = (int)(blockIdx.x - t * (a.hk * parts)), kh = rest / parts, g0 = (rest - kh * parts) * G;
  const int h0 = kh * a.group + g0, nh = a.group - g0 < G ? a.group - g0 : G;
  const int total = a.cu[a.batch] < a.tokens ? a.cu[a.batch] : (int)a.tokens;
  const int64_t room = (int64_t)a.width * a.page;
  if (blockIdx.x == 0)  // what is cut below
    for (int i = threadIdx.x; i < a.batch; i += kRowThreads)
      if (a.cu[i] < 0 || a.cu[i + 1] < a.cu[i] || a.cu[i + 1] > a.tokens || a.lens[i] < 0 || a.lens[i] > room)
        atomicOr(&g_attn_status, 1u);
  if (t >= total || t < a.cu[0]) return;  // rows outside the requests stay as they are
  // the request of token t: the last r with cu[r] <= t
  int r = 0, hi = a.batch;
  while (hi - r > 1) {
    const int mid = (r + hi) >> 1;
    if (a.cu[mid] <= t)
      r = mid;
    else
      hi = mid;
  }
  const int64_t len = a.lens[r] < room ? a.lens[r] : room;
  const int c0 = a.cu[r] < 0 ? 0 : a.cu[r], c1 = a.cu[r + 1] < total ? a.cu[r + 1] : total;
  const int64_t n = c1 - c0, j = t - c0;
  int64_t own = len - n + j + 1;
  own = own < 0 ? 0 : (own > len ? len : own);
  const int32_t keys = (int32_t)(a.prefix_len + own);

  const int lane = threadIdx.x % L, grp = threadIdx.x / L, ngrp = kRowThreads / L;
  const int vecs = a.dim / V::N;
  const float scale = a.scale * 1.4426950408889634f;
  float q[G][E], o[G][E], m[G], l[G];
#pragma unroll
  for (int h = 0; h < G; ++h) {
    m[h] = -INFINITY;
    l[h] = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int v = lane + c * L;
      uint4 w = vzero();
      if (v < vecs && h < nh) w = *reinterpret_cast<const uint4*>(a.q + t * a.q_pitch + (h0 + h) * a.q_head + v * 16);
      V::unpack(w, q[h] + c * V::N);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      q[h][e] *= scale;
      o[h][e] = 0.f;
    }
  }
  // kAhead keys' vectors are on their way at a time
  constexpr int kAhead = NC == 1 ? 4 : 2;
  const int rounds = (keys + ngrp - 1) / ngrp;
  bool bad = false;  // a page outside the pool
  for (int it = 0; it < rounds; it += kAhead) {
    uint4 kw[kAhead][NC], vw[kAhead][NC];
    int64_t slots[kAhead];  // all lookups before the first load that waits for one
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int64_t x = (int64_t)(it + u) * ngrp + grp;
      slots[u] = x < keys ? key_slot(a, r, (int32_t)x) : -1;
      bad |= x < keys && slots[u] < 0;
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int64_t slot = slots[u];
      const char* rec = a.pool + slot * a.pitch + (int64_t)kh * a.dim * sizeof(T);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int i = lane + c * L;
        const bool is = slot >= 0 && i < vecs;
        kw[u][c] = is ? load(reinterpret_cast<const uint4*>(rec) + i) : vzero();
        vw[u][c] = is ? load(reinterpret_cast<const uint4*>(rec + a.plane) + i) : vzero();
      }
    }
    float s[kAhead][G];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      float k[E];
#pragma unroll
      for (int c = 0; c < NC; ++c) V::unpack(kw[u][c], k + c * V::N);
#pragma unroll
      for (int h = 0; h < G; ++h) {
        s[u][h] = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) s[u][h] += q[h][e] * k[e];
      }
    }
    for (int d = L >> 1; d; d >>= 1) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
#pragma unroll
        for (int h = 0; h < G; ++h) s[u][h] += __shfl_xor_sync(0xffffffffu, s[u][h], d);
    }
#pragma unroll
    for (int h = 0; h < G; ++h) {
      float top = m[h];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if ((int64_t)(it + u) * ngrp + grp >= keys) s[u][h] = -INFINITY;
        top = fmaxf(top, s[u][h]);
      }
      const float old = top == -INFINITY ? 1.f : exp2f(m[h] - top);  // all empty: nothing to scale
      m[h] = top;
      l[h] *= old;
#pragma unroll
      for (int e = 0; e < E; ++e) o[h][e] *= old;
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        s[u][h] = s[u][h] == -INFINITY ? 0.f : exp2f(s[u][h] - top);
        l[h] += s[u][h];
      }
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      float v[E];
#pragma unroll
      for (int c = 0; c < NC; ++c) V::unpack(vw[u][c], v + c * V::N);
#pragma unroll
      for (int h = 0; h < G; ++h)
#pragma unroll
        for (int e = 0; e < E; ++e) o[h][e] += s[u][h] * v[e];
    }
  }
  if (bad) atomicOr(&g_attn_status, 1u);
  // the groups meet in shared memory
#pragma unroll
  for (int h = 0; h < G; ++h) {
    float* mine = sm + (grp * G + h) * (a.dim + 2);
    if (lane == 0) {
      mine[a.dim] = m[h];
      mine[a.dim + 1] = l[h];
    }
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < V::N; ++e)
        if (lane + c * L < vecs) mine[(lane + c * L) * V::N + e] = o[h][c * V::N + e];
  }
  __syncthreads();
  for (int h = 0; h < nh; ++h) {
    const float* at = sm + h * (a.dim + 2);
    const int step = G * (a.dim + 2);
    float top = -INFINITY, sum = 0.f;
    for (int g = 0; g < ngrp; ++g) top = fmaxf(top, at[g * step + a.dim]);
    // a group without a maximum has l = o = 0, or they are not numbers (a maximum passes those over) and stay so
    const auto weight = [&](int g) {
      const float mg = at[g * step + a.dim];
      return mg == -INFINITY ? 1.f : exp2f(mg - top);
    };
    for (int g = 0; g < ngrp; ++g) sum += at[g * step + a.dim + 1] * weight(g);
    const int64_t row = t * a.hq + h0 + h;
    for (int d = threadIdx.x; d < a.dim; d += kRowThreads) {
      float x = 0.f;
      for (int g = 0; g < ngrp; ++g) x += at[g * step + d] * weight(g);
      reinterpret_cast<T*>(a.out)[row * a.dim + d] = (T)(sum == 0.f ? 0.f : x / sum);
    }
    if (threadIdx.x == 0 && a.lse) a.lse[row] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
  }
}

template <typename T, int NC, int G>
int launch_rows(const AttnArgs& a, int L, cudaStream_t s) {
  const size_t smem = (size_t)(kRowThreads / L) * G * (a.dim + 2) * sizeof(float);
  if (launch_cache().blocks_per_sm(attend_row_kernel<T, NC, G>, kRowThreads, smem) < 0)
    return check_launch("attend_row launch shape");
  const int64_t grid = a.tokens * a.hk * ((a.group + G - 1) / G);  // at most tokens * hq
  return launch_rc(launch_pdl(attend_row_kernel<T, NC, G>, dim3((unsigned)grid), dim3(kRowThreads), smem, s, a, L),
                   "prefix_attention");
}

// Heads together as long as half of the SMs are busy. (fp32, groups of 4 on one KV head of
// 128, 1000 keys, four heads together and one by one: 1 request 65 and 41 us, 8 of them 66
// and 55; 64 of them 191 and 324.)
template <typename T, int NC>
int launch_rows(const AttnArgs& a, int L, cudaStream_t s) {
  const int64_t heads = a.tokens * a.hk;
  if (a.group >= 4 && heads * ((a.group + 3) / 4) * 2 >= sm_count()) return launch_rows<T, NC, 4>(a, L, s);
  if (a.group >= 2 && heads * ((a.group + 1) / 2) * 2 >= sm_count()) return launch_rows<T, NC, 2>(a, L, s);
  return launch_rows<T, NC, 1>(a, L, s);
}

template <typename T>
int attend_rows(const AttnArgs& a, cudaStream_t s) {
  const int vecs = a.dim / Vec16<T>::N;
  int L = 1;
  while (L < vecs && L < 32) L <<= 1;
  return vecs > 32 ? launch_rows<T, 2>(a, L, s) : launch_rows<T, 1>(a, L, s);
}


// ---------------------------------------------------------- 128-row tiles -----
// Rows that read the same keys are stacked: `group` query heads of a KV head,
// for the shared prefix the tokens of all requests, for a request's own keys its
// new tokens. A block is up to 256 such rows of one KV head; a segment is a block
// with its keys, cut into tiles of 128. Scores S = Q K^T (128 x 128) and O += P V
// run on the tensor core with S, P and O in tensor memory; one thread holds one
// row, keeps its reference m and sum l in registers, and replaces S by
// P = 2^(S c - m c) in place.
//
// Two warpgroups take turns, so that one's exponentials run under the other's
// products. A tile of a block with more than 128 rows is two steps, one for each
// half of the rows; otherwise it is one. Steps go to the warpgroups in turn
// without a break between segments; a block of one half with several tiles has
// its even and its odd tiles in different hands, which are added up at its end.
//
// Work is dealt out evenly whatever the lengths: the segments form one line,
// measured in units of about what a step costs, and each of the resident CTAs
// takes an equal stretch of it. A segment cut by a stretch's end, and the two
// segments (prefix, own keys) of a row, are joined by a second kernel from fp32
// partial results and their log sums.
//
// The code of a warp that meets a new path comes from L2 at some hundred cycles
// a line, and a segment of one tile takes every path once: the walk along the
// line is one warp's work, which hands the pieces to the others through shared
// memory, and loops are unrolled only as far as they have to be (with the walk in
// every role and 128-column bodies a one-tile segment took 12000 cycles).
// Measured (bf16, 32 heads on 8 KV heads of 128, pages of 16): 16 decode requests
// behind 32768 keys 42 us, 3.7 TB/s; 128 ragged ones behind 2047 146 us, 4.5 TB/s;
// 256 behind 24576 182 us, 568 TFLOP/s; a 2048-token chunk behind 30720 1100 us, 970
// TFLOP/s, power capped (990 us alone). The first two are bound by DRAM and the
// beginnings and ends of segments, the others by a step's chain: scores, softmax
// (1700 cycles), sums, and only then the next scores, in the same tensor memory.
constexpr int kTileThreads = 384;   // 2 softmax warpgroups; a warp each issues products, loads K, loads V, walks and loads Q
constexpr int kRows = 128, kKeys = 128, kBlock = 256;
// Units of the line: a tile of a whole block, half a block's tile being half of
// that; a segment's beginning and end. (Three quarters and 16: 128 ragged decode
// requests behind 2047 keys took 205 us instead of 145, 16 behind 32768 60 instead
// of 50: the blocks of the prefix were late. With segments of 64 and more it is the
// requests' own keys that are.) Rows loaded four at a time cost half a block as
// much as a whole one, and an eighth more is what came out (extends of 64-wide
// heads 131 -> 124 us).
constexpr int kUnitTile = 32, kUnitSegment = 32;
// Registers: a softmax thread holds 64 scores and 64 words of P. The launch has 168
// per thread; the third warpgroup hands over what it does not need.
constexpr int kLaunchRegs = 168, kSoftmaxRegs = 200, kOtherRegs = 104;
static_assert(2 * kSoftmaxRegs + kOtherRegs <= 3 * kLaunchRegs, "register shares");
// A stretch is at least half a block's tile. (Four of them, with less to join: one
// request of 1000 keys on one KV head 14.0 us instead of 11.9, eight of 100 to 600
// 14.0 instead of 11.9, one of 300 11.3 instead of 11.5.)
constexpr int kMinShare = 16;

// A block and its keys: rows [blk * kBlock, ...) of the row space that starts at
// token `tok`; row x of it is token tok + x / group, head kh * group + x % group.
struct Segment {
  int req;               // request, -1: all requests over the prefix
  int tok, ntok, len;    // query tokens of the row space; the request's own keys
  int kh, blk, nblk;
  int tiles;
};

struct Start {           // a point on the line
  Segment g;
  int y;                 // units into the segment
};

// Rows of a box of queries: a few, since a piece of a single token has `group` of them.
// (Boxes of 4: 16 extends of 8 tokens behind 4096 keys 38 us instead of 36, a 2048-token
// chunk 1075 instead of 1035. Boxes of 64: no difference.)
constexpr int kQueryBox = 16;

struct TilePlan {
  int run;               // rows of a box: the largest power of two dividing the page, at most a tile; 0: rows one by one
  int run_log;
  int q_run;             // rows of a box of queries
  int q_ratio;           // a token's pitch in head pitches: queries are loaded four rows at a time; 0: in boxes
  int slope;             // units by which a request's blocks grow
  int joint;             // prefix and own keys of a request are one segment (no stacking over requests)
  int ctas;
  // rows of uncut segments (0 prefix, 1 own) that have another part
  float* whole;          // [2][tokens * hq][dim]
  float* whole_lse;      // [2][tokens * hq]
  int2* place;           // [2][tokens * hq] where the parts are: (-1, -1) whole, (first CTA | row << 16, last CTA)
  // rows of cut segments: slot 2 c holds the one that goes on at the start of CTA c's stretch, 2 c + 1 the one
  // that begins in it and goes on behind its end
  float* cut;            // [2 * ctas][kBlock][dim]
  float* cut_lse;        // [2 * ctas][kBlock]
  int32_t* used;         // [2 * ctas] whether the slot holds something
  struct CutEnd* end;    // [ctas] the cut segment that ends in CTA c's stretch, if it is all its rows have
};

// Rows [x0, x0 + nrow) of the row space at token `tok`, parts with CTAs c0 .. c.
struct CutEnd {
  int nrow, c0, tok, kh, x0;
};

// Tensor maps of the pool's K and V rows ([pool_rows, hk * dim], 128-byte
// swizzle): boxes of 64 values x `run` rows, and single rows. The queries':
// [tokens, hq, dim] in boxes of 64 values x `q_run` rows, or single rows.
struct PoolMaps {
  CUtensorMap box[2], row[2];
  CUtensorMap q;
};

__device__ __forceinline__ int tile_count(int keys) { return (keys + kKeys - 1) / kKeys; }

__device__ __forceinline__ int live_tokens(const AttnArgs& a) {
  const int n = load(a.cu + a.batch);
  return n < 0 ? 0 : (n > a.tokens ? (int)a.tokens : n);
}
// The first request's first token: not 0 where a call takes a part of a batch.
__device__ __forceinline__ int first_token(const AttnArgs& a) {
  const int n = load(a.cu);
  return n < 0 ? 0 : n;
}

// The line as a thread walks it.
struct Walk {
  const AttnArgs& a;
  const TilePlan& p;
  int live;              // where the batch's query tokens end
  Segment g;
  __device__ __forceinline__ Walk(const AttnArgs& a_, const TilePlan& p_, int live_) : a(a_), p(p_), live(live_) {}

  __device__ __forceinline__ int blocks() const { return (int)(((uint32_t)g.ntok * a.group + kBlock - 1) / kBlock); }
  // Query tokens and own keys of request r, cut to what exists.
  __device__ __forceinline__ void request(int r) {
    const int c0 = load(a.cu + r), c1 = load(a.cu + r + 1), n = load(a.lens + r);
    const int lo = c0 < 0 ? 0 : (c0 > live ? live : c0), hi = c1 < lo ? lo : (c1 > live ? live : c1);
    const int room = a.width * a.page;
    g.req = r;
    g.tok = lo;
    g.ntok = hi - lo;
    g.len = n < 0 ? 0 : (n > room ? room : n);
    g.nblk = blocks();
  }
  // Whether request r's numbers did not have to be cut.
  __device__ __forceinline__ bool fits(int r) const {
    const int c0 = load(a.cu + r), c1 = load(a.cu + r + 1);
    return c0 >= 0 && c1 >= c0 && c1 <= a.tokens && load(a.lens + r) == g.len;
  }
  __device__ __forceinline__ void prefix() {
    g.req = -1;
    g.tok = first_token(a);
    g.ntok = live > g.tok ? live - g.tok : 0;
    g.len = 0;
    g.nblk = blocks();
  }
  // Own keys that row x of the row space sees.
  __device__ __forceinline__ int row_seen(int x) const {
    if (g.req < 0) return 0;
    const int k = g.len - g.ntok + (int)a.group_div.div((uint32_t)x) + 1;
    return k < 0 ? 0 : (k > g.len ? g.len : k);
  }
  __device__ __forceinline__ int rows() const {
    const int r = g.ntok * a.group - g.blk * kBlock;
    return r < kBlock ? r : kBlock;
  }
  __device__ __forceinline__ bool pair() const { return rows() > kRows; }
  // Own keys of the block: what its last row sees.
  __device__ __forceinline__ int own_keys() const { return row_seen(g.blk * kBlock + rows() - 1); }
  // Prefix tiles of the segment come first; no tile holds both kinds of keys. A
  // block without keys still has a tile, which writes its empty rows.
  __device__ __forceinline__ int prefix_part() const { return g.req < 0 || p.joint ? tile_count(a.prefix_len) : 0; }
  __device__ __forceinline__ void size() {
    const int n = prefix_part() + tile_count(own_keys());
    g.tiles = n < 1 ? 1 : n;
  }
  // Units of the segment and of the first m (whole) blocks of a head. A block's
  // own keys grow by 256 / group tokens from one to the next; taken as a straight
  // line, the sums have a closed form, and where the line is off the true count
  // only the balance is. A segment has fewer than 2^30 units (2^30 keys, blocks of
  // 2^30 rows), a head and the line more than 32 bits hold: many queries count
  // as if each block saw 256 / group keys more than the one before, on few keys too.
  __device__ __forceinline__ int base_units() const {
    const int more = g.len - g.ntok;
    return prefix_part() * kUnitTile + (more > 0 ? more / (kKeys / kUnitTile) : 0);
  }
  __device__ __forceinline__ int slope() const { return g.req < 0 ? 0 : p.slope; }
  __device__ __forceinline__ int units() const {
    const int u = base_units() + slope() * (g.blk + 1);
    return kUnitSegment + (pair() ? u : u / 2 + (p.run ? 0 : u / 8));
  }
  __device__ __forceinline__ int64_t units_before(int m) const {
    return (int64_t)m * (kUnitSegment + base_units()) + (int64_t)m * (m + 1) / 2 * slope();
  }
  // Tiles of the segment that begin before unit y of it: any rule will do that
  // only grows with y, from 0 to all of them.
  __device__ __forceinline__ int tile_at(int y) const {
    const int u = units();
    if (y >= u) return g.tiles;
    if (y <= kUnitSegment) return 0;
    const int i = (int)__fmul_rn((float)(y - kUnitSegment), __fdiv_rn((float)g.tiles, (float)(u - kUnitSegment)));
    return i < g.tiles ? i : g.tiles;
  }
  // Units of one head of the row space.
  __device__ __forceinline__ int64_t head_units() {
    if (g.nblk == 0) return 0;
    g.blk = g.nblk - 1;
    return units_before(g.blk) + units();
  }
  // To the segment that holds unit y of the row space, `one` units a head; returns the unit in the segment.
  __device__ __forceinline__ int seek(int64_t y, int64_t one) {
    g.kh = (int)(y / one);
    y -= g.kh * one;
    int lo = 0, hi = g.nblk;  // the last block that begins at or before y
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (units_before(mid) <= y)
        lo = mid;
      else
        hi = mid;
    }
    g.blk = lo;
    size();
    return (int)(y - units_before(lo));
  }
  // The next segment of the line.
  __device__ __forceinline__ void next() {
    if (++g.blk >= g.nblk) {
      g.blk = 0;
      if (++g.kh >= a.hk) {
        g.kh = 0;
        int r = g.req;
        do {
          if (++r >= a.batch) return;  // behind the line's end: not walked
          request(r);
        } while (g.nblk == 0);
      }
    }
    size();
  }
};

// Units of one head of the prefix's row space.
__device__ __forceinline__ int64_t prefix_head_units(Walk& w) {
  if (w.p.joint || w.a.prefix_len == 0) return 0;
  w.prefix();
  return w.head_units();
}

// A piece as the other warps get it.
struct alignas(16) Piece {
  int n, off, np, own;   // tiles (0: none are left), the first one's number, prefix tiles, own keys of the block
  int x0, nrow, tok, kh; // rows
  int req, more, len;    // row x sees own keys below more + x / group + 1 (at most len)
  int kind;              // 1: the rows' only segment, in one piece; 2: its last piece; 4: the segment in one piece
  int c0;                // first CTA of the segment
  int tail[2], tail_keys[2];  // the last tile of the prefix and of the own keys, and their sixteens
};
constexpr int kPieces = 4;

// Keys of tile i of a piece: how many, with `own` own keys in sight; the first one's index among its kind.
__device__ __forceinline__ int piece_key0(const Piece& g, int i) {
  const int ti = g.off + i;
  return (ti < g.np ? ti : ti - g.np) * kKeys;
}
__device__ __forceinline__ int piece_keys(const Piece& g, int i, int prefix_len, int own) {
  const int rest = (g.off + i < g.np ? prefix_len : own) - piece_key0(g, i);
  return rest < 0 ? 0 : (rest < kKeys ? rest : kKeys);
}

// Keys of a tile as the products take them: sixteens, at least one.
__device__ __forceinline__ int sixteens(int keys) { return keys <= 16 ? 1 : (keys + 15) >> 4; }

__device__ __forceinline__ int tile_sixteens(const Piece& g, int i) {
  return i == g.tail[0] ? g.tail_keys[0] : (i == g.tail[1] ? g.tail_keys[1] : kKeys / 16);
}

__device__ __forceinline__ int64_t share(int64_t total, int ctas) {
  const int64_t n = (total + ctas - 1) / ctas;
  return n < kMinShare ? kMinShare : n;
}

// A wait gives up after so many turns (TileShared::quit) and raises `quit`, which
// ends every other wait of the CTA.
__device__ __forceinline__ bool long_wait(uint64_t* bar, uint32_t parity, volatile int* quit) {
  const int turns = quit[1];
#pragma unroll 1
  for (int i = 0; i < turns; ++i) {
    if (pipe::bar_try(bar, parity)) return true;
    if (*quit) return false;
  }
  *quit = 1;
  return false;
}
// Of the thread that issues the products, whose barriers are mostly through: a
// wait on such a one costs some 200 cycles, a test 50.
__device__ __forceinline__ bool thread_wait(uint64_t* bar, uint32_t parity, volatile int* quit) {
  return pipe::bar_test(bar, parity) || long_wait(bar, parity, quit);
}
// Every lane of the warp gets the same answer.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* quit) {
  return __all_sync(0xffffffffu, long_wait(bar, parity, quit)) != 0;
}

constexpr int kBehind = 3 * 1024;  // bytes of shared memory behind the tiles (TileShared)
template <int DP>
struct TileShape {
  static constexpr int tile = kRows * DP * 2;                     // bytes of a Q, K or V tile
  // K and V tiles in flight, a ring each: a warp that waits for a stage has seen all
  // of its turns (a barrier tells only odd ones from even ones)
  static constexpr uint32_t ks = DP == 128 ? 2 : 6, vs = DP == 128 ? 3 : 6;
  static constexpr int stages = ks + vs;
  static constexpr int data = (2 + stages) * tile;
  static constexpr int smem = data + kBehind;
};

// Shared memory behind the tiles.
struct TileShared {
  float m[kRows], l[kRows];         // what one warpgroup hands to the other
  alignas(16) int32_t rows[2][kKeys];  // pool rows of the K and the V tile being loaded
  uint64_t full[12], empty[12], q_full[2], q_empty[2], s_full[2], p_full[2], o_full[2], o_empty[2], handed, taken;
  uint64_t piece_full[kPieces], piece_empty[kPieces];
  Piece piece[kPieces];
  Start first;                      // where this CTA's stretch starts
  int64_t total, unit, wsum[kTileThreads / 32];  // units of the line, of a stretch, of each warp's requests
  uint32_t tmem;
  int quit[2];                      // a wait gave up; after so many turns: more than the CTA's stretch can take
  int bad;                          // a page was outside the pool
};
static_assert(sizeof(TileShared) <= kBehind, "shared memory behind the tiles");

// 16 words of P from 32 scores, their sum and their maximum (with `top`). P is
// rounded to the type of the values, the only one that the tensor core multiplies
// with them: each by up to half a step (2^-8 of it in bf16, 2^-11 in fp16, and below
// 2^-14 half of fp16's smallest step), independently. The sum takes them unrounded, in
// 32 bits, as are scores, maxima, O and partial results. Beside the rounding of the
// result that leaves o 0.0023 of its norm off in bf16 and 0.00029 in fp16, where the
// exact o rounded is 0.0017 and 0.00021 off; lse 5e-8. (Two
// scores to an instruction, fma.f32x2 and add.f32x2, took longer: 1550 cycles a
// tile instead of 1290.)
template <typename T>
__device__ __forceinline__ float exp32(const uint32_t* x, uint32_t* w, float c, float mc, float& top) {
  float sum[4] = {0.f, 0.f, 0.f, 0.f}, t[2] = {top, top};
#pragma unroll
  for (int e = 0; e < 32; e += 2) {
    const float s0 = __uint_as_float(x[e]), s1 = __uint_as_float(x[e + 1]);
    const float p0 = tc::ex2(fmaf(s0, c, -mc)), p1 = tc::ex2(fmaf(s1, c, -mc));
    sum[(e >> 1) & 3] += p0 + p1;
    t[(e >> 1) & 1] = fmaxf(fmaxf(t[(e >> 1) & 1], s0), s1);
    w[e >> 1] = Vec16<T>::pack2(p0, p1);
  }
  top = fmaxf(t[0], t[1]);
  return (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

// A tile in two passes: where keys of it are hidden from some row of the warp
// (those from column `cols` on), or its maximum moves the reference of one.
// Maximum first, then O and l to the new reference, then P. Columns from `end` on
// are no keys of any row, and no product takes them.
template <typename T, int DP>
__device__ __noinline__ float2 careful_tile(uint32_t ts, uint32_t to, float c, int cols, int end, bool on, bool has_o,
                                            float m, float l) {
  uint32_t x[32], w[16];
  float top = m, seen = -INFINITY, mc = 0.f;
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
#pragma unroll 1
    for (int k = 0; k < end; k += 32) {
      tc::ld32(ts + k, x);
      tc::wait_ld(x);
      const int left = cols - k;
      if (__any_sync(0xffffffffu, left < 32)) {
#pragma unroll
        for (int e = 0; e < 32; ++e) x[e] = e < left ? x[e] : 0xff800000u;
      }
      if (pass == 0) {
#pragma unroll
        for (int e = 0; e < 32; ++e) top = fmaxf(top, __uint_as_float(x[e]));
      } else {
        // P's words overlay the scores from the left, behind the reading
        l += exp32<T>(x, w, c, mc, seen);
        tc::st16(ts + k / 2, w);
      }
    }
    if (pass == 0) {
      const bool move = on && ((top - m) * c > 8.f || (m == -INFINITY && top > -INFINITY));
      if (__any_sync(0xffffffffu, move)) {
        const float f = !move ? 1.f : (m == -INFINITY ? 0.f : tc::ex2((m - top) * c));
        if (move) m = top;
        l *= f;
#pragma unroll 1
        for (int k = 0; has_o && k < DP; k += 32) {
          tc::ld32(to + k, x);
          tc::wait_ld(x);
#pragma unroll
          for (int e = 0; e < 32; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) * f);
          tc::st32(to + k, x);
        }
      }
      mc = m == -INFINITY ? 0.f : m * c;
    }
  }
  tc::wait_st();
  return make_float2(m, l);
}

// One row's share of a tile: the scores at tensor memory `ts` (128 columns) become
// 16-bit P there, (m, l) follow, and O at `to` (when it holds something) where the
// reference moves. What a lane without a row (!on) computes is not read.
//
// P is taken relative to the reference m that the row has, or to the largest of
// its first 32 scores, while the tile's maximum is found on the way: one pass over
// the scores, and no branch in it, so that the exponentials of one part run under
// the loads, sums and conversions of another (1300 cycles; 1900 in a loop over 64
// columns; 1024 are the exponentials). Only where the maximum turns out 8 binary
// places ahead is the reference moved and the tile done again; until then P
// exceeds 1, by 2^8 at most, which sums and 16-bit P hold as well as they hold 1.
template <typename T, int DP>
__device__ __forceinline__ void softmax_tile(uint32_t ts, uint32_t to, float c, int cols, int end, bool on, bool has_o,
                                             float& m, float& l) {
  bool again = __any_sync(0xffffffffu, cols < kKeys);
  if (!again) {
    uint32_t x[32], y[32], w[64];
    tc::ld32(ts, x);
    tc::wait_ld(x);
    tc::ld32(ts + 32, y);
    if (__any_sync(0xffffffffu, m == -INFINITY)) {
      float first = -INFINITY;
#pragma unroll
      for (int e = 0; e < 32; ++e) first = fmaxf(first, __uint_as_float(x[e]));
      if (m == -INFINITY) m = first;
      again = __any_sync(0xffffffffu, on && m == -INFINITY);
    }
    const float mc = m == -INFINITY ? 0.f : m * c;
    float top = m, sum;
    sum = exp32<T>(x, w, c, mc, top);
    tc::wait_ld(y);
    tc::ld32(ts + 64, x);
    sum += exp32<T>(y, w + 16, c, mc, top);
    tc::wait_ld(x);
    tc::ld32(ts + 96, y);
    sum += exp32<T>(x, w + 32, c, mc, top);
    tc::wait_ld(y);
    sum += exp32<T>(y, w + 48, c, mc, top);
    again = again || __any_sync(0xffffffffu, on && (top - m) * c > 8.f);
    if (!again) {
      l += sum;
      tc::st32(ts, w);
      tc::st32(ts + 32, w + 32);
      tc::wait_st();
    }
  }
  if (again) {
    const float2 r = careful_tile<T, DP>(ts, to, c, cols, end, on, has_o, m, l);
    m = r.x;
    l = r.y;
  }
}

// ROWS: pages of less than eight rows, loaded four rows at a time.
template <typename T, int DP, bool ROWS>
__global__ void __launch_bounds__(kTileThreads, 1) attend_tile_kernel(const AttnArgs a, const TilePlan p,
                                                                     const __grid_constant__ PoolMaps maps) {
  using Shape = TileShape<DP>;
  constexpr uint32_t KS = Shape::ks, VS = Shape::vs;
  extern __shared__ __align__(1024) unsigned char smem[];
  TileShared& sh = *reinterpret_cast<TileShared*>(smem + Shape::data);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < Shape::stages; ++i) {
      pipe::bar_init(sh.full + i, 1);
      pipe::bar_init(sh.empty + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      pipe::bar_init(sh.q_full + i, 1);
      pipe::bar_init(sh.q_empty + i, 1);
      pipe::bar_init(sh.s_full + i, 1);
      pipe::bar_init(sh.p_full + i, 4);
      pipe::bar_init(sh.o_full + i, 1);
      pipe::bar_init(sh.o_empty + i, 4);
    }
    for (int i = 0; i < kPieces; ++i) {
      pipe::bar_init(sh.piece_full + i, 1);
      pipe::bar_init(sh.piece_empty + i, 12);  // 8 softmax warps, both loads, scores and sums of the products
    }
    pipe::bar_init(&sh.handed, 4);
    pipe::bar_init(&sh.taken, 4);
    pipe::bar_init_fence();
    sh.quit[0] = (tc::smem_addr(smem) & 1023u) != 0;  // the swizzle counts from 1024-byte patterns
    sh.bad = 0;
  }
  if (warp == 8) {
    tc::alloc(&sh.tmem, 512);
    tc::relinquish();
  }
  if (warp == 9 && lane < 2) {
    tc::prefetch_map(maps.box + lane);
    tc::prefetch_map(maps.row + lane);
  }
  if (warp == 11 && lane == 0) tc::prefetch_map(&maps.q);
  grid_dep_wait();
  grid_dep_launch();

  // The line: units of every request (a run of requests per thread), their sums,
  // and the place where this CTA's stretch starts.
  const int live = live_tokens(a);
  {
    Walk w(a, p, live);
    // not in the tiles' memory: tensor copies write that, and nothing would order them behind these words
    int64_t* wsum = sh.wsum;
    const int per = (a.batch + kTileThreads - 1) / kTileThreads;
    const int r0 = tid * per < a.batch ? tid * per : a.batch, r1 = r0 + per < a.batch ? r0 + per : a.batch;
    int64_t mine = 0, one = 0;  // units of the run, of one head of its last request
    for (int r = r0; r < r1; ++r) {
      w.request(r);
      one = w.head_units();
      mine += one * a.hk;
      if (blockIdx.x == 0 && !w.fits(r)) atomicOr(&g_attn_status, 1u);
    }
    int64_t x = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, x, d);
      if (lane >= d) x += y;
    }
    if (lane == 31) wsum[warp] = x;
    const int64_t pre_one = prefix_head_units(w), pre = pre_one * a.hk;
    __syncthreads();
    int64_t at = pre + x - mine, total = pre;
#pragma unroll
    for (int i = 0; i < kTileThreads / 32; ++i) {
      const int64_t v = wsum[i];
      if (i < warp) at += v;
      total += v;
    }
    const int64_t unit = share(total, p.ctas), x0 = blockIdx.x * unit;
    if (tid == 0) {
      sh.total = total;
      sh.unit = unit;
      // a wait may last as long as a piece; a unit of the line takes 70 ns, a turn 20 and more
      sh.quit[1] = (1 << 24) + 64 * (unit < 1 << 24 ? (int)unit : 1 << 24);
      if (x0 < pre) {
        w.prefix();
        sh.first.y = w.seek(x0, pre_one);
        sh.first.g = w.g;
      }
    }
    for (int r = r0; r < r1; ++r) {
      if (per > 1) {
        w.request(r);
        one = w.head_units();
      }
      if (x0 >= at && x0 < at + one * a.hk) {
        w.request(r);
        sh.first.y = w.seek(x0 - at, one);
        sh.first.g = w.g;
      }
      at += one * a.hk;
    }
    if (tid < 2) p.used[2 * blockIdx.x + tid] = 0;
    if (tid == 2) p.end[blockIdx.x].nrow = 0;
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
  }
  const uint32_t tmem = sh.tmem;
  const int64_t unit = sh.unit, x0 = blockIdx.x * unit, x1 = sh.total - x0 < unit ? sh.total : x0 + unit;
  volatile int* quit = sh.quit;
  const float c = fabsf(a.scale) * 1.4426950408889634f;
  if (x0 < x1 && !*quit) {
    // Reads piece number `i` of the CTA; whoever has read it says so with done_piece.
    const auto next_piece = [&](uint32_t i) { return warp_wait(sh.piece_full + i % kPieces, (i / kPieces) & 1, quit); };
    const auto done_piece = [&](uint32_t i) {
      __syncwarp();
      if (lane == 0) pipe::bar_arrive(sh.piece_empty + i % kPieces);
    };
    const uint32_t base = tc::smem_addr(smem), ring = base + 2 * Shape::tile;
    if (warp < 8) {
      tc::regs_up<kSoftmaxRegs>();
      // ------------------------------------------------ softmax warpgroups ----
      const int t = warp >> 2, r = tid & (kRows - 1);
      const uint32_t row = (uint32_t)((warp & 3) * 32) << 16;
      const uint32_t ts = tmem + row + t * 128, to = tmem + row + 256 + t * 128;
      uint32_t n_s = 0, n_handed = 0, n_o[2] = {0, 0}, step = 0;
      for (uint32_t pi = 0;; ++pi) {
        if (!next_piece(pi)) break;
        const Piece& g = sh.piece[pi % kPieces];
        const int n = g.n;
        if (n == 0) break;
        const int u0 = step & 1, half = t ^ u0;                 // half of the block, or first tile
        const bool two = g.nrow > kRows, shared = !two && n > 1;  // shared: both warpgroups hold tiles of the rows
        step += two ? 2 * n : n;
        const uint32_t turn = n_o[t], turn_other = n_o[t ^ 1];
        n_o[u0] += 1;
        n_o[u0 ^ 1] += two || shared;
        if (!two && !shared && half) {
          done_piece(pi);
          continue;
        }
        const int brow = (two ? half * kRows : 0) + r, x = g.x0 + brow;  // this thread's row: of the block, of the row space
        const bool on = brow < g.nrow;
        const bool warp_on = __any_sync(0xffffffffu, on);
        const int jt = (int)a.group_div.div((uint32_t)x);
        int see = g.more + jt + 1;
        see = see < 0 ? 0 : (see > g.len ? g.len : see);
        float m = -INFINITY, l = 0.f;                          // reference, sum relative to it
        bool ok = true;
#pragma unroll 1
        for (int i = two ? 0 : half; i < n; i += two ? 1 : 2) {
          const int cols = on ? piece_keys(g, i, a.prefix_len, see) : kKeys;
          const int keys = piece_keys(g, i, a.prefix_len, g.own), end = keys > 0 ? keys : 1;
          if (!(ok = warp_wait(sh.s_full + t, n_s & 1, quit))) break;
          ++n_s;
          tc::fence_after();
          if (warp_on) softmax_tile<T, DP>(ts, to, c, cols, end, on, two ? i > 0 : i >= 2, m, l);
          tc::fence_before();
          __syncwarp();
          if (lane == 0) pipe::bar_arrive(sh.p_full + t);
        }
        if (!ok) break;
        // -------------------------------------------------------- results ----
        // The warpgroup that has the last tile takes over the other's maximum and
        // sum; it can read both results in tensor memory.
        float w0 = 1.f, w1 = 0.f;
        if (shared) {
          const uint32_t turn_h = n_handed++;
          if (half != ((n - 1) & 1)) {
            if (turn_h > 0 && !warp_wait(&sh.taken, (turn_h - 1) & 1, quit)) break;
            sh.m[r] = m;
            sh.l[r] = l;
            __syncwarp();
            if (lane == 0) pipe::bar_arrive(&sh.handed);
            done_piece(pi);
            continue;
          }
          if (!warp_wait(&sh.handed, turn_h & 1, quit)) break;
          const float mb = sh.m[r], lb = sh.l[r];
          __syncwarp();
          if (lane == 0) pipe::bar_arrive(&sh.taken);
          const float ref = fmaxf(m, mb);
          w0 = m == -INFINITY ? 0.f : tc::ex2((m - ref) * c);
          w1 = mb == -INFINITY ? 0.f : tc::ex2((mb - ref) * c);
          // a sum that is not a number stays so, whatever its maximum
          l = (l == l ? w0 * l : l) + (lb == lb ? w1 * lb : lb);
          m = ref;
          if (!warp_wait(sh.o_full + (t ^ 1), turn_other & 1, quit)) break;
        }
        if (!warp_wait(sh.o_full + t, turn & 1, quit)) break;
        tc::fence_after();
        if (warp_on) {
          const bool direct = g.kind & 1, whole = g.kind & 4;
          const int u = g.req < 0 ? 0 : 1;
          const int64_t all = a.tokens * a.hq;
          const int64_t grow = ((int64_t)g.tok + jt) * a.hq + g.kh * a.group + (x - jt * a.group);
          const int slot = 2 * blockIdx.x + (g.off == 0 ? 1 : 0);
          const int64_t part = whole ? u * all + grow : (int64_t)slot * kBlock + brow;
          float* dst = (whole ? p.whole : p.cut) + part * a.dim;
          const float inv = l == 0.f ? 0.f : 1.f / l;
          if (on) {
            const float ls = l == 0.f ? -INFINITY : m * c + log2f(l);
            if (direct) {
              if (a.lse) a.lse[grow] = ls * 0.6931471805599453f;
            } else {
              (whole ? p.whole_lse : p.cut_lse)[part] = ls;
              if (!whole && brow == 0) p.used[slot] = 1;
              if ((g.kind & 2) && !p.joint)
                p.place[u * all + grow] = whole ? make_int2(-1, -1) : make_int2(g.c0 | brow << 16, blockIdx.x);
              if ((g.kind & 2) && p.joint && brow == 0)
                p.end[blockIdx.x] = CutEnd{g.nrow, g.c0, g.tok, g.kh, g.x0};
            }
          }
          w0 *= inv;
          w1 *= inv;
#pragma unroll 1
          for (int k = 0; k < a.dim; k += 32) {
            uint32_t o[32], o2[32];
            tc::ld32(to + k, o);
            if (shared) tc::ld32(tmem + row + 256 + (t ^ 1) * 128 + k, o2);
            tc::wait_ld(o);
            if (shared) {
              tc::wait_ld(o2);
#pragma unroll
              for (int e = 0; e < 32; ++e)
                o[e] = __float_as_uint(__uint_as_float(o[e]) * w0 + __uint_as_float(o2[e]) * w1);
            } else {
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * w0);
            }
            if (l == 0.f) {
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = 0u;
            }
            if (!on) continue;
            if (direct) {
              char* to_row = a.out + (grow * a.dim + k) * 2;
#pragma unroll
              for (int e = 0; e < 32; e += 8)
                if (k + e < a.dim)
                  *reinterpret_cast<uint4*>(to_row + e * 2) = Vec16<T>::pack(reinterpret_cast<const float*>(o) + e);
            } else {
#pragma unroll
              for (int e = 0; e < 32; e += 4)
                if (k + e < a.dim) *reinterpret_cast<uint4*>(dst + k + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
            }
          }
        }
        tc::fence_before();
        __syncwarp();
        if (lane == 0) {
          pipe::bar_arrive(sh.o_empty + t);
          if (shared) pipe::bar_arrive(sh.o_empty + (t ^ 1));
        }
        done_piece(pi);
      }
    } else {
    tc::regs_down<kOtherRegs>();
    if (warp == 8) {
      // -------------------------------------------------------- products ----
      // One thread. Step s runs on S, P and O number s & 1; its scores are issued
      // right after the P V of step s - 2. A lone thread takes five cycles and more
      // for an instruction, so what can be done before P arrives is. (The scores'
      // products in a loop: a 2048-token chunk 1205 us instead of 1140. The sums' are:
      // unrolled 256 requests on one prefix took 183 us instead of 180.)
      if (tc::elect()) {
        const uint32_t id_s = tc::idesc(Vec16<T>::bf16, kRows, 0, false, a.scale < 0.f);
        const uint32_t id_o = tc::idesc(Vec16<T>::bf16, kRows, a.dim, true);
        const int ks = a.dim / 16;
        const uint64_t qdesc = tc::desc(base, 16, 1024), kdesc = tc::desc(ring, 16, 1024),
                       vdesc = tc::desc(ring + KS * Shape::tile, kKeys * 128, 1024);
        uint32_t n_o0 = 0, n_o1 = 0, n_q = 0, id = 0;                   // uses of the O's, Q tiles
        // the scores' place: piece, tile of it, step of the tile; the sums' place
        uint32_t qp = 0, wp = 0;
        int qi = 0, qsub = 0, qn = 0, wi = 0, wsub = 0, wn = 0, kk = 0;
        uint32_t k_st = 0, k_turn = 0, v_st = 0, v_turn = 0;    // ring stages and the parity of their turns
        bool qtwo = false, wtwo = false, have = false;          // have: the scores' piece is known
        for (uint32_t s = 0;; ++s) {                            // sums of step s - 2, scores of step s
          const uint32_t l2 = s & 1;
          bool ready = false;                                   // the scores' operands are there
          const auto open_piece = [&] {
            const Piece& g = sh.piece[qp % kPieces];
            qn = g.n;
            qtwo = g.nrow > kRows;
            have = true;
          };
          if (s >= 2) {
            if (wi == 0 && wsub == 0) {
              if (!thread_wait(sh.piece_full + wp % kPieces, (wp / kPieces) & 1, quit)) break;
              wn = sh.piece[wp % kPieces].n;
              if (wn == 0) break;
              wtwo = sh.piece[wp % kPieces].nrow > kRows;
            }
            const bool fresh = wi < (wtwo ? 1 : 2), last = wi >= wn - (wtwo ? 1 : 2), tile_done = !wtwo || wsub;
            if (wsub == 0) {
              kk = tile_sixteens(sh.piece[wp % kPieces], wi);
              if (!thread_wait(sh.full + KS + v_st, v_turn, quit)) break;
            }
            if (fresh) {
              const uint32_t uses = l2 ? n_o1 : n_o0;
              if (uses > 0 && !thread_wait(sh.o_empty + l2, (uses - 1) & 1, quit)) break;
              n_o0 += l2 ^ 1;
              n_o1 += l2;
            }
            if (!have && pipe::bar_test(sh.piece_full + qp % kPieces, (qp / kPieces) & 1)) open_piece();
            ready = have && qn > 0 && (qsub || pipe::bar_test(sh.full + k_st, k_turn)) &&
                    (qi > 0 || pipe::bar_test(sh.q_full + ((n_q + qsub) & 1), ((n_q + qsub) >> 1) & 1));
            const uint64_t vd = vdesc + v_st * (Shape::tile >> 4);
            const uint32_t o = tmem + 256 + l2 * 128, pa = tmem + l2 * 128;
            if (!thread_wait(sh.p_full + l2, ((s - 2) >> 1) & 1, quit)) break;
            tc::fence_after();
#pragma unroll 1
            for (int j = 0; j < kk; ++j) tc::mma_ts(o, pa + j * 8, vd + j * (2048 >> 4), id_o, !fresh || j > 0);
            if (tile_done) tc::commit(sh.empty + KS + v_st);
            if (last) tc::commit(sh.o_full + l2);
            wsub = !tile_done;
            if (tile_done) {
              if (++v_st == VS) {
                v_st = 0;
                v_turn ^= 1;
              }
              if (++wi == wn) {
                wi = 0;
                pipe::bar_arrive(sh.piece_empty + wp++ % kPieces);
              }
            }
          }
          if (!ready) {
            if (!have) {
              if (!thread_wait(sh.piece_full + qp % kPieces, (qp / kPieces) & 1, quit)) break;
              open_piece();
            }
            if (qn == 0) continue;                              // behind the last piece
            if (qi == 0 && !thread_wait(sh.q_full + ((n_q + qsub) & 1), ((n_q + qsub) >> 1) & 1, quit)) break;
            if (!thread_wait(sh.full + k_st, k_turn, quit)) break;
          }
          if (qsub == 0) id = id_s | (uint32_t)(2 * tile_sixteens(sh.piece[qp % kPieces], qi)) << 17;
          const uint64_t qd = qdesc + ((n_q + qsub) & 1) * (Shape::tile >> 4), kd = kdesc + k_st * (Shape::tile >> 4);
#pragma unroll
          for (int j = 0; j < DP / 16; ++j) {                   // 32 bytes on, or to the next 64 values
            const int at = (j & 3) * 2 + (j >> 2) * (kRows * 128 >> 4);
            if (j < ks) tc::mma_ss(tmem + l2 * 128, qd + at, kd + at, id, j > 0);
          }
          const bool tile_done = !qtwo || qsub, done = tile_done && qi == qn - 1;
          tc::commit(sh.s_full + l2);
          if (tile_done) tc::commit(sh.empty + k_st);
          qsub = !tile_done;
          if (tile_done) {
            if (++k_st == KS) {
              k_st = 0;
              k_turn ^= 1;
            }
            ++qi;
          }
          if (done) {
            tc::commit(sh.q_empty + (n_q & 1));
            if (qtwo) tc::commit(sh.q_empty + ((n_q + 1) & 1));
            n_q += qtwo ? 2 : 1;
            qi = 0;
            have = false;
            pipe::bar_arrive(sh.piece_empty + qp++ % kPieces);
          }
        }
      }
      __syncwarp();
    } else if (warp < 11) {
      // --------------------------------------------------- loads of K, V ----
      // Whole pages as boxes; the rest of a tile, or a tile with a page outside
      // the pool, four rows at a time, with zeros for what is not there (a slot
      // behind the end may hold anything). Only the sixteens that the products
      // take are loaded. (Four-row gathers move a tile in about twice a box's time:
      // 128 ragged decode requests 226 us on pages of one, 126 on pages of 16. By
      // 16-byte copies of the whole warp it was 311.)
      constexpr int PN = DP / 64;                               // 64-value panels of a row
      constexpr uint32_t kPanel = kRows * 128;
      const int kv = warp - 9, none = (int)a.pool_rows;         // none: a row outside the map
      const CUtensorMap *box = maps.box + kv, *one_row = maps.row + kv;
      int32_t* rows = sh.rows[kv];
      const uint32_t turns = kv ? VS : KS, stage0 = kv ? KS : 0;
      uint32_t pos = 0;
      bool ok = true;
      for (uint32_t pi = 0; ok; ++pi) {
        if (!next_piece(pi)) break;
        const Piece& g = sh.piece[pi % kPieces];
        const int n = g.n, x = g.kh * a.dim;
        if (n == 0) break;
#pragma unroll 1
        for (int i = 0; i < n; ++i, ++pos) {
          const int k0 = piece_key0(g, i) + (g.off + i < g.np ? 0 : a.prefix_len), valid = piece_keys(g, i, a.prefix_len, g.own);
          int boxes = 0;
          if (!ROWS) {
            boxes = valid >> p.run_log;
            int32_t y = 0;
            if (lane < boxes) {
              const int64_t sl = key_slot(a, g.req, k0 + (lane << p.run_log));
              y = sl < 0 || sl + p.run > a.pool_rows ? -1 : (int32_t)sl;
            }
            if (__any_sync(0xffffffffu, y < 0)) boxes = 0;
            if (lane < boxes) rows[lane] = y;
          }
          const int quad0 = (boxes << p.run_log) >> 2, quads = sixteens(valid) * 4;
          const auto look = [&](int k) {                        // rows behind the boxes' entries
            const bool is = k < valid;
            const int64_t sl = is ? key_slot(a, g.req, k0 + k) : -1;
            if (is && sl < 0) sh.bad = 1;
            rows[k] = sl < 0 ? none : (int32_t)sl;
          };
          if (ROWS) {                                           // every tile: four lookups in flight
            if (lane < quads) {
#pragma unroll
              for (int j = 0; j < 4; ++j) look(lane * 4 + j);
            }
          } else {                                              // a tail, mostly less than 32 rows: little code
#pragma unroll 1
            for (int k = quad0 * 4 + lane; k < quads * 4; k += 32) look(k);
          }
          const uint32_t st = stage0 + pos % turns;
          __syncwarp();
          if (pos >= turns && !(ok = warp_wait(sh.empty + st, (pos / turns - 1) & 1, quit))) break;
          if (tc::elect()) {
            uint32_t dst = ring + st * Shape::tile;
            pipe::bar_expect_tx(sh.full + st, (uint32_t)quads * 4 * DP * 2);
#pragma unroll 1
            for (int b = 0; b < boxes; ++b, dst += p.run * 128) {
              const int yb = rows[b];
#pragma unroll
              for (int pn = 0; pn < PN; ++pn) tc::load_box(dst + pn * kPanel, box, x + pn * 64, yb, sh.full + st);
            }
#pragma unroll 1
            for (int b = quad0; b < quads; ++b, dst += 512) {
              const int4 z = *reinterpret_cast<const int4*>(rows + b * 4);
#pragma unroll
              for (int pn = 0; pn < PN; ++pn) tc::load_rows(dst + pn * kPanel, one_row, x + pn * 64, z, sh.full + st);
            }
          }
          __syncwarp();
        }
        done_piece(pi);
      }
      // copies must not outlive the CTA, and whoever waits for the last of them may still give up
      for (uint32_t q = pos > turns ? pos - turns : 0; q < pos; ++q)
        (void)pipe::bar_wait(sh.full + stage0 + q % turns, (q / turns) & 1);
    } else {
      // ------------------------------------------ the walk, loads of Q ----
      // Row x of a block is head x % group of token x / group: boxes of whole groups
      // over a few tokens (or of a part of a group) where that makes a power of two
      // of rows, else four rows at a time.
      constexpr int PN = DP / 64;
      constexpr uint32_t kPanel = kRows * 128;
      Walk w(a, p, live);
      w.g = sh.first.g;
      int y = sh.first.y;                                       // units into the segment
      int64_t left = x1 - x0, at = x0 - y;                      // left of the stretch; the segment's start
      uint32_t n_q = 0, pi = 0;
      bool ok = true;
#pragma unroll 1
      while (true) {
        const int units = left > 0 ? w.units() : 0;
        const int off = left > 0 && y > 0 ? w.tile_at(y) : 0;
        const int end = left <= 0 ? 0 : (left >= units - y ? w.g.tiles : w.tile_at(y + (int)left));
        if (left > 0 && end == off) {                           // no tile of the segment begins here
          left -= units - y;
          at += units;
          y = 0;
          if (left > 0) w.next();
          continue;
        }
        const int slot = pi % kPieces, nrow = w.rows();
        if (pi >= kPieces && !(ok = warp_wait(sh.piece_empty + slot, (pi / kPieces - 1) & 1, quit))) break;
        if (lane == 0) {
          Piece& g = sh.piece[slot];
          g.n = end - off;
          if (left > 0) {
            const bool whole = end - off == w.g.tiles;
            g.off = off;
            const int np = w.prefix_part(), own = w.own_keys();
            g.np = np;
            g.own = own;
            g.tail[0] = np - 1 - off;
            g.tail_keys[0] = sixteens(a.prefix_len - (np - 1) * kKeys);
            g.tail[1] = w.g.tiles - 1 - off;
            g.tail_keys[1] = sixteens(own - (w.g.tiles - 1 - np) * kKeys);
            g.x0 = w.g.blk * kBlock;
            g.nrow = nrow;
            g.tok = w.g.tok;
            g.kh = w.g.kh;
            g.req = w.g.req;
            g.more = w.g.len - w.g.ntok;
            g.len = w.g.len;
            g.kind = (whole && p.joint ? 1 : 0) | (end == w.g.tiles ? 2 : 0) | (whole ? 4 : 0);
            if (!whole) {
              int c0 = (int)(at / unit);                        // the stretch in which its first tile begins
              const auto before = [&](int64_t v) { return w.tile_at(v < INT_MAX ? (int)v : INT_MAX); };
              while (c0 < (int)blockIdx.x && before((c0 + 1) * unit - at) == 0) ++c0;
              g.c0 = c0;
            }
          }
        }
        __syncwarp();
        if (lane == 0) pipe::bar_arrive(sh.piece_full + slot);
        if (left <= 0) break;
        ++pi;
        const int nq = nrow > kRows ? 2 : 1, head0 = w.g.kh * a.group;
        for (int b = 0; b < nq; ++b, ++n_q) {                   // whole boxes of the rows that exist: a product's rows do not mix
          const int buf = n_q & 1, here = nrow - b * kRows < kRows ? nrow - b * kRows : kRows;
          const int xb = w.g.blk * kBlock + b * kRows;
          uint32_t dst = base + buf * Shape::tile;
          if (n_q >= 2 && !(ok = warp_wait(sh.q_empty + buf, ((n_q >> 1) - 1) & 1, quit))) break;
          if (p.q_ratio > 0) {
            int4 z;
            int* zj = &z.x;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int x = xb + lane * 4 + j, jt = (int)a.group_div.div((uint32_t)x);
              zj[j] = (w.g.tok + jt) * p.q_ratio + head0 + x - jt * a.group;
            }
            if (tc::elect()) pipe::bar_expect_tx(sh.q_full + buf, (uint32_t)((here + 3) / 4 * 512 * PN));
            __syncwarp();
#pragma unroll 1
            for (int q = 0; q < (here + 3) / 4; ++q, dst += 512) {
              const int4 y4 = make_int4(__shfl_sync(0xffffffffu, z.x, q), __shfl_sync(0xffffffffu, z.y, q),
                                        __shfl_sync(0xffffffffu, z.z, q), __shfl_sync(0xffffffffu, z.w, q));
              if (tc::elect()) {
#pragma unroll
                for (int pn = 0; pn < PN; ++pn) tc::load_rows(dst + pn * kPanel, &maps.q, pn * 64, y4, sh.q_full + buf);
              }
              __syncwarp();
            }
          } else if (tc::elect()) {
            const int boxes = (here + p.q_run - 1) / p.q_run;
            pipe::bar_expect_tx(sh.q_full + buf, (uint32_t)(boxes * p.q_run * 128 * PN));
#pragma unroll 1
            for (int q = 0; q < boxes; ++q, dst += p.q_run * 128) {
              const int x = xb + q * p.q_run, jt = (int)a.group_div.div((uint32_t)x);
#pragma unroll
              for (int pn = 0; pn < PN; ++pn)
                tc::load_box3(dst + pn * kPanel, &maps.q, pn * 64, head0 + x - jt * a.group, w.g.tok + jt, sh.q_full + buf);
            }
          }
          __syncwarp();
        }
        if (!ok) break;
        left -= units - y;
        at += units;
        y = 0;
        if (left > 0) w.next();
      }
      for (uint32_t q = n_q > 2 ? n_q - 2 : 0; q < n_q; ++q) (void)pipe::bar_wait(sh.q_full + (q & 1), (q >> 1) & 1);
    }
    }
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  // No product may be in flight when tensor memory is given back: the softmax
  // warps have waited for the last of them, unless a wait gave up.
  if (warp == 8) {
    if (*quit) {
      const uint64_t t0 = pipe::now_ns();
      while (pipe::now_ns() - t0 < 1000000ull) {
      }
      __syncwarp();
    }
    tc::dealloc(tmem, 512);
  }
  if (tid == 0 && (sh.quit[0] || sh.bad)) atomicOr(&g_attn_status, (sh.quit[0] ? 2u : 0u) | (sh.bad ? 1u : 0u));
}

// ------------------------------------------------------------ joining parts ---
// Row: o = sum w_k o_k / sum w_k, w_k = 2^(lse_k - max lse) over its parts.
struct Sum {
  float m = -INFINITY, l = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
  __device__ __forceinline__ void add(float4 v, float ls) {
    if (ls == -INFINITY) return;
    const float top = fmaxf(m, ls), f = m == -INFINITY ? 0.f : tc::ex2(m - top), g = tc::ex2(ls - top);
    l = (l == l ? l * f : l) + g;
    m = top;
    x[0] = x[0] * f + v.x * g;
    x[1] = x[1] * f + v.y * g;
    x[2] = x[2] * f + v.z * g;
    x[3] = x[3] * f + v.w * g;
  }
};

__device__ __forceinline__ float4 row4(const float* o, int dim, int lane) {
  return lane * 4 < dim ? load(reinterpret_cast<const float4*>(o) + lane) : make_float4(0.f, 0.f, 0.f, 0.f);
}

// Adds every step-th part of row `brow` of a segment cut over CTAs c0 .. c1.
__device__ __forceinline__ void add_cuts(Sum& sum, const TilePlan& p, int dim, int c0, int c1, int brow, int k0, int step,
                                         int lane) {
#pragma unroll 4
  for (int c = c0 + k0; c <= c1; c += step) {
    const int slot = 2 * c + (c == c0 ? 1 : 0);
    const int64_t row = (int64_t)slot * kBlock + brow;
    const int used = load(p.used + slot);  // a stretch so short that no tile begins in it leaves none
    const float4 v = row4(p.cut + row * dim, dim, lane);
    const float ls = load(p.cut_lse + row);
    if (used) sum.add(v, ls);
  }
}

// The block's eight warps' sums of one row, in warp 0.
__device__ __forceinline__ void sum_warps(Sum& s, int warp, int lane) {
  __shared__ float s_m[8], s_l[8], s_o[8][128];
  if (lane == 0) {
    s_m[warp] = s.m;
    s_l[warp] = s.l;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) s_o[warp][lane * 4 + e] = s.x[e];
  __syncthreads();
  if (warp != 0) return;
  float top = s.m;
#pragma unroll
  for (int k = 1; k < 8; ++k) top = fmaxf(top, s_m[k]);
  float l = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float f = s_m[k] == -INFINITY ? 0.f : tc::ex2(s_m[k] - top);
    l += s_l[k] == s_l[k] ? s_l[k] * f : s_l[k];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] += s_o[k][lane * 4 + e] * f;
  }
  s.m = top;
  s.l = l;
#pragma unroll
  for (int e = 0; e < 4; ++e) s.x[e] = x[e];
}

template <typename T>
__device__ __forceinline__ void write_row(const AttnArgs& a, int64_t grow, const Sum& s, int lane) {
  const float inv = s.l == 0.f ? 0.f : 1.f / s.l;
  if (lane * 4 < a.dim)
    *reinterpret_cast<uint2*>(a.out + (grow * a.dim + lane * 4) * 2) =
        make_uint2(Vec16<T>::pack2(s.x[0] * inv, s.x[1] * inv), Vec16<T>::pack2(s.x[2] * inv, s.x[3] * inv));
  if (lane == 0 && a.lse) a.lse[grow] = s.l == 0.f ? -INFINITY : (s.m + log2f(s.l)) * 0.6931471805599453f;
}

// Bound by latency: about 4 us behind the tiles, 12 to 17 us with thousands of cut
// rows and a cold cache.
//
// Rows with one segment each (prefix and own keys in one, or no prefix): only
// those of cut segments. Block (c, i) does the share i of the rows of the cut
// segment that ends in CTA c's stretch.
template <typename T>
__global__ void __launch_bounds__(256) attend_join_cuts_kernel(const AttnArgs a, const TilePlan p) {
  grid_dep_wait();
  grid_dep_launch();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = blockIdx.x;
  const CutEnd e = p.end[c];
  if (e.nrow == 0) return;
  // few rows, maybe with many parts: a block to a row, a warp to an eighth of the parts
  const bool split = e.nrow <= (int)gridDim.y;
  for (int brow = split ? blockIdx.y : blockIdx.y * 8 + warp; brow < e.nrow; brow += gridDim.y * 8) {
    const int x = e.x0 + brow, jt = (int)a.group_div.div((uint32_t)x);
    const int64_t grow = ((int64_t)e.tok + jt) * a.hq + e.kh * a.group + (x - jt * a.group);
    Sum s;
    add_cuts(s, p, a.dim, e.c0, c, brow, split ? warp : 0, split ? 8 : 1, lane);
    if (split) {
      sum_warps(s, warp, lane);
      if (warp != 0) return;
    }
    write_row<T>(a, grow, s, lane);
  }
}

// Rows with a part over the prefix and a part over their own keys. W warps share
// a row.
template <typename T, int W>
__global__ void __launch_bounds__(256) attend_join_kernel(const AttnArgs a, const TilePlan p) {
  grid_dep_wait();
  grid_dep_launch();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = warp % W;
  const int64_t grow = (int64_t)blockIdx.x * (8 / W) + warp / W, all = a.tokens * a.hq;
  const bool on = grow >= (int64_t)first_token(a) * a.hq && grow < (int64_t)live_tokens(a) * a.hq;
  Sum sum;
  if (on) {
    const int2 at[2] = {p.place[grow], p.place[all + grow]};
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      // the own keys' parts start with the last warp, the prefix's with the first
      const int k0 = u ? W - 1 - part : part;
      if (at[u].x < 0) {
        if (k0 == 0) sum.add(row4(p.whole + (u * all + grow) * a.dim, a.dim, lane), load(p.whole_lse + u * all + grow));
      } else {
        // (a token that offsets out of order leave out has no place: what is read stays inside the workspace)
        const int c0 = (at[u].x & 0xffff) < p.ctas ? at[u].x & 0xffff : 0, c1 = at[u].y < p.ctas ? at[u].y : 0;
        add_cuts(sum, p, a.dim, c0, c1, (at[u].x >> 16) & (kBlock - 1), k0, W, lane);
      }
    }
  }
  if (W > 1) {
    sum_warps(sum, warp, lane);
    if (warp != 0) return;
  }
  if (on) write_row<T>(a, grow, sum, lane);
}

// The tensor core takes 16-bit values, sixteen at a time; a head of more than
// 128 of them, of an odd half of sixteen, or of 32-bit values goes row by row.
// So does a scale next to nothing, under which a masked score would not vanish.
// (bf16, 32 heads on 8 KV heads of 128, in tiles and row by row: 16 decode requests behind
// 4096 keys 22 and 157 us, 128 ragged ones behind 2047 129 and 879, 16 extends of 8 tokens
// 36 and 958. Only a few short rows would be quicker row by row: three requests of up to
// 300 keys on one KV head 13.5 and 10.3, one of 1000 keys 13.7 and 24.6.)
bool takes_tiles(const AttnArgs& a, int dtype) {
  return dtype != GSEC_F32 && a.dim <= 128 && a.dim % 16 == 0 && !(fabsf(a.scale) < 1e-20f);
}

// Stacking the requests' rows over the prefix pays when they would not fill
// tiles by themselves; with about a tile of rows each (or one request) prefix and
// own keys are better taken in one go, which leaves little to join. (16 extends of 8,
// 16, 32 and 64 tokens, groups of 4, behind 4096 keys: stacked 36, 45, 71 and 198 us, in
// one go 58, 58, 57 and 89; a 2048-token chunk behind 30720 keys 1240 and 1030; 256 decode
// requests behind 24576 177 and 3290. The rule goes by the batch's mean, padding included:
// a chunk of 512 tokens among 15 decode requests behind 30720 keys, which it takes in one
// go, is 496 us, stacked 469.)
TilePlan tile_plan(const AttnArgs& a, int64_t* bytes) {
  TilePlan p{};
  p.ctas = sm_count();
  p.run = a.page & -a.page;  // boxes start at pages, tiles at multiples of 128 keys
  p.run = p.run < 8 ? 0 : (p.run > kKeys ? kKeys : p.run);
  while (p.run >> (p.run_log + 1)) ++p.run_log;
  p.slope = kBlock / (kKeys / kUnitTile) / a.group;
  p.slope = p.slope < 1 ? 1 : p.slope;
  p.joint = a.prefix_len == 0 || a.batch == 1 || a.tokens * a.group >= (int64_t)a.batch * kRows;
  char* at = a.workspace;
  const auto take = [&](int64_t n) {
    char* x = at;
    at += (n + 255) / 256 * 256;
    return x;
  };
  const int64_t rows = a.tokens * a.hq, parts = p.joint ? 0 : 2;
  p.used = reinterpret_cast<int32_t*>(take((int64_t)2 * p.ctas * 4));
  p.end = reinterpret_cast<CutEnd*>(take(p.ctas * (int64_t)sizeof(CutEnd)));
  p.place = reinterpret_cast<int2*>(take(parts * rows * 8));
  p.whole_lse = reinterpret_cast<float*>(take(parts * rows * 4));
  p.cut_lse = reinterpret_cast<float*>(take((int64_t)2 * p.ctas * kBlock * 4));
  p.whole = reinterpret_cast<float*>(take(parts * rows * a.dim * 4));
  p.cut = reinterpret_cast<float*>(take((int64_t)2 * p.ctas * kBlock * a.dim * 4));
  *bytes = at - a.workspace;
  return p;
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// The driver's encoder of tensor maps, or null.
EncodeTiled encode_tiled() {
  static const EncodeTiled fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult found = cudaDriverEntryPointSymbolNotFound;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found) !=
            cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<EncodeTiled>(f);
  }();
  return fn;
}

// Map of N dimensions of 16-bit values at `at`, 64 values wide in a box.
template <int N>
bool tile_map(CUtensorMap* m, bool bf16, const char* at, const cuuint64_t (&size)[N], const cuuint64_t (&stride)[N - 1],
              const cuuint32_t (&box)[N]) {
  cuuint32_t step[N];
  for (int i = 0; i < N; ++i) step[i] = 1;
  const EncodeTiled encode = encode_tiled();
  return encode != nullptr &&
         encode(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, N, const_cast<char*>(at),
                size, stride, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool query_map(CUtensorMap* m, bool bf16, const AttnArgs& a, const TilePlan& p) {
  using Z = cuuint64_t;
  if (p.q_ratio > 0)
    return tile_map<2>(m, bf16, a.q, {(Z)a.dim, (Z)((a.tokens - 1) * p.q_ratio + a.hq)}, {(Z)a.q_head}, {64, 1});
  const int heads = a.group < p.q_run ? a.group : p.q_run;
  return tile_map<3>(m, bf16, a.q, {(Z)a.dim, (Z)a.hq, (Z)a.tokens}, {(Z)a.q_head, (Z)a.q_pitch},
                     {64, (cuuint32_t)heads, (cuuint32_t)(p.q_run / heads)});
}

template <typename T, int DP>
int launch_tiles(const AttnArgs& a, cudaStream_t s) {
  int64_t bytes = 0;
  TilePlan p = tile_plan(a, &bytes);
  const int even = a.group & -a.group;  // heads of a box: a power of two
  p.q_run = even < kQueryBox && even < a.group ? even : kQueryBox;
  p.q_ratio = p.q_run < 4 && a.q_pitch % a.q_head == 0 && a.tokens * (a.q_pitch / a.q_head) < INT_MAX
                  ? (int)(a.q_pitch / a.q_head)
                  : 0;
  GSEC_REQUIRE(a.tokens * a.group < (1ll << 30), "prefix_attention: %lld tokens of %d heads on a KV head are too many",
               (long long)a.tokens, a.group);
  PoolMaps maps;
  bool ok = true;
  for (int kv = 0; kv < 2; ++kv) {
    const char* at = a.pool + (kv ? a.plane : 0);
    const cuuint64_t size[2] = {(cuuint64_t)a.hk * a.dim, (cuuint64_t)a.pool_rows}, pitch[1] = {(cuuint64_t)a.pitch};
    ok = ok && tile_map<2>(maps.box + kv, Vec16<T>::bf16, at, size, pitch, {64, (cuuint32_t)(p.run ? p.run : 1)}) &&
         tile_map<2>(maps.row + kv, Vec16<T>::bf16, at, size, pitch, {64, 1});
  }
  if (!ok || !query_map(&maps.q, Vec16<T>::bf16, a, p)) {
    set_error("prefix_attention: the tensor maps of pool and queries were refused");
    return GSEC_ECUDA;
  }
  constexpr int smem = TileShape<DP>::smem;
  const auto kernel = p.run ? attend_tile_kernel<T, DP, false> : attend_tile_kernel<T, DP, true>;
  if (launch_cache().blocks_per_sm(kernel, kTileThreads, smem) < 0)
    return check_launch("attend_tile launch shape");
  // a smaller launch would leave the softmax warpgroups waiting for registers that are not there
  static const bool regs_ok = [] {
    cudaFuncAttributes x{}, y{};
    return cudaFuncGetAttributes(&x, attend_tile_kernel<T, DP, false>) == cudaSuccess && x.numRegs == kLaunchRegs &&
           cudaFuncGetAttributes(&y, attend_tile_kernel<T, DP, true>) == cudaSuccess && y.numRegs == kLaunchRegs;
  }();
  GSEC_REQUIRE(regs_ok, "attend_tile: launch registers are not %d", kLaunchRegs);
  const int rc = launch_rc(
      launch_pdl(kernel, dim3((unsigned)p.ctas), dim3(kTileThreads), smem, s, a, p, maps),
      "prefix_attention");
  if (rc) return rc;
  // A warp to a row of a whole block, or a block to a row of a few. (8 blocks a segment and
  // 32: one request of 1000 keys 13.7 us and 17.2, 4 extends of 256 tokens 94 and 91.5.)
  if (p.joint) {
    const unsigned y = a.tokens * a.group < kBlock ? 8 : kBlock / 8;
    return launch_rc(launch_pdl(attend_join_cuts_kernel<T>, dim3((unsigned)p.ctas, y), dim3(256), 0, s, a, p),
                     "prefix_attention join");
  }
  const int64_t rows = a.tokens * a.hq;
  // few rows: eight warps to a row, since each may have a part from every CTA. (Eight warps and
  // one: 16 requests behind 32768 keys 42 us and 53, 256 behind 24576 198 and 177.)
  if (rows <= (int64_t)p.ctas * 16)
    return launch_rc(launch_pdl(attend_join_kernel<T, 8>, dim3((unsigned)rows), dim3(256), 0, s, a, p),
                     "prefix_attention join");
  return launch_rc(launch_pdl(attend_join_kernel<T, 1>, dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, s, a, p),
                   "prefix_attention join");
}

template <typename T>
int attend_tiles(const AttnArgs& a, cudaStream_t s) {
  return a.dim <= 64 ? launch_tiles<T, 64>(a, s) : launch_tiles<T, 128>(a, s);
}

}  // namespace

int64_t attention_workspace(const AttnArgs& a, int dtype) {
  if (!takes_tiles(a, dtype) || a.tokens == 0) return 0;
  int64_t bytes = 0;
  tile_plan(a, &bytes);
  return bytes;
}

int attention(const AttnArgs& a, int dtype, cudaStream_t s) {
  if (a.tokens == 0) return GSEC_OK;
  if (dtype == GSEC_F32) return attend_rows<float>(a, s);
  const bool tiles = takes_tiles(a, dtype);
  if (dtype == GSEC_BF16) return tiles ? attend_tiles<__nv_bfloat16>(a, s) : attend_rows<__nv_bfloat16>(a, s);
  return tiles ? attend_tiles<__half>(a, s) : attend_rows<__half>(a, s);
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
