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


// ---------------------------------------------------------- 128-row tiles -----
// Rows that read the same keys are stacked: `group` query heads of a KV head,
// for the shared prefix the tokens of all requests, for a request's own keys its
// new tokens. A block is up to 256 such rows of one KV head; a segment is a block
// with its keys, cut into tiles of 128. Scores S = Q K^T (128 x 128) and O += P V
// run on the tensor core with S, P and O in tensor memory; one thread holds one
// row, keeps its maximum m and sum l in registers, and replaces S by
// P = 2^(S c - m c) in place. O is scaled by 2^(m_old - m) only when the maximum
// has grown by more than 8 binary places since P was last taken relative to it;
// until then P exceeds 1 by at most 2^8, which fp32 sums and 16-bit P hold as
// well as they hold 1.
//
// Two warpgroups take turns, so that one's exponentials run under the other's
// products: with more than 128 rows in the block each has its own 128 rows and
// both see every tile; otherwise they take the even and the odd tiles of the
// same rows and add up their halves at the end.
//
// Work is dealt out evenly whatever the lengths: all tiles of all segments form
// one line, and each of the resident CTAs takes an equal stretch of it. A segment
// cut by a stretch's end, and the two halves (prefix, own keys) of a row, are
// joined by attend_join_kernel from fp32 partial results and their log sums.
constexpr int kTileThreads = 384;   // 2 softmax warpgroups; 1 issuing warp, 3 loading warps
constexpr int kRows = 128, kKeys = 128, kBlock = 256;
// Registers: a softmax thread holds a row of 128 scores. The launch has 168 per
// thread; the third warpgroup hands over what it does not need.
constexpr int kLaunchRegs = 168, kSoftmaxRegs = 216, kOtherRegs = 72;
static_assert(2 * kSoftmaxRegs + kOtherRegs <= 3 * kLaunchRegs, "register shares");

struct TilePlan {
  int run;               // rows of a box: the largest power of two dividing the page, at most a tile; 0: rows one by one
  int joint;             // prefix and own keys of a request are one segment (no stacking over requests)
  int ctas;
  int64_t* start;        // [batch + 1] first tile of request i on the line
  float* whole;          // [2][tokens * hq][dim] rows of uncut segments (prefix, own) that have another part
  float* whole_lse;      // [2][tokens * hq]
  float* cut;            // [2 * ctas][kBlock][dim] rows of cut segments: CTA's first and last stretch
  float* cut_lse;        // [2 * ctas][kBlock]
};

// Tensor maps of the pool's K and V rows ([pool_rows, hk * dim], 128-byte
// swizzle): boxes of 64 values x `run` rows, and single rows.
struct PoolMaps {
  CUtensorMap box[2], row[2];
};

// One segment: nrow rows from row `row0` of the row space that starts at token
// `tok`; row x is token tok + x / group, head kh * group + x % group.
struct Segment {
  int req;               // request, -1: prefix of all
  int tok, ntok, kh, blk, nblk, own;
  int64_t len;
  int tiles;
};

__device__ __forceinline__ int tile_count(int64_t keys) { return (int)((keys + kKeys - 1) / kKeys); }

// The line of tiles as one thread walks it.
struct Walk {
  const AttnArgs& a;
  const TilePlan& p;
  int live;              // query tokens of the batch
  Segment g;
  __device__ __forceinline__ Walk(const AttnArgs& a_, const TilePlan& p_, int live_) : a(a_), p(p_), live(live_) {}

  __device__ __forceinline__ int prefix_keys() const { return p.joint ? 0 : a.prefix_len; }
  // Query tokens [tok, tok + ntok) and own keys of request r, cut to what exists.
  __device__ __forceinline__ void request(int r) {
    const int c0 = __ldg(a.cu + r), c1 = __ldg(a.cu + r + 1);
    const int lo = c0 < 0 ? 0 : (c0 > live ? live : c0), hi = c1 < lo ? lo : (c1 > live ? live : c1);
    const int64_t room = (int64_t)a.width * a.page, n = __ldg(a.lens + r);
    g.req = r;
    g.tok = lo;
    g.ntok = hi - lo;
    g.len = n < 0 ? 0 : (n > room ? room : n);
    g.nblk = (int)(((int64_t)g.ntok * a.group + kBlock - 1) / kBlock);
  }
  // Own keys that token j of the request sees.
  __device__ __forceinline__ int64_t own_seen(int j) const {
    const int64_t x = g.len - g.ntok + j + 1;
    return x < 0 ? 0 : (x > g.len ? g.len : x);
  }
  // Own keys that row x of the segment sees.
  __device__ __forceinline__ int64_t row_seen(int x) const {
    return g.req < 0 ? 0 : own_seen((int)a.group_div.div((uint32_t)x));
  }
  __device__ __forceinline__ int rows() const {
    const int64_t r = (int64_t)g.ntok * a.group - (int64_t)g.blk * kBlock;
    return r < kBlock ? (int)r : kBlock;
  }
  // Own keys of the block: what its last row sees.
  __device__ __forceinline__ int64_t own_keys() const { return row_seen(g.blk * kBlock + rows() - 1); }
  // Prefix tiles of the segment come first; no tile holds both kinds of keys. A
  // block without keys still has a tile, which writes its empty rows.
  __device__ __forceinline__ int prefix_part() const { return g.req < 0 || p.joint ? tile_count(a.prefix_len) : 0; }
  __device__ __forceinline__ int block_tiles() const {
    const int n = prefix_part() + tile_count(own_keys());
    return n < 1 ? 1 : n;
  }
  __device__ __forceinline__ void size() { g.tiles = block_tiles(); }
  // Tiles of one head of the request.
  __device__ __forceinline__ int64_t head_tiles() {
    int64_t n = 0;
    for (g.blk = 0; g.blk < g.nblk; ++g.blk) n += block_tiles();
    return n;
  }
  __device__ __forceinline__ void prefix_space() {
    g.req = -1;
    g.tok = 0;
    g.ntok = live;
    g.len = 0;
    g.nblk = (int)(((int64_t)live * a.group + kBlock - 1) / kBlock);
  }
  // The next segment of the line.
  __device__ __forceinline__ void next() {
    if (++g.blk == g.nblk) {
      g.blk = 0;
      if (++g.kh == a.hk) {
        g.kh = 0;
        int r = g.req;
        do {
          if (++r >= a.batch) {  // past the last tile: not walked
            g.nblk = 0;
            return;
          }
          request(r);
        } while (g.nblk == 0);
      }
    }
    size();
  }
};

// What the line holds before request r, prefix first.
__device__ __forceinline__ int64_t prefix_tiles(const AttnArgs& a, const TilePlan& p, int live) {
  if (p.joint || a.prefix_len == 0) return 0;
  return (int64_t)a.hk * (((int64_t)live * a.group + kBlock - 1) / kBlock) * tile_count(a.prefix_len);
}

__device__ __forceinline__ int live_tokens(const AttnArgs& a) {
  const int n = __ldg(a.cu + a.batch);
  return n < 0 ? 0 : (n > a.tokens ? (int)a.tokens : n);
}

// Tiles per CTA.
__device__ __forceinline__ int64_t share(int64_t total, int ctas) { return (total + ctas - 1) / ctas; }

// A wait that gives up raises `quit`, which ends every other wait of the CTA.
__device__ __forceinline__ bool wait_or_quit(uint64_t* bar, uint32_t parity, volatile int* quit) {
  if (pipe::bar_try(bar, parity)) return true;
  const uint64_t t0 = pipe::now_ns();
  while (!pipe::bar_try(bar, parity)) {
    if (*quit) return false;
    if (pipe::now_ns() - t0 > pipe::kWaitNs) {
      *quit = 1;
      atomicOr(&g_attn_status, 2u);
      return false;
    }
  }
  return true;
}

// The same for a whole warp: every lane gets the same answer.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* quit) {
  return __all_sync(0xffffffffu, wait_or_quit(bar, parity, quit)) != 0;
}

template <int DP>
struct TileShape {
  static constexpr int tile = kRows * DP * 2;                     // bytes of a Q, K or V tile
  static constexpr int stages = DP == 128 ? 5 : 12;               // K and V tiles in flight
  static constexpr int data = (2 + stages) * tile;
  static constexpr int smem = data + 3072;
};

// Shared memory behind the tiles.
struct TileShared {
  float m[2][kRows], l[2][kRows];   // the two warpgroups' halves of the same rows
  uint64_t full[12], empty[12], q_full[2], q_empty[2], s_full[2], p_full[2], o_full[2], o_empty, halves, halves_read;
  alignas(16) int32_t rows[kKeys];  // pool rows of the tile being loaded
  Segment first;                    // where this CTA's stretch starts
  int64_t first_off, total;
  uint32_t tmem;
  int quit;
};
static_assert(sizeof(TileShared) <= 3072, "shared memory behind the tiles");

// Positions in the ring are counted in 32 bits and taken back by a multiple of
// two turns (which keeps stage and parity) long before they overflow.
template <int ST>
constexpr uint32_t kTurn = (1u << 30) / (2 * ST) * (2 * ST);
template <int ST>
__device__ __forceinline__ uint32_t next_pos(uint32_t pos, int tiles) {
  pos += 2 * (uint32_t)tiles;
  return pos >= kTurn<ST> ? pos - kTurn<ST> : pos;
}

// One row's share of a tile: the scores at tensor memory `ts` (128 columns) become
// 16-bit P there; (m, l) follow, and O at `to` (when it holds something) is
// brought to the new reference. CUT: only the first `cols` keys are seen.
template <typename T, int DP, bool CUT>
__device__ __forceinline__ void softmax_tile(uint32_t ts, uint32_t to, float c, int cols, bool has_o, float& m,
                                             float& l) {
  uint32_t s[128];
#pragma unroll
  for (int k = 0; k < 4; ++k) tc::ld32(ts + k * 32, s + k * 32);
  tc::wait_ld();
  float t4[4] = {m, m, m, m};
#pragma unroll
  for (int k = 0; k < 128; ++k)
    if (!CUT || k < cols) t4[k & 3] = fmaxf(t4[k & 3], __uint_as_float(s[k]));
  const float top = fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3]));
  // move the reference when it is too far behind (or there is none yet)
  const bool move = (top - m) * c > 8.f || (m == -INFINITY && top > -INFINITY);
  if (__any_sync(0xffffffffu, move)) {
    const float f = !move ? 1.f : (m == -INFINITY ? 0.f : tc::ex2((m - top) * c));
    if (move) m = top;
    l *= f;
    if (has_o) {
      uint32_t o[32];
#pragma unroll 1
      for (int k = 0; k < DP; k += 32) {
        tc::ld32(to + k, o);
        tc::wait_ld();
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
        tc::st32(to + k, o);
      }
    }
  }
  const float mc = m == -INFINITY ? 0.f : m * c;
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int k = h * 64; k < h * 64 + 64; k += 2) {
      float p0 = tc::ex2(fmaf(__uint_as_float(s[k]), c, -mc));
      float p1 = tc::ex2(fmaf(__uint_as_float(s[k + 1]), c, -mc));
      if (CUT) {
        p0 = k < cols ? p0 : 0.f;
        p1 = k + 1 < cols ? p1 : 0.f;
      }
      sum[(k >> 1) & 3] += p0 + p1;
      s[k >> 1] = Vec16<T>::pack2(p0, p1);
    }
    tc::st32(ts + h * 32, s + h * 32);
  }
  l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

template <typename T, int DP>
__global__ void __launch_bounds__(kTileThreads, 1) attend_tile_kernel(const AttnArgs a, const TilePlan p,
                                                                     const __grid_constant__ PoolMaps maps) {
  using Shape = TileShape<DP>;
  constexpr int ST = Shape::stages;
  constexpr bool kBf16 = Vec16<T>::bf16;
  extern __shared__ __align__(1024) unsigned char smem[];
  TileShared& sh = *reinterpret_cast<TileShared*>(smem + Shape::data);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < ST; ++i) {
      pipe::bar_init(sh.full + i, 1);
      pipe::bar_init(sh.empty + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      pipe::bar_init(sh.q_full + i, 2);
      pipe::bar_init(sh.q_empty + i, 1);
      pipe::bar_init(sh.s_full + i, 1);
      pipe::bar_init(sh.p_full + i, 4);
      pipe::bar_init(sh.o_full + i, 1);
    }
    pipe::bar_init(&sh.o_empty, 8);
    pipe::bar_init(&sh.halves, 8);
    pipe::bar_init(&sh.halves_read, 8);
    pipe::bar_init_fence();
    sh.quit = (tc::smem_addr(smem) & 1023u) != 0;  // the swizzle counts from 1024-byte patterns
    if (sh.quit) atomicOr(&g_attn_status, 2u);
  }
  if (warp == 8) {
    tc::alloc(&sh.tmem, 512);
    tc::relinquish();
  }
  grid_dep_wait();
  grid_dep_launch();

  // The line: tiles of every request (a run of requests per thread), their sum,
  // and the place where this CTA's stretch starts.
  const int live = live_tokens(a);
  {
    Walk w(a, p, live);
    int64_t* wsum = reinterpret_cast<int64_t*>(smem);  // the tiles' memory is not in use yet
    const int per = (a.batch + kTileThreads - 1) / kTileThreads;
    const int r0 = tid * per < a.batch ? tid * per : a.batch, r1 = r0 + per < a.batch ? r0 + per : a.batch;
    int64_t mine = 0, last = 0;  // tiles of the run, of one head of its last request
    for (int r = r0; r < r1; ++r) {
      w.request(r);
      last = w.head_tiles();
      mine += last * a.hk;
      if (blockIdx.x == 0 && (__ldg(a.lens + r) > (int64_t)a.width * a.page || __ldg(a.lens + r) < 0 ||
                              __ldg(a.cu + r) < 0 || __ldg(a.cu + r + 1) > a.tokens ||
                              __ldg(a.cu + r + 1) < __ldg(a.cu + r)))
        atomicOr(&g_attn_status, 1u);
    }
    int64_t x = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, x, d);
      if (lane >= d) x += y;
    }
    if (lane == 31) wsum[warp] = x;
    __syncthreads();
    const int64_t pre = prefix_tiles(a, p, live);
    int64_t at = pre + x - mine, total = pre;
    for (int i = 0; i < kTileThreads / 32; ++i) {
      if (i < warp) at += wsum[i];
      total += wsum[i];
    }
    const int64_t x0 = (int64_t)blockIdx.x * share(total, p.ctas);
    if (tid == 0) {
      sh.total = total;
      if (x0 < pre) {
        w.prefix_space();
        const int tp = tile_count(a.prefix_len);
        const int64_t si = x0 / tp;
        w.g.kh = (int)(si / w.g.nblk);
        w.g.blk = (int)(si - (int64_t)w.g.kh * w.g.nblk);
        w.g.tiles = tp;
        sh.first = w.g;
        sh.first_off = x0 - si * tp;
      }
    }
    for (int r = r0; r < r1; ++r) {
      if (per > 1) {
        w.request(r);
        last = w.head_tiles();
      }
      const int64_t one = last;
      if (blockIdx.x == 0) p.start[r] = at;
      if (x0 >= at && x0 < at + one * a.hk) {
        int64_t y = x0 - at;
        w.g.kh = (int)(y / one);
        y -= w.g.kh * one;
        for (w.g.blk = 0;; ++w.g.blk) {
          w.size();
          if (y < w.g.tiles) break;
          y -= w.g.tiles;
        }
        sh.first = w.g;
        sh.first_off = y;
      }
      at += one * a.hk;
    }
    if (blockIdx.x == 0 && tid == 0) p.start[a.batch] = total;
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
  }
  const uint32_t tmem = sh.tmem;
  const int64_t unit = share(sh.total, p.ctas);
  const int64_t x0 = (int64_t)blockIdx.x * unit, x1 = x0 + unit < sh.total ? x0 + unit : sh.total;
  volatile int* quit = &sh.quit;
  const float c = fabsf(a.scale) * 1.4426950408889634f;

  if (x0 < x1 && !*quit) {
    Walk w(a, p, live);
    w.g = sh.first;
    int64_t left = x1 - x0;
    int off = (int)sh.first_off;
    if (warp < 8) {
      // ------------------------------------------------ softmax warpgroups ----
      tc::regs_up<kSoftmaxRegs>();
      const int t = warp >> 2, r = tid & (kRows - 1);
      const uint32_t row = (uint32_t)((warp & 3) * 32) << 16;
      const uint32_t ts = tmem + row + t * 128, to = tmem + row + 256 + t * 128;
      uint32_t n_s = 0, n_piece = 0, n_halves = 0, n_o[2] = {0, 0};
      while (true) {
        const int rows = w.rows(), n = (int)(w.g.tiles - off < left ? w.g.tiles - off : left);
        const bool pair = rows > kRows;
        const int mine = pair ? t * kRows + r : r;             // this thread's row of the block
        const int np = w.prefix_part();
        const int64_t see = mine < rows ? w.row_seen(w.g.blk * kBlock + mine) : 0;
        const bool warp_on = __any_sync(0xffffffffu, mine < rows);
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        for (int i = pair ? 0 : t; i < n; i += pair ? 1 : 2) {
          ok = warp_wait(sh.s_full + t, n_s & 1, quit);
          if (!ok) break;
          ++n_s;
          tc::fence_after();
          if (warp_on) {
            const int ti = off + i;
            const int64_t rest = ti >= np ? see - (int64_t)(ti - np) * kKeys
                                          : (mine < rows ? a.prefix_len - ti * kKeys : 0);
            const int cols = rest < 0 ? 0 : (rest < kKeys ? (int)rest : kKeys);
            const bool has_o = pair ? i > 0 : i >= 2;
            if (__any_sync(0xffffffffu, cols < kKeys))
              softmax_tile<T, DP, true>(ts, to, c, cols, has_o, m, l);
            else
              softmax_tile<T, DP, false>(ts, to, c, cols, has_o, m, l);
            tc::wait_st();
          }
          tc::fence_before();
          __syncwarp();
          if (lane == 0) pipe::bar_arrive(sh.p_full + t);
        }
        if (!ok) break;
        // -------------------------------------------------------- results ----
        // the product of the last tile; in single blocks both halves' products
        const bool has[2] = {true, pair || n > 1};
        for (int u = 0; u < 2; ++u) {
          if (has[u] && (!pair || u == t)) ok = ok && warp_wait(sh.o_full + u, n_o[u] & 1, quit);
          n_o[u] += has[u];
        }
        if (!ok) break;
        tc::fence_after();
        float w0 = 1.f, w1 = 0.f;
        if (!pair && n > 1) {
          if (n_halves > 0 && !(ok = warp_wait(&sh.halves_read, (n_halves - 1) & 1, quit))) break;
          sh.m[t][r] = m;
          sh.l[t][r] = l;
          __syncwarp();
          if (lane == 0) pipe::bar_arrive(&sh.halves);
          if (!(ok = warp_wait(&sh.halves, n_halves & 1, quit))) break;
          const float ma = sh.m[0][r], mb = sh.m[1][r], la = sh.l[0][r], lb = sh.l[1][r];
          __syncwarp();
          if (lane == 0) pipe::bar_arrive(&sh.halves_read);
          ++n_halves;
          m = fmaxf(ma, mb);
          w0 = ma == -INFINITY ? 0.f : tc::ex2((ma - m) * c);
          w1 = mb == -INFINITY ? 0.f : tc::ex2((mb - m) * c);
          // a sum that is not a number stays so, whatever its maximum
          l = (la == la ? w0 * la : la) + (lb == lb ? w1 * lb : lb);
        }
        const bool whole = off == 0 && n == w.g.tiles;
        const bool direct = whole && (p.joint || a.prefix_len == 0);
        const bool split_cols = !pair && n > 1;                 // both warpgroups write half the columns
        const bool writes = mine < rows && (pair || n > 1 || t == 0);
        const int x = w.g.blk * kBlock + mine;
        const int jt = (int)a.group_div.div((uint32_t)x);
        const int64_t grow = ((int64_t)w.g.tok + jt) * a.hq + w.g.kh * a.group + (x - jt * a.group);
        const int64_t crow = ((int64_t)2 * blockIdx.x + (off == 0 ? 1 : 0)) * kBlock + mine;
        const int64_t wrow = (w.g.req < 0 ? 0 : (int64_t)a.tokens * a.hq) + grow;
        float* dst = whole ? p.whole + wrow * a.dim : p.cut + crow * a.dim;
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const float ls = l == 0.f ? -INFINITY : m * c + log2f(l);
        if (writes && (t == 0 || pair)) {
          if (direct) {
            if (a.lse) a.lse[grow] = ls * 0.6931471805599453f;
          } else {
            (whole ? p.whole_lse[wrow] : p.cut_lse[crow]) = ls;
          }
        }
        if (warp_on && (pair || n > 1 || t == 0)) {
          const int k0 = split_cols ? t * (DP / 2) : 0, k1 = split_cols ? k0 + DP / 2 : DP;
          const uint32_t oa = pair ? to : tmem + row + 256, ob = tmem + row + 384;
#pragma unroll 1
          for (int k = k0; k < k1; k += 32) {
            if (k >= a.dim) break;
            uint32_t o[32], o2[32];
            tc::ld32(oa + k, o);
            if (split_cols) tc::ld32(ob + k, o2);
            tc::wait_ld();
            float f[32];
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              f[e] = __uint_as_float(o[e]);
              if (split_cols) f[e] = f[e] * w0 + __uint_as_float(o2[e]) * w1;
              f[e] = l == 0.f ? 0.f : f[e] * inv;
            }
            if (writes) {
              if (direct) {
                char* to_row = a.out + (grow * a.dim + k) * 2;
#pragma unroll
                for (int e = 0; e < 32; e += 8)
                  if (k + e < a.dim) *reinterpret_cast<uint4*>(to_row + e * 2) = Vec16<T>::pack(f + e);
              } else {
#pragma unroll
                for (int e = 0; e < 32; e += 4)
                  if (k + e < a.dim)
                    *reinterpret_cast<float4*>(dst + k + e) = make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]);
              }
            }
          }
        }
        tc::fence_before();
        __syncwarp();
        if (lane == 0) pipe::bar_arrive(&sh.o_empty);
        ++n_piece;
        left -= n;
        if (left <= 0) break;
        off = 0;
        w.next();
      }
    } else {
    tc::regs_down<kOtherRegs>();
    if (warp == 8) {
      // -------------------------------------------------------- products ----
      // The whole warp walks along; one lane issues.
      const uint32_t id_s = tc::idesc(kBf16, kRows, kKeys, false, a.scale < 0.f);
      const uint32_t id_o = tc::idesc(kBf16, kRows, a.dim, true);
      const int ks = a.dim / 16;
      const uint32_t base = tc::smem_addr(smem), ring = base + 2 * Shape::tile;
      uint32_t n_p[2] = {0, 0}, n_piece = 0, n_q = 0;
      uint32_t pos = 0;  // counts K and V tiles, modulo 2^32 in whole turns of the ring
      bool ok = true;
      while (ok) {
        const int rows = w.rows(), n = (int)(w.g.tiles - off < left ? w.g.tiles - off : left);
        const bool pair = rows > kRows;
        const int nq = pair ? 2 : 1;
        for (int b = 0; b < nq && ok; ++b)
          ok = warp_wait(sh.q_full + ((n_q + b) & 1), ((n_q + b) >> 1) & 1, quit);
        if (!ok) break;
        const uint32_t q0 = base + (n_q & 1) * Shape::tile, q1 = pair ? base + ((n_q + 1) & 1) * Shape::tile : q0;
        const auto tile_of = [&](int k, int t) { return pair ? k : 2 * k + t; };
        const auto scores = [&](int k, int t) {
          const int i = tile_of(k, t);
          if (i >= n) return true;
          const uint32_t at = pos + 2 * (uint32_t)i, st = at % ST;
          if (!warp_wait(sh.full + st, (at / ST) & 1, quit)) return false;
          tc::fence_after();
          const uint64_t qd = tc::desc(t ? q1 : q0, 16, 1024), kd = tc::desc(ring + st * Shape::tile, 16, 1024);
          if (tc::elect()) {
#pragma unroll
            for (int j = 0; j < DP / 16; ++j) {
              const uint32_t o = ((j >> 2) * (kRows * 128) + (j & 3) * 32) >> 4;
              if (j < ks) tc::mma_ss(tmem + t * 128, qd + o, kd + o, id_s, j > 0);
            }
            tc::commit(sh.s_full + t);
            if (!pair || t == 1) tc::commit(sh.empty + st);
          }
          __syncwarp();
          return true;
        };
        ok = scores(0, 0) && scores(0, 1);
        for (int k = 0; ok && tile_of(k, 0) < n; ++k) {
          for (int t = 0; ok && t < 2; ++t) {
            const int i = tile_of(k, t);
            if (i >= n) break;
            const uint32_t at = pos + 2 * (uint32_t)i + 1, st = at % ST;
            ok = warp_wait(sh.full + st, (at / ST) & 1, quit) && warp_wait(sh.p_full + t, n_p[t] & 1, quit);
            if (!ok) break;
            ++n_p[t];
            if (k == 0 && t == 0 && n_piece > 0 && !(ok = warp_wait(&sh.o_empty, (n_piece - 1) & 1, quit))) break;
            tc::fence_after();
            const uint64_t vd = tc::desc(ring + st * Shape::tile, kKeys * 128, 1024);
            if (tc::elect()) {
#pragma unroll
              for (int j = 0; j < kKeys / 16; ++j)
                tc::mma_ts(tmem + 256 + t * 128, tmem + t * 128 + j * 8, vd + ((j * 2048) >> 4), id_o, k > 0 || j > 0);
              if (!pair || t == 1) tc::commit(sh.empty + st);
              if (tile_of(k + 1, t) >= n) tc::commit(sh.o_full + t);
            }
            __syncwarp();
            ok = scores(k + 1, t);
          }
        }
        if (!ok) break;
        if (tc::elect())
          for (int b = 0; b < nq; ++b) tc::commit(sh.q_empty + ((n_q + b) & 1));
        __syncwarp();
        n_q += nq;
        pos = next_pos<ST>(pos, n);
        ++n_piece;
        left -= n;
        if (left <= 0) break;
        off = 0;
        w.next();
      }
    } else {
      // ----------------------------------------------------------- loads ----
      constexpr int CH = DP / 8, PN = DP / 64;                  // 16-byte chunks and 64-value panels of a row
      constexpr uint32_t kPanel = kRows * 128;
      const uint32_t base = tc::smem_addr(smem), ring = base + 2 * Shape::tile;
      if (warp == 9) {
        // keys and values: whole pages as boxes; a tile with a page that is cut
        // short, or outside the pool, row by row, four rows at a time, with zeros
        // for what is not there (a slot behind the end may hold anything)
        if (lane < 2) {
          tc::prefetch_map(maps.box + lane);
          tc::prefetch_map(maps.row + lane);
        }
        const int none = (int)a.pool_rows;                      // a row outside the map
        uint32_t pos = 0;
        bool ok = true;
        while (ok) {
          const int n = (int)(w.g.tiles - off < left ? w.g.tiles - off : left);
          const int np = w.prefix_part();
          const int64_t own = w.own_keys();
          for (int i = 0; i < n && ok; ++i) {
            const int ti = off + i;
            const bool pre = ti < np;
            const int64_t key0 = (int64_t)(pre ? ti : ti - np) * kKeys;
            const int64_t rest = (pre ? a.prefix_len : own) - key0;
            const int valid = rest < 0 ? 0 : (rest < kKeys ? (int)rest : kKeys);
            const int shift = pre ? 0 : a.prefix_len;           // own keys follow the prefix
            bool boxes = p.run > 0 && valid == kKeys;
            if (boxes) {
              int32_t y = 0;
              if (lane * p.run < kKeys) {
                const int64_t sl = key_slot(a, w.g.req, (int32_t)key0 + lane * p.run + shift);
                y = sl < 0 || sl + p.run > a.pool_rows ? -1 : (int32_t)sl;
                sh.rows[lane] = y;
              }
              boxes = !__any_sync(0xffffffffu, y < 0);
            }
            if (!boxes) {
              int4 y = make_int4(none, none, none, none);
              int32_t* e = &y.x;
#pragma unroll
              for (int j = 0; j < 4; ++j)
                if (lane * 4 + j < valid) {
                  const int64_t sl = key_slot(a, w.g.req, (int32_t)key0 + lane * 4 + j + shift);
                  if (sl >= 0) e[j] = (int32_t)sl;
                }
              *reinterpret_cast<int4*>(sh.rows + lane * 4) = y;
            }
            __syncwarp();
            for (int kv = 0; kv < 2; ++kv, ++pos) {
              const uint32_t st = pos % ST;
              if (pos >= ST && !(ok = warp_wait(sh.empty + st, (pos / ST - 1) & 1, quit))) break;
              if (tc::elect()) {
                pipe::bar_expect_tx(sh.full + st, Shape::tile);
                const uint32_t dst = ring + st * Shape::tile;
                const int x = w.g.kh * a.dim;
                if (boxes) {
                  const int nb = kKeys / p.run;
#pragma unroll 2
                  for (int b = 0; b < nb; ++b) {
                    const int y = sh.rows[b];
#pragma unroll
                    for (int pn = 0; pn < PN; ++pn)
                      tc::load_box(dst + pn * kPanel + b * p.run * 128, maps.box + kv, x + pn * 64, y, sh.full + st);
                  }
                } else {
#pragma unroll 2
                  for (int b = 0; b < kKeys / 4; ++b) {
                    const int4 y = *reinterpret_cast<const int4*>(sh.rows + b * 4);
#pragma unroll
                    for (int pn = 0; pn < PN; ++pn)
                      tc::load_rows(dst + pn * kPanel + b * 512, maps.row + kv, x + pn * 64, y, sh.full + st);
                  }
                }
              }
              __syncwarp();
            }
            if (pos >= kTurn<ST>) pos -= kTurn<ST> - ST * 2;  // keeps stage and parity, and counts as a full ring
          }
          left -= n;
          if (left <= 0) break;
          off = 0;
          w.next();
        }
        // copies must not outlive the CTA: all are waited for by the products, unless a wait gave up
        if (*quit)
          for (uint32_t q = pos > ST ? pos - ST : 0; q < pos; ++q) (void)pipe::bar_wait(sh.full + q % ST, (q / ST) & 1);
      } else {
        // queries: only the rows that exist (a product's rows do not mix)
        constexpr int RI = 32 / CH;                             // rows per instruction
        const int lw = warp - 10, ch = lane % CH, sub = lane / CH;
        const bool in_dim = ch * 8 < a.dim;
        const uint32_t panel = (uint32_t)(ch >> 3) * kPanel;
        uint32_t n_q = 0;
        bool ok = true;
        while (ok) {
          const int rows = w.rows(), n = (int)(w.g.tiles - off < left ? w.g.tiles - off : left);
          const int nq = rows > kRows ? 2 : 1;
          for (int b = 0; b < nq; ++b, ++n_q) {
            const int buf = n_q & 1;
            if (n_q >= 2 && !(ok = warp_wait(sh.q_empty + buf, ((n_q >> 1) - 1) & 1, quit))) break;
            const uint32_t dst = base + buf * Shape::tile;
            const int here = rows - b * kRows < kRows ? rows - b * kRows : kRows;
#pragma unroll 4
            for (int rr = lw * RI + sub; rr < here; rr += 2 * RI) {
              const int x = w.g.blk * kBlock + b * kRows + rr;
              const int jt = (int)a.group_div.div((uint32_t)x);
              const char* src = a.q + ((int64_t)w.g.tok + jt) * a.q_pitch +
                                (int64_t)(w.g.kh * a.group + x - jt * a.group) * a.q_head + ch * 16;
              if (in_dim) tc::copy16(dst + panel + rr * 128 + (((ch & 7) ^ (rr & 7)) << 4), src, true);
            }
            tc::copy_commit();
            tc::copy_wait<0>();
            tc::fence_async();
            __syncwarp();
            if (lane == 0) pipe::bar_arrive(sh.q_full + buf);
          }
          left -= n;
          if (left <= 0) break;
          off = 0;
          w.next();
        }
      }
    }
    }
  }
  // No product may be in flight when tensor memory is given back: the softmax
  // warps have waited for the last of them, unless a wait gave up.
  if (warp == 8 && *quit && !(tc::smem_addr(smem) & 1023u)) {
    if (lane == 0) {
      tc::commit(&sh.halves_read);  // its count is 8: the wait below only bounds the time the products get
      const uint64_t t0 = pipe::now_ns();
      while (pipe::now_ns() - t0 < 1000000ull) {
      }
    }
    __syncwarp();
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  if (warp == 8) tc::dealloc(tmem, 512);
}

// ------------------------------------------------------------ joining parts ---
// Row (token, head): o = sum w_k o_k / sum w_k, w_k = 2^(lse_k - max lse), over
// the parts of its prefix segment and of its own segment. Rows of uncut segments
// without a second part have been written already. W warps share a row: a cut
// segment can have as many parts as there are CTAs.
template <typename T, int W>
__global__ void __launch_bounds__(256) attend_join_kernel(const AttnArgs a, const TilePlan p) {
  grid_dep_wait();
  grid_dep_launch();
  __shared__ float s_m[8], s_l[8], s_o[8][128];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t grow = (int64_t)blockIdx.x * (8 / W) + warp / W;
  const int live = live_tokens(a), part = warp % W;
  const int64_t rows = (int64_t)live * a.hq;
  int n0 = 0, n1 = 0;          // parts of the prefix segment, of the own segment
  int64_t c0[2] = {0, 0};      // their first CTA
  int brow[2] = {0, 0};        // row in the block
  bool cut0 = false, cut1 = false;
  if (grow < rows) {
    const int t = (int)(grow / a.hq), h = (int)(grow - (int64_t)t * a.hq);
    const int kh = (int)a.group_div.div((uint32_t)h), gi = h - kh * a.group;
    const int64_t total = __ldg(p.start + a.batch), unit = share(total, p.ctas);
    Walk w(a, p, live);
    const int pk = w.prefix_keys();
    if (pk > 0) {
      w.prefix_space();
      const int64_t x = (int64_t)t * a.group + gi;
      const int tp = tile_count(a.prefix_len), blk = (int)(x / kBlock);
      const int64_t s = ((int64_t)kh * w.g.nblk + blk) * tp, e = s + tp - 1;
      c0[0] = s / unit;
      n0 = (int)(e / unit - c0[0]) + 1;
      cut0 = n0 > 1;
      brow[0] = (int)(x - (int64_t)blk * kBlock);
    }
    int r = 0, hi = a.batch;   // the last r with cu[r] <= t
    while (hi - r > 1) {
      const int mid = (r + hi) >> 1;
      if (__ldg(a.cu + mid) <= t)
        r = mid;
      else
        hi = mid;
    }
    w.request(r);
    if (t >= w.g.tok && t < w.g.tok + w.g.ntok) {
      const int64_t x = (int64_t)(t - w.g.tok) * a.group + gi;
      const int blk = (int)(x / kBlock);
      int64_t before = 0, one = 0, here = 0;  // tiles of the blocks before this one, of all, of this one
      for (int b = lane; b < w.g.nblk; b += 32) {
        w.g.blk = b;
        const int n = w.block_tiles();
        one += n;
        if (b < blk) before += n;
        if (b == blk) here = n;
      }
#pragma unroll
      for (int d = 16; d; d >>= 1) {
        one += __shfl_xor_sync(0xffffffffu, one, d);
        before += __shfl_xor_sync(0xffffffffu, before, d);
        here += __shfl_xor_sync(0xffffffffu, here, d);
      }
      const int64_t s = __ldg(p.start + r) + kh * one + before, e = s + here - 1;
      c0[1] = s / unit;
      n1 = (int)(e / unit - c0[1]) + 1;
      cut1 = n1 > 1;
      brow[1] = (int)(x - (int64_t)blk * kBlock);
    }
  }
  const int n = n0 + n1;
  const bool on = n > 1 || (n == 1 && !p.joint && a.prefix_len > 0);
  const auto locate = [&](int k, const float*& o, float& ls) {
    const int u = k < n0 ? 0 : 1, i = u ? k - n0 : k;
    if (u ? cut1 : cut0) {
      // its first part is the last stretch of its first CTA, the others first stretches
      const int64_t row = (2 * (c0[u] + i) + (i == 0 ? 1 : 0)) * kBlock + brow[u];
      o = p.cut + row * a.dim;
      ls = __ldg(p.cut_lse + row);
    } else {
      const int64_t row = (u ? a.tokens * a.hq : 0) + grow;
      o = p.whole + row * a.dim;
      ls = __ldg(p.whole_lse + row);
    }
  };
  float m = -INFINITY, l = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
  if (on) {
    for (int k = part; k < n; k += W) {
      const float* o;
      float ls;
      locate(k, o, ls);
      if (ls == -INFINITY) continue;
      const float top = fmaxf(m, ls), f = m == -INFINITY ? 0.f : tc::ex2(m - top), g = tc::ex2(ls - top);
      l = l * f + g;
      m = top;
      if (lane * 4 < a.dim) {
        const float4 v = __ldg(reinterpret_cast<const float4*>(o) + lane);
        x[0] = x[0] * f + v.x * g;
        x[1] = x[1] * f + v.y * g;
        x[2] = x[2] * f + v.z * g;
        x[3] = x[3] * f + v.w * g;
      }
    }
  }
  if (W > 1) {
    s_m[warp] = m;
    s_l[warp] = l;
#pragma unroll
    for (int e = 0; e < 4; ++e) s_o[warp][lane * 4 + e] = x[e];
    __syncthreads();
    if (part != 0) return;
    float top = m;
    for (int k = 1; k < W; ++k) top = fmaxf(top, s_m[warp + k]);
    float f = m == -INFINITY ? 0.f : tc::ex2(m - top);
    l = l == l ? l * f : l;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] *= f;
    for (int k = 1; k < W; ++k) {
      f = s_m[warp + k] == -INFINITY ? 0.f : tc::ex2(s_m[warp + k] - top);
      l += s_l[warp + k] == s_l[warp + k] ? s_l[warp + k] * f : s_l[warp + k];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] += s_o[warp + k][lane * 4 + e] * f;
    }
    m = top;
  }
  if (!on) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  if (lane * 4 < a.dim) {
    const uint2 v = make_uint2(Vec16<T>::pack2(x[0] * inv, x[1] * inv), Vec16<T>::pack2(x[2] * inv, x[3] * inv));
    *reinterpret_cast<uint2*>(a.out + (grow * a.dim + lane * 4) * 2) = v;
  }
  if (lane == 0 && a.lse) a.lse[grow] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

// The tensor core takes 16-bit values, sixteen at a time; a head of more than
// 128 of them, of an odd half of sixteen, or of 32-bit values goes row by row.
bool takes_tiles(const AttnArgs& a, int dtype) {
  return dtype != GSEC_F32 && a.dim <= 128 && a.dim % 16 == 0;
}

// Stacking the requests' rows over the prefix pays when they would not fill
// tiles by themselves; with about a tile of rows each (or one request) prefix and
// own keys are better taken in one go, which leaves nothing to join.
TilePlan tile_plan(const AttnArgs& a, int64_t* bytes) {
  TilePlan p{};
  p.ctas = sm_count();
  p.run = a.page & -a.page;  // boxes start at pages, tiles at multiples of 128 keys
  p.run = p.run < 8 ? 0 : (p.run > kKeys ? kKeys : p.run);
  p.joint = a.prefix_len == 0 || a.batch == 1 || a.tokens * a.group >= (int64_t)a.batch * kRows;
  char* at = a.workspace;
  const auto take = [&](int64_t n) {
    char* x = at;
    at += (n + 255) / 256 * 256;
    return x;
  };
  const int64_t rows = a.tokens * a.hq, parts = p.joint ? 0 : 2;
  p.start = reinterpret_cast<int64_t*>(take((a.batch + 1) * 8));
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

bool pool_map(CUtensorMap* m, bool bf16, const char* at, int64_t values, int64_t rows, int64_t pitch, int box_rows) {
  const cuuint64_t size[2] = {(cuuint64_t)values, (cuuint64_t)rows}, stride[1] = {(cuuint64_t)pitch};
  const cuuint32_t box[2] = {64, (cuuint32_t)box_rows}, step[2] = {1, 1};
  const EncodeTiled encode = encode_tiled();
  return encode != nullptr &&
         encode(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
                const_cast<char*>(at), size, stride, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int DP>
int launch_tiles(const AttnArgs& a, cudaStream_t s) {
  int64_t bytes = 0;
  const TilePlan p = tile_plan(a, &bytes);
  PoolMaps maps;
  bool ok = true;
  for (int kv = 0; kv < 2; ++kv) {
    const char* at = a.pool + (kv ? a.plane : 0);
    ok = ok && pool_map(maps.box + kv, Vec16<T>::bf16, at, (int64_t)a.hk * a.dim, a.pool_rows, a.pitch, p.run ? p.run : 1) &&
         pool_map(maps.row + kv, Vec16<T>::bf16, at, (int64_t)a.hk * a.dim, a.pool_rows, a.pitch, 1);
  }
  if (!ok) {
    set_error("prefix_attention: the pool's tensor maps were refused");
    return GSEC_ECUDA;
  }
  constexpr int smem = TileShape<DP>::smem;
  if (launch_cache().blocks_per_sm(attend_tile_kernel<T, DP>, kTileThreads, smem) < 0)
    return check_launch("attend_tile launch shape");
  // a smaller launch would leave the softmax warpgroups waiting for registers that are not there
  static const bool regs_ok = [] {
    cudaFuncAttributes at{};
    return cudaFuncGetAttributes(&at, attend_tile_kernel<T, DP>) == cudaSuccess && at.numRegs == kLaunchRegs;
  }();
  GSEC_REQUIRE(regs_ok, "attend_tile: launch registers are not %d", kLaunchRegs);
  const int rc = launch_rc(launch_pdl(attend_tile_kernel<T, DP>, dim3((unsigned)p.ctas), dim3(kTileThreads), smem, s, a, p, maps),
                           "prefix_attention");
  if (rc) return rc;
  const int64_t rows = a.tokens * a.hq;
  // few rows: eight warps to a row, since each may have a part from every CTA
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
