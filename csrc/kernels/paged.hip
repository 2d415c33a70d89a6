// A key-value cache in pages: block tables and slot maps from request lengths, and the attention of one new token per
// request over its pages.
//
// K cache [P][Hk][page][D]; V cache [P][Hk][page / 8][D][8]: eight tokens of one dimension side by side, so that V^T,
// the matrix operand of P V that wants tokens along its contraction, loads 16 bytes a lane like K does -- no transpose
// in shared memory on the path that reads the whole cache for every token (the append writes two bytes at a time
// instead, once a token).
#include "common.h"

struct PlanDesc {
  const int *cached, *nnew;            // [B] tokens held, tokens to append
  int* table;                          // [B][ld] page ids, entries of new pages are written
  const int *free, *nfree;             // [P] stack of unused page ids, its height
  int *slots;                          // [T] out: page id * page + offset, -1: none
  long long* pos;                      // [T] out: position of each token in its request
  int *start, *lens, *nfree_out;       // [B + 1], [B], [1] out
  int B, W, ld, page, T, P;
};
static_assert(sizeof(PlanDesc) == 104);   // as ops/_lib.py packs it

struct PagedDesc {
  const void *q, *k, *v;
  void* o;
  const int *table, *lens;
  float* part;                         // partial outputs [B][Hq][nsplit][D], then maxima and sums [B][Hq][nsplit][2]
  long long q_bs, q_hs;                // strides of q's batch and head, in elements
  int B, Hq, Hk, D, P, cap, ld, shift, dtype, nsplit, split;   // cap: lengths count up to it; page = 1 << shift
  int most;                            // > 0: splits grow from `split` until all tokens together make at most so many
  float scale;
};
static_assert(sizeof(PagedDesc) == 128);  // as ops/_lib.py packs it

namespace {
constexpr int NTH = 256;

// ---- block tables and slot maps
// Requests are served in order. Request b holds c tokens in ceil(c / page) pages and wants n more. It is refused -- no
// slots, its length stays -- where its pages pass the table's width, its length 31 bits, its tokens the step's buffer,
// or the pages asked for up to and including it the stack. Its i-th new page is the stack's entry nfree - 1 - (pages asked for
// before it) - i. Sums over the requests before b are all that a group needs, so every block forms them itself from
// the lengths (a few KB out of the caches) and one launch does it all: the call's latency is what matters here.
//
// Bound by the latency of its dependent loads (lengths, then stack): 5 us for a decode step of 64 requests, 7 for
// 203 ragged prompts.
struct Want { long long n, need; bool fits; };

__device__ __forceinline__ unsigned pages_of(unsigned tokens, unsigned page) {
  return tokens ? (tokens - 1) / page + 1 : 0;
}

__device__ __forceinline__ Want want_of(const PlanDesc& d, int b, int& c) {
  c = max(d.cached[b], 0);
  const int n = max(d.nnew[b], 0);
  const unsigned old = pages_of(c, d.page), all = pages_of((unsigned)c + n, d.page);   // c + n < 2^32
  const bool fits = all <= (unsigned)d.W && (unsigned)c + n <= 0x7fffffffu;
  return {n, fits ? all - old : 0, fits};
}

__device__ __forceinline__ long long wave_sum_ll(long long v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// sum over the threads before this one
__device__ __forceinline__ long long block_before(long long v, long long* red) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  long long x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const long long y = __shfl_up(x, o, 64);
    x += lane >= o ? y : 0;
  }
  __syncthreads();
  if (lane == 63) red[w] = x;
  __syncthreads();
  x -= v;
  for (int i = 0; i < w; ++i) x += red[i];
  return x;
}

// grid (request groups + 1, token segments): 8 requests a block, 32 lanes each; the last group's block forms what all
// requests share
constexpr int GR = 8, GL = NTH / GR;

__global__ __launch_bounds__(NTH) void page_plan_kernel(const PlanDesc d) {
  __shared__ long long red[3][NTH / 64];
  __shared__ long long s_n[GR], s_need[GR];
  const int tid = threadIdx.x, r0 = blockIdx.x * GR;
  const int avail = min(max(*d.nfree, 0), d.P);
  const bool first = blockIdx.y == 0;
  if (blockIdx.x == gridDim.x - 1) {
    if (!first) return;
    // what is left of the stack: the pages asked for up to the last request that got some. Thread t takes its run of
    // requests
    const int per = (d.B + NTH - 1) / NTH, j0 = min(d.B, tid * per), j1 = min(d.B, j0 + per);
    int c;
    long long n = 0, need = 0, taken = 0;
    for (int j = j0; j < j1; ++j) n += want_of(d, j, c).n;
    const long long at0 = block_before(n, red[0]);
    if (tid == NTH - 1) d.start[d.B] = (int)min(at0 + n, (long long)0x7fffffff);
    long long at = at0;
    for (int j = j0; j < j1; ++j) {
      const Want x = want_of(d, j, c);
      at += x.n;
      if (at <= d.T) need += x.need;
    }
    long long asked = block_before(need, red[1]);
    at = at0;
    for (int j = j0; j < j1; ++j) {
      const Want x = want_of(d, j, c);
      at += x.n;
      if (at > d.T) break;
      asked += x.need;
      if (x.need > 0 && asked <= avail) taken = asked;
    }
    for (int o = 32; o > 0; o >>= 1) taken = max(taken, (long long)__shfl_xor(taken, o, 64));
    if ((tid & 63) == 0) red[2][tid >> 6] = taken;
    __syncthreads();
    if (tid == 0) {
      for (int i = 0; i < NTH / 64; ++i) taken = max(taken, red[2][i]);
      *d.nfree_out = (int)(avail - taken);
    }
    return;
  }
  long long n0 = 0, need0 = 0, total = 0;        // tokens and pages before the block's requests; all tokens
  for (int j = tid; j < d.B; j += NTH) {
    int c;
    const Want w = want_of(d, j, c);
    total += w.n;
    if (j < r0) { n0 += w.n; need0 += w.need; }
  }
  n0 = wave_sum_ll(n0);
  need0 = wave_sum_ll(need0);
  total = wave_sum_ll(total);
  if ((tid & 63) == 0) { red[0][tid >> 6] = n0; red[1][tid >> 6] = need0; red[2][tid >> 6] = total; }
  const int g = tid / GL, l = tid % GL, b = r0 + g;
  int c = 0;
  Want w = {0, 0, false};
  if (b < d.B) w = want_of(d, b, c);
  if (l == 0) { s_n[g] = w.n; s_need[g] = w.need; }
  __syncthreads();
  n0 = need0 = total = 0;
#pragma unroll
  for (int i = 0; i < NTH / 64; ++i) { n0 += red[0][i]; need0 += red[1][i]; total += red[2][i]; }
  for (int i = 0; i < g; ++i) { n0 += s_n[i]; need0 += s_need[i]; }
  if (b < d.B) {
    const bool room = w.fits && n0 + w.n <= d.T;
    const bool ok = room && (w.need == 0 || need0 + w.need <= avail);
    const unsigned old = pages_of(c, d.page);
    if (first && l == 0) {
      d.lens[b] = ok ? (int)(c + w.n) : c;
      d.start[b] = (int)min(n0, (long long)0x7fffffff);
    }
    // (an entry of the stack is used only where ok: its index is then below avail)
    if (first && ok)
      for (long long i = l; i < w.need; i += GL) d.table[(long long)b * d.ld + old + i] = d.free[avail - 1 - need0 - i];
    for (long long i = (long long)blockIdx.y * GL + l; i < w.n && n0 + i < d.T; i += (long long)gridDim.y * GL) {
      const long long p = c + i;
      int slot = -1;
      if (ok) {                                    // p < W * page, below 2^32
        const unsigned e = (unsigned)p / (unsigned)d.page, off = (unsigned)p % (unsigned)d.page;
        const int id = e < old ? d.table[(long long)b * d.ld + e] : d.free[avail - 1 - need0 - (e - old)];
        if ((unsigned)id < (unsigned)d.P) slot = id * d.page + (int)off;
      }
      d.slots[n0 + i] = slot;
      d.pos[n0 + i] = p;
    }
  }
  // places of the step's buffer behind the last token
  const long long gx = gridDim.x - 1;
  for (long long t = total + (blockIdx.y * gx + blockIdx.x) * NTH + tid; t < d.T; t += gx * gridDim.y * NTH) {
    d.slots[t] = -1;
    d.pos[t] = 0;
  }
}

// pages of the requests that are done go back onto the stack, in request order; their lengths become 0. Ids outside the
// pool are left out. One block, a piece of 1024 requests at a time: a thread a request for its length, a wave a request
// for its row (once to count its ids, up to what the stack has room for; once to copy them)
__global__ __launch_bounds__(1024) void page_release_kernel(const unsigned char* __restrict__ done, int* lens,
                                                           const int* __restrict__ table, int* stack, int* nfree, int B,
                                                           int W, int ld, int page, int P) {
  __shared__ int rows[1024];                      // entries of a request's row
  __shared__ long long cnt[1024];                 // its ids; 1024 times the stack's room may pass 31 bits
  __shared__ int base;
  const int tid = threadIdx.x, lane = tid & 63;
  if (tid == 0) base = min(max(*nfree, 0), P);
  for (int b0 = 0; b0 < B; b0 += 1024) {
    const int b = b0 + tid;
    int n = 0;
    if (b < B && done[b]) n = (int)min(((long long)max(lens[b], 0) + page - 1) / page, (long long)W);
    __syncthreads();                              // the piece before this one has read rows, cnt and base
    rows[tid] = n;
    cnt[tid] = 0;
    __syncthreads();
    const int at0 = base, room = P - at0;
    for (int r = tid >> 6; r < 1024 && b0 + r < B; r += 16) {
      const int m = rows[r];
      if (m == 0) continue;
      const int* row = table + (long long)(b0 + r) * ld;
      int c = 0;
      for (long long i = 0; i < m && c < room; i += 64)
        c += __popcll(__ballot(i + lane < m && (unsigned)row[min(i + lane, m - 1LL)] < (unsigned)P));
      if (lane == 0) cnt[r] = c;
    }
    __syncthreads();
    for (int o = 1; o < 1024; o <<= 1) {          // inclusive prefix sums
      const long long v = tid >= o ? cnt[tid - o] : 0;
      __syncthreads();
      cnt[tid] += v;
      __syncthreads();
    }
    if (b < B && done[b]) lens[b] = 0;
    for (int r = tid >> 6; r < 1024 && b0 + r < B; r += 16) {
      long long at = r ? cnt[r - 1] : 0;          // where the row's ids go, behind at0
      const int m = rows[r];
      const int* row = table + (long long)(b0 + r) * ld;
      for (long long i = 0; i < m && at < room; i += 64) {
        const int id = row[min(i + lane, m - 1LL)];
        const unsigned long long live = __ballot(i + lane < m && (unsigned)id < (unsigned)P);
        const long long to = at + __popcll(live & ((1ULL << lane) - 1));
        if (live >> lane & 1 && to < room) stack[at0 + to] = id;
        at += __popcll(live);
      }
    }
    __syncthreads();
    if (tid == 0) base = (int)min(at0 + cnt[1023], (long long)P);
  }
  __syncthreads();
  if (tid == 0) *nfree = base;
}

// ---- attention of one token per request
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8_t;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4_t;

template <int TYPE> struct Mat;
template <> struct Mat<1> {
  typedef bf16x8_t v;
  static constexpr int PARTS = 3;                 // summands of a softmax weight, and the unit that it counts in
  static constexpr float UNIT = 1.f;
  static constexpr uint16_t LEAST = 0x0080;       // a least number above 0
  static __device__ __forceinline__ f32x4_t mul(v a, v b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint16_t bits(float f) { return f2bf(f); }
  static __device__ __forceinline__ float back(uint16_t b) { return bf2f(b); }
};
template <> struct Mat<2> {
  typedef f16x8_t v;
  static constexpr int PARTS = 2;
  static constexpr float UNIT = 32768.f;          // the largest power of two in fp16
  static constexpr uint16_t LEAST = 0x0001;
  static __device__ __forceinline__ f32x4_t mul(v a, v b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint16_t bits(float f) { return __builtin_bit_cast(uint16_t, (_Float16)f); }
  static __device__ __forceinline__ float back(uint16_t b) { return (float)__builtin_bit_cast(_Float16, b); }
};

// o[b][h] = sum_j softmax_j(scale q[b][h] . k_j) v_j over the lens[b] tokens of request b; 0 where it holds none.
//
// A block takes one request, one key head and its (up to 16) query heads, and one split of the length; a wave takes
// every fourth tile of 32 keys. S^T = K Q^T: 16x16x32 products with 16 keys as rows, the query heads as columns. Row m
// of the two products of a tile is key 8 (m / 4) + 4 t + m % 4, so a lane ends up with the scores of eight
// neighbouring keys 8 (lane / 16) + 0..7 of one query head: just what the P operand of O^T = V^T P takes from it. P
// never leaves its lane. With one query head per key head 15 of the 16 columns are idle: the products' time is
// still a small part of the loads' (32 products in bf16 to 16 KB a tile and wave, heads of 128: 8 for S, 24 for O).
//
// Softmax in one pass with the running maximum; P enters the product as summands of the cache's type, each what the
// rounding of those before it left: in bf16 three, all 24 bits of a weight (two, 16 bits, are up to 2 % faster: 64 heads
// x 96 64.4 -> 65.6 us). In fp16, which ends at 2^-24, two, and weights count in units of 2^-15 (UNIT; the sum l too, so
// the quotient is the same): 22 bits of those above 2^-28 of the largest, 2^-40 of it for the smaller ones. (In units of
// 1, a key 16 nats above 2047 others left these 6 % too heavy, 19.5 nats nothing.) Waves, then splits, are joined by
// their maxima and sums.
//
// Blocks are ordered by key head, request, split, and the requests turn by one with each split. With the split first,
// the blocks that have work in a table much wider than its requests' lengths all met one XCD (16 requests of 1 to 2000
// tokens, 64 splits of 2048: 175 us, 24 in this order); without the turn the splits of one long request among short
// ones met the same CUs (120000 tokens among 63 short: 239 us, 135 with it).
//
// Keys past the length, and pages whose id is not one, have weight 0 and a value of 0 whatever the cache holds there.
// An infinite value that counts, times its weight's second summand, is NaN (0 is common there) or the other infinity: a
// wave whose sums are not all finite goes over its keys once more with the first summands alone, and takes those of the
// dims that are not. The check costs 150 short requests 0.3 us of 10. The waves a SIMD are asked for because the compiler
// would take registers that leave room for two waves with heads of 128, where there are three (8 requests of up to 2048
// tokens 22.1 -> 20.7 us).
//
// Bound by the read of the cache. V goes past the caches: a load takes whole lines of it. K's loads take half a line
// of each key row, the next load the other half out of the cache; past it they cost 7 % more. At 64 x ~6100 tokens, 8
// key heads x 128, 4 query heads each (1.6 GB): 262 us with the join, 6.1 TB/s, where a bare read of such data reaches
// 7.1.
constexpr float LOG2E = 1.4426950408889634f;
constexpr float NEG = -3.0e38f;                   // a running maximum before any key

// tokens a split of this call. `most` > 0 (only for few requests): it follows from the lengths that the requests have,
// which the host does not know, so that a table much wider than they are costs nothing. No request then has more than
// `most` splits: ceil(a / ceil(n / most)) <= most for its share a of all n
constexpr int MAX_SUM = 16;

__device__ __forceinline__ int split_of(const PagedDesc& d) {
  if (d.most == 0) return d.split;
  const int lane = threadIdx.x & 63;
  int n = lane < d.B ? (min(max(d.lens[lane], 0), d.cap) + 127) >> 7 : 0;   // units of 128 tokens, below 2^28
#pragma unroll
  for (int o = MAX_SUM / 2; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
  n = __builtin_amdgcn_readfirstlane(n);
  return max(d.split, min((n + d.most - 1) / d.most, 1 << 23) * 128);
}

template <int TYPE, int D>
__global__ __launch_bounds__(NTH, D <= 64 ? 4 : D <= 128 ? 3 : 1) void paged_attn_kernel(const PagedDesc d) {
  typedef typename Mat<TYPE>::v vec;
  constexpr int NK = D / 32, NV = D / 16, NW = NTH / 64;
  __shared__ float sm[NW][16], sl[NW][16];
  // [NW][query heads of the block][D + 4]: one head's 2 KB leave room for four blocks a CU, 16 heads' for three
  extern __shared__ float sacc[];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, n = lane & 15, g = lane >> 4;
  const int sp = blockIdx.z, b = (blockIdx.y + blockIdx.z) % gridDim.y;
  const int len = min(max(d.lens[b], 0), d.cap), split = split_of(d);
  if (sp > 0 && (long long)sp * split >= len) return;
  const int k0 = sp * split, k1 = min(len, k0 + split);
  const int G = d.Hq / d.Hk, gi = blockIdx.x / d.Hk, hk = blockIdx.x % d.Hk;
  const int h0 = hk * G + gi * 16, gc = min(16, G - gi * 16);

  const uint16_t* qp = (const uint16_t*)d.q + b * d.q_bs + (long long)(h0 + min(n, gc - 1)) * d.q_hs + 8 * g;
  vec q[NK];
#pragma unroll
  for (int j = 0; j < NK; ++j) q[j] = *reinterpret_cast<const vec*>(qp + 32 * j);
  f32x4_t acc[NV];
  float m, l;
  const float sc = d.scale * LOG2E;
  const int* tb = d.table + (long long)b * d.ld;
  const uint16_t *K = (const uint16_t*)d.k, *V = (const uint16_t*)d.v;
  const int in_page = (1 << d.shift) - 1;
  const long long row = (long long)D << d.shift, pst = d.Hk * row, hoff = hk * row;

  // this lane's key rows (one per product) and the first of its eight value tokens of a tile; their page ids are loaded
  // one tile ahead (never past the table: a tile behind the length reads whatever ids stand there, none is followed
  // outside the pool)
  const int ra = 8 * (n >> 2) + (n & 3), rv = 8 * g;
  int ia, ib, iv;
  auto ids = [&](int t0) {
    ia = tb[min(t0 + ra, d.cap - 1) >> d.shift];
    ib = tb[min(t0 + ra + 4, d.cap - 1) >> d.shift];
    iv = tb[min(t0 + rv, d.cap - 1) >> d.shift];
  };
  // one pass over the wave's keys. INF: by the weights' first summands alone, 0 only where the weight is
  auto pass = [&](auto which) {
    constexpr bool INF = decltype(which)::value;
    m = NEG;
    l = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) acc[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    if (d.cap > 0) ids(k0 + 32 * w);
    for (int t0 = k0 + 32 * w; t0 < k1; t0 += 32 * NW) {
      const bool bad_v = (unsigned)iv >= (unsigned)d.P;
      const long long ja = (unsigned)ia < (unsigned)d.P ? ia : 0, jb = (unsigned)ib < (unsigned)d.P ? ib : 0;
      const long long jv = bad_v ? 0 : iv;
      const uint16_t* pa = K + ja * pst + hoff + ((t0 + ra) & in_page) * D + 8 * g;
      const uint16_t* pb = K + jb * pst + hoff + ((t0 + ra + 4) & in_page) * D + 8 * g;
      const uint16_t* pv = V + jv * pst + hoff + ((t0 + rv) & in_page) * D + 8 * n;
      f32x4_t s0{0.f, 0.f, 0.f, 0.f}, s1{0.f, 0.f, 0.f, 0.f};
      vec a[NK], c[NK], v[NV];
#pragma unroll
      for (int j = 0; j < NK; ++j) {
        a[j] = *reinterpret_cast<const vec*>(pa + 32 * j);
        c[j] = *reinterpret_cast<const vec*>(pb + 32 * j);
      }
#pragma unroll
      for (int j = 0; j < NV; ++j) v[j] = __builtin_nontemporal_load(reinterpret_cast<const vec*>(pv + 128 * j));
      ids(t0 + 32 * NW);
      // all loads before the products: within the registers of three waves a SIMD the compiler starts some behind them
      // (64 long grouped contexts x 128: 255 us, 248 so; heads of 256, one wave a SIMD: 213 us, 223 so)
      if constexpr (D <= 128) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < NK; ++j) {
        s0 = Mat<TYPE>::mul(a[j], q[j], s0);
        s1 = Mat<TYPE>::mul(c[j], q[j], s1);
      }
      float p[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) { p[i] = s0[i] * sc; p[4 + i] = s1[i] * sc; }
      const int left = bad_v ? 0 : k1 - (t0 + 8 * g);         // how many of the lane's eight keys count
      if (__any(left < 8)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = i < left ? p[i] : -INFINITY;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          u32x4_t x = __builtin_bit_cast(u32x4_t, v[j]);
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = left >= 2 * i + 2 ? x[i] : left == 2 * i + 1 ? x[i] & 0xffffu : 0u;
          v[j] = __builtin_bit_cast(vec, x);
        }
      }
      float mx = p[0];
#pragma unroll
      for (int i = 1; i < 8; ++i) mx = fmaxf(mx, p[i]);
      mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
      mx = fmaxf(m, fmaxf(mx, __shfl_xor(mx, 32, 64)));
      const float f = __builtin_amdgcn_exp2f(m - mx);
      m = mx;
      l *= f;
#pragma unroll
      for (int i = 0; i < NV; ++i) acc[i] *= f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        p[i] = __builtin_amdgcn_exp2f(p[i] - m);
        l += p[i];
        p[i] *= Mat<TYPE>::UNIT;
      }
#pragma unroll
      for (int s = 0; s < (INF ? 1 : Mat<TYPE>::PARTS); ++s) {
        u32x4_t part;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint16_t h[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float& x = p[2 * i + e];
            h[e] = Mat<TYPE>::bits(x);
            if (INF && x > 0.f && h[e] < Mat<TYPE>::LEAST) h[e] = Mat<TYPE>::LEAST;
            x -= Mat<TYPE>::back(h[e]);
          }
          part[i] = h[0] | (uint32_t)h[1] << 16;
        }
#pragma unroll
        for (int j = 0; j < NV; ++j) acc[j] = Mat<TYPE>::mul(v[j], __builtin_bit_cast(vec, part), acc[j]);
      }
    }
  };
  float* const mine = &sacc[(w * gc + min(n, gc - 1)) * (D + 4) + 4 * g];
  pass(std::false_type{});
  f32x4_t odd{0.f, 0.f, 0.f, 0.f};                // NaN where a sum is not finite
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    if (n < gc) *reinterpret_cast<f32x4_t*>(mine + 16 * j) = acc[j];
#pragma unroll
    for (int i = 0; i < 4; ++i) odd[i] = fmaf(acc[j][i], 0.f, odd[i]);
  }
  if (__any(!(odd[0] + odd[1] + odd[2] + odd[3] == 0.f))) {
    pass(std::true_type{});
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n < gc && !(fabsf(mine[16 * j + i]) < INFINITY)) mine[16 * j + i] = acc[j][i];
  }
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  if (g == 0) { sm[w][n] = m; sl[w][n] = l * Mat<TYPE>::UNIT; }
  __syncthreads();
  const bool whole = len <= split;
  for (int e = threadIdx.x; e < gc * D; e += NTH) {
    const int h = e / D, i = e % D;
    float M = sm[0][h], L = 0.f, o = 0.f;
#pragma unroll
    for (int x = 1; x < NW; ++x) M = fmaxf(M, sm[x][h]);
#pragma unroll
    for (int x = 0; x < NW; ++x) {
      const float f = __builtin_amdgcn_exp2f(sm[x][h] - M);
      L += f * sl[x][h];
      o += f * sacc[(x * gc + h) * (D + 4) + i];
    }
    if (whole) {
      ((uint16_t*)d.o)[((long long)b * d.Hq + h0 + h) * D + i] = Mat<TYPE>::bits(L != 0.f ? o / L : 0.f);
    } else {
      const long long at = ((long long)b * d.Hq + h0 + h) * d.nsplit + sp;
      d.part[at * D + i] = o;
      if (i == 0) {
        float* ml = d.part + (long long)d.B * d.Hq * d.nsplit * D + at * 2;
        ml[0] = M;
        ml[1] = L;
      }
    }
  }
}

// Splits of one request joined, up to NS of them: a wave a query head, its lanes over the dims, every row and weight
// loaded at once -- no exchange, one round trip after the length's (64 requests x 32 heads, 4 splits: 4.2 us; the
// kernel for many, three round trips: 5.4)
template <int TYPE, int D, int NS>
__global__ __launch_bounds__(NTH) void paged_join_few_kernel(const PagedDesc d) {
  const long long u = (long long)blockIdx.x * (NTH / 64) + (threadIdx.x >> 6);
  if (u >= (long long)d.B * d.Hq) return;
  const int lane = threadIdx.x & 63;
  const int len = min(max(d.lens[u / d.Hq], 0), d.cap), split = split_of(d);
  if (len <= split) return;
  const int ns = (len + split - 1) / split;
  const float* ml = d.part + (long long)d.B * d.Hq * d.nsplit * D + u * d.nsplit * 2;
  const float* pt = d.part + u * d.nsplit * D;
  constexpr int R = (D + 63) / 64;                   // dims lane, lane + 64, ...
  float m[NS], l[NS], x[NS][R];
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    const int j = min(s, ns - 1);                    // past the last split: its row again, with weight 0
    m[s] = ml[2 * j];
    l[s] = ml[2 * j + 1];
#pragma unroll
    for (int r = 0; r < R; ++r) x[s][r] = pt[j * D + min(lane + 64 * r, D - 1)];
  }
  float M = m[0];
#pragma unroll
  for (int s = 1; s < NS; ++s) M = fmaxf(M, m[s]);
  float L = 0.f, o[R];
#pragma unroll
  for (int r = 0; r < R; ++r) o[r] = 0.f;
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    const float f = __builtin_amdgcn_exp2f(m[s] - M);
    if (s < ns) {
      L += f * l[s];
#pragma unroll
      for (int r = 0; r < R; ++r) o[r] += f * x[s][r];
    }
  }
  uint16_t* out = (uint16_t*)d.o + u * D;
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (lane + 64 * r < D) out[lane + 64 * r] = Mat<TYPE>::bits(L != 0.f ? o[r] / L : 0.f);
}

// Many splits of one query head: block (Hq, B). The weights of the splits first, each by a thread; then D / 4 threads a
// split row, 1024 / D rows side by side, joined in a fixed order
constexpr int MAX_SPLITS = 1024;

template <int TYPE>
__global__ __launch_bounds__(NTH) void paged_join_kernel(const PagedDesc d) {
  __shared__ float wt[MAX_SPLITS], red[2][NTH / 64];
  __shared__ f32x4_t so[NTH];
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const int len = min(max(d.lens[b], 0), d.cap), split = split_of(d);
  if (len <= split) return;
  const int ns = (len + split - 1) / split;
  const long long at = ((long long)b * d.Hq + h) * d.nsplit;
  const float* ml = d.part + (long long)d.B * d.Hq * d.nsplit * d.D + at * 2;
  float M = NEG;
  for (int s = tid; s < ns; s += NTH) M = fmaxf(M, ml[2 * s]);
  M = wave_max(M);
  if ((tid & 63) == 0) red[0][tid >> 6] = M;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NTH / 64; ++i) M = fmaxf(M, red[0][i]);
  float L = 0.f;
  for (int s = tid; s < ns; s += NTH) {
    const float f = __builtin_amdgcn_exp2f(ml[2 * s] - M);
    wt[s] = f;
    L += f * ml[2 * s + 1];
  }
  L = wave_sum(L);
  if ((tid & 63) == 0) red[1][tid >> 6] = L;
  __syncthreads();
  L = 0.f;
#pragma unroll
  for (int i = 0; i < NTH / 64; ++i) L += red[1][i];
  const int per = d.D / 4, rows = NTH / per, r = tid / per, c = tid % per;
  const f32x4_t* pt = reinterpret_cast<const f32x4_t*>(d.part) + at * per + c;
  f32x4_t o{0.f, 0.f, 0.f, 0.f};
  if (r < rows)
#pragma unroll 4
    for (int s = r; s < ns; s += rows) o += pt[(long long)s * per] * wt[s];
  so[tid] = o;
  __syncthreads();
  if (r != 0) return;
  for (int i = 1; i < rows; ++i) o += so[i * per + c];
  uint16_t* out = (uint16_t*)d.o + ((long long)b * d.Hq + h) * d.D + 4 * c;
#pragma unroll
  for (int i = 0; i < 4; ++i) out[i] = Mat<TYPE>::bits(L != 0.f ? o[i] / L : 0.f);
}

template <int TYPE, int D>
int attn_of(const PagedDesc& d, hipStream_t st) {
  const int G = d.Hq / d.Hk, ng = (G + 15) / 16, gc = G < 16 ? G : 16;
  hipLaunchKernelGGL((paged_attn_kernel<TYPE, D>), dim3(d.Hk * ng, d.B, d.nsplit), dim3(NTH),
                     NTH / 64 * gc * (D + 4) * sizeof(float), st, d);
  const int rc = (int)hipGetLastError();
  if (rc || d.nsplit == 1) return rc;
  const long long rows = (long long)d.B * d.Hq;
  const dim3 few((unsigned)((rows + NTH / 64 - 1) / (NTH / 64)));
  if (d.nsplit <= 4) hipLaunchKernelGGL((paged_join_few_kernel<TYPE, D, 4>), few, dim3(NTH), 0, st, d);
  else if (d.nsplit <= 12) hipLaunchKernelGGL((paged_join_few_kernel<TYPE, D, 12>), few, dim3(NTH), 0, st, d);
  else hipLaunchKernelGGL(paged_join_kernel<TYPE>, dim3(d.Hq, d.B), dim3(NTH), 0, st, d);
  return (int)hipGetLastError();
}

template <int TYPE>
int attn(const PagedDesc& d, hipStream_t st) {
  switch (d.D) {
    case 32: return attn_of<TYPE, 32>(d, st);
    case 64: return attn_of<TYPE, 64>(d, st);
    case 96: return attn_of<TYPE, 96>(d, st);
    case 128: return attn_of<TYPE, 128>(d, st);
    case 256: return attn_of<TYPE, 256>(d, st);
  }
  return -2;
}

// whether a buffer that the plan writes shares memory with another of its buffers
bool plan_overlaps(const PlanDesc& d) {
  struct { const void* p; size_t n; } s[10] = {
      {d.table, 4 * ((size_t)(d.B - 1) * d.ld + d.W)}, {d.slots, 4 * (size_t)d.T}, {d.pos, 8 * (size_t)d.T},
      {d.start, 4 * ((size_t)d.B + 1)}, {d.lens, 4 * (size_t)d.B}, {d.nfree_out, 4}, {d.cached, 4 * (size_t)d.B},
      {d.nnew, 4 * (size_t)d.B}, {d.free, 4 * (size_t)d.P}, {d.nfree, 4}};
  for (int i = 0; i < 6; ++i)
    for (int j = i + 1; j < 10; ++j)
      if (overlap(s[i].p, s[i].n, s[j].p, s[j].n)) return true;
  return false;
}

// the outputs may take the queries' own place (a block reads its rows first), but no other part of what the call reads
bool out_overlaps(const PagedDesc& d) {
  const size_t n = 2 * (size_t)d.B * d.Hq * d.D, pool = 2 * ((size_t)d.P << d.shift) * d.Hk * d.D;
  const bool own = d.o == d.q && (d.q_hs == d.D || d.Hq == 1) && (d.q_bs == (long long)d.Hq * d.D || d.B == 1);
  return (!own && overlap(d.o, n, d.q, 2 * ((d.B - 1) * d.q_bs + (d.Hq - 1) * d.q_hs + d.D))) ||
         overlap(d.o, n, d.k, pool) || overlap(d.o, n, d.v, pool) || overlap(d.o, n, d.lens, 4 * (size_t)d.B) ||
         overlap(d.o, n, d.table, 4 * ((size_t)(d.B - 1) * d.ld + ((d.cap - 1) >> d.shift) + 1));
}
}  // namespace

OBST_API int obst_page_plan(const PlanDesc* d, hipStream_t st) {
  if (!d || d->B < 1 || d->W < 1 || d->ld < d->W || d->page < 1 || d->T < 0 || d->P < 1) return -1;
  if (plan_overlaps(*d)) return -2;
  const int gx = (d->B + GR - 1) / GR;
  long long gy = d->T / ((long long)d->B * GL * 4);      // a few rounds of a request's tokens per lane
  gy = gy < 1 ? 1 : gy > 64 ? 64 : gy;
  hipLaunchKernelGGL(page_plan_kernel, dim3(gx + 1, (unsigned)gy), dim3(NTH), 0, st, *d);
  return (int)hipGetLastError();
}

OBST_API int obst_page_release(const void* done, void* lens, const void* table, void* stack, void* nfree, int B, int W,
                               int ld, int page, int P, hipStream_t st) {
  if (B < 1 || W < 1 || ld < W || page < 1 || P < 1) return -1;
  hipLaunchKernelGGL(page_release_kernel, dim3(1), dim3(1024), 0, st, (const unsigned char*)done, (int*)lens,
                     (const int*)table, (int*)stack, (int*)nfree, B, W, ld, page, P);
  return (int)hipGetLastError();
}

OBST_API int obst_paged_attn(const PagedDesc* d, hipStream_t st) {
  if (!d || d->B < 1 || d->B > 65535 || d->Hk < 1 || d->Hq < 1 || d->Hq % d->Hk || d->P < 1 || d->cap < 0 ||
      d->cap > 1 << 30 ||
      d->nsplit < 1 || d->nsplit > MAX_SPLITS || d->split < 32 || d->split % 32 || (d->nsplit > 1 && !d->part))
    return -1;
  if (d->shift < 4 || d->shift > 8 || (long long)d->ld << d->shift < d->cap) return -3;
  if (d->most < 0 || (d->most > 0 && (d->B > MAX_SUM || d->split % 128))) return -6;
  if (d->cap > (long long)d->nsplit * d->split && (d->most == 0 || d->nsplit < d->most)) return -4;
  if (out_overlaps(*d)) return -7;
  if (d->dtype == 1) return attn<1>(*d, st);
  if (d->dtype == 2) return attn<2>(*d, st);
  return -5;
}
