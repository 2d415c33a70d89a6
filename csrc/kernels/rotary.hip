// Per-head norm and rotary positions of queries and keys in one pass, forward and backward, and the serving form that
// writes the turned keys and the values into the pages of a key-value cache.
//
// x is one head of one token (D elements). With a weight w:  n = x r w,  r = (mean x^2 + eps)^-1/2;  without: n = x.
// The first R dims of n form R/2 pairs (a, b) -- (i, i + R/2), or (2i, 2i + 1) interleaved -- and turn by the angle
// pos * freq[i], scaled by m:  a' = m (a cos - b sin),  b' = m (b cos + a sin).  The rest passes through.
// Backward: g = the output gradient turned by the negative angle (times m);  with h = g w and u = x r:
// dx = r (h - u mean(h u)),  dw = sum over tokens and heads of g u.
//
// Angles are formed in 64 bits as turns (pos * freq / 2 pi, minus its nearest integer): at position 10^5 a 32-bit
// product is off by 10^-2 radians. sin and cos then see an argument within half a turn.
//
// A head's elements are cut into items of two chunks of VEC elements (16 bytes): one lane holds both members of its
// pairs, so the rotation needs no exchange between lanes, and an angle is computed once per lane and token and used for
// every head of the wave's unit. LPH lanes hold a head, a wave 64 / LPH heads. Memory-bound: each element is read once
// and written once. VEC = 1 takes what 16-byte accesses cannot (odd head widths, strides or addresses).
#include <hip/hip_fp16.h>
#include "common.h"

struct RotDesc {
  const void *q, *k, *v, *gq, *gk;      // inputs [T, H, D] (strides below); output gradients (backward)
  void *qo, *ko, *vo;                   // outputs, contiguous [T, H, D]; ko / vo: the caches when slots is set
  const void *wq, *wk;                  // norm weights [D] or null
  const double* freqs;                  // [R / 2]
  const long long* pos;                 // [T]
  const int* slots;                     // [T] or null
  float* part;                          // backward: weight-gradient partials [blocks][2][D]
  void *dwq, *dwk;                      // backward: weight gradients
  long long q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, gq_ts, gq_hs, gk_ts, gk_hs;   // token / head strides, in elements
  long long T, nslots;
  int Hq, Hk, D, R, inter, dtype, wtype, dwtype, dwacc, page;   // types: 0 fp32, 1 bf16, 2 fp16
  float mscale, eps;
};

namespace {
constexpr int NTH = 256;

template <int T> struct Elem;
template <> struct Elem<0> { typedef float t; static constexpr int VEC = 4; };
template <> struct Elem<1> { typedef bf16_t t; static constexpr int VEC = 8; };
template <> struct Elem<2> { typedef __half t; static constexpr int VEC = 8; };

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(bf16_t v) { return bf2f(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ void from_f(float f, float& o) { o = f; }
__device__ __forceinline__ void from_f(float f, bf16_t& o) { o = f2bf(f); }
__device__ __forceinline__ void from_f(float f, __half& o) { o = __float2half(f); }

template <typename E, int VEC>
struct alignas(sizeof(E) * VEC) Chunk { E e[VEC]; };

// lanes without an element read `safe` and see zeros: a load under a branch would be waited for inside it
template <typename E, int VEC>
__device__ __forceinline__ void load(const E* p, const E* safe, bool on, float* f) {
  const Chunk<E, VEC> c = *reinterpret_cast<const Chunk<E, VEC>*>(on ? p : safe);
#pragma unroll
  for (int i = 0; i < VEC; ++i) f[i] = on ? to_f(c.e[i]) : 0.f;
}
template <typename E, int VEC>
__device__ __forceinline__ void store(E* p, const float* f) {
  Chunk<E, VEC> c;
#pragma unroll
  for (int i = 0; i < VEC; ++i) from_f(f[i], c.e[i]);
  *reinterpret_cast<Chunk<E, VEC>*>(p) = c;
}

__device__ __forceinline__ float load_w(const void* w, int type, int i) {
  return type == 0 ? ((const float*)w)[i] : type == 1 ? bf2f(((const bf16_t*)w)[i]) : __half2float(((const __half*)w)[i]);
}

// first elements of the two chunks of item `i` of a head; -1: no such chunk
template <int VEC>
__device__ __forceinline__ void item_chunks(int i, int D, int R, int inter, int& a, int& b) {
  if (VEC > 1 && inter) {                        // pairs lie inside a chunk: the head's two halves, chunk by chunk
    const int nc = D / VEC, n = (nc + 1) / 2;
    a = i < n ? i * VEC : -1;
    b = i < n && i + n < nc ? (i + n) * VEC : -1;
    return;
  }
  const int nr = R / (2 * VEC);
  if (i < nr) {
    a = VEC == 1 && inter ? 2 * i : i * VEC;
    b = VEC == 1 && inter ? 2 * i + 1 : R / 2 + i * VEC;
    return;
  }
  const int nt = (D - R) / VEC, n = (nt + 1) / 2, j = i - nr;
  a = j < n ? R + j * VEC : -1;
  b = j < n && j + n < nt ? R + (j + n) * VEC : -1;
}

// the pairs of a lane's two chunks: (a[i], b[i]), or inside each chunk
template <int VEC, bool INSIDE>
__device__ __forceinline__ void turn(float* a, float* b, const float* c, const float* s) {
  if (INSIDE) {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) {
      const float x = a[2 * i], y = a[2 * i + 1], z = b[2 * i], w = b[2 * i + 1];
      a[2 * i] = x * c[i] - y * s[i];
      a[2 * i + 1] = y * c[i] + x * s[i];
      b[2 * i] = z * c[VEC / 2 + i] - w * s[VEC / 2 + i];
      b[2 * i + 1] = w * c[VEC / 2 + i] + z * s[VEC / 2 + i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float x = a[i], y = b[i];
      a[i] = x * c[i] - y * s[i];
      b[i] = y * c[i] + x * s[i];
    }
  }
}

// the frequencies (in turns per position) of a lane's VEC pairs; -1 stands for "does not turn"
template <int VEC, bool INSIDE>
__device__ __forceinline__ void pair_freqs(const RotDesc& d, int a, int b, int item, double* f) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    int p;
    if (INSIDE) {
      const int e = i < VEC / 2 ? a : b;
      p = e >= 0 && e < d.R ? e / 2 + i % (VEC / 2) : -1;
    } else {
      p = a >= 0 && a < d.R ? (VEC == 1 ? item : a + i) : -1;
    }
    f[i] = p >= 0 ? d.freqs[p] * 0.15915494309189535 : -1.0;
  }
}

template <int VEC>
__device__ __forceinline__ void angles(const double* f, double pos, float m, float sign, float* c, float* s) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    const double t = pos * f[i];
    const float x = 2.f * (float)(t - rint(t));
    float sn, cs;
    sincospif(x, &sn, &cs);
    const bool on = f[i] >= 0.0;
    c[i] = on ? m * cs : 1.f;
    s[i] = on ? sign * m * sn : 0.f;
  }
}

__device__ __forceinline__ float sum_lanes(float v, int lph) {
  for (int o = lph >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// ---- forward. A unit is U passes of 64 / LPH heads of one token; heads are q's, then k's, then (CACHE) v's.
template <int TYPE, int VEC, int ITEMS, int U, bool INSIDE, bool CACHE>
__global__ __launch_bounds__(NTH) void rotary_fwd_kernel(const RotDesc d, int lph, int npg) {
  typedef typename Elem<TYPE>::t E;
  const int lane = threadIdx.x & 63, hl = lane / lph, il = lane % lph, hpw = 64 / lph;
  const int heads = d.Hq + d.Hk + (CACHE ? d.Hk : 0);
  int ca[ITEMS], cb[ITEMS];
  double f[ITEMS][VEC];
  float wa[2][ITEMS][VEC], wb[2][ITEMS][VEC];
#pragma unroll
  for (int it = 0; it < ITEMS; ++it) {
    item_chunks<VEC>(il + it * lph, d.D, d.R, d.inter, ca[it], cb[it]);
    pair_freqs<VEC, INSIDE>(d, ca[it], cb[it], il + it * lph, f[it]);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const void* w = j ? d.wk : d.wq;
        wa[j][it][i] = w && ca[it] >= 0 ? load_w(w, d.wtype, ca[it] + i) : 1.f;
        wb[j][it][i] = w && cb[it] >= 0 ? load_w(w, d.wtype, cb[it] + i) : 1.f;
      }
    }
  }
  const float inv_d = 1.f / d.D;
  const long long units = d.T * npg, nw = (long long)gridDim.x * (NTH / 64);
  for (long long u = (long long)blockIdx.x * (NTH / 64) + (threadIdx.x >> 6); u < units; u += nw) {
    const long long t = u / npg;
    const int h0 = (int)(u % npg) * U * hpw + hl;
    float a[U][ITEMS][VEC], b[U][ITEMS][VEC];
#pragma unroll
    for (int p = 0; p < U; ++p) {
      const int h = h0 + p * hpw;
      const E* x = h < d.Hq ? (const E*)d.q + t * d.q_ts + h * d.q_hs
                   : h < d.Hq + d.Hk ? (const E*)d.k + t * d.k_ts + (h - d.Hq) * d.k_hs
                                     : (const E*)d.v + t * d.v_ts + (h - d.Hq - d.Hk) * d.v_hs;
#pragma unroll
      for (int it = 0; it < ITEMS; ++it) {
        load<E, VEC>(x + ca[it], (const E*)d.q, h < heads && ca[it] >= 0, a[p][it]);
        load<E, VEC>(x + cb[it], (const E*)d.q, h < heads && cb[it] >= 0, b[p][it]);
      }
    }
    const long long slot = CACHE ? d.slots[t] : 0;
    const bool live = CACHE && slot >= 0 && slot < d.nslots;
    const long long page = CACHE ? slot / d.page : 0;
    const int off = CACHE ? (int)(slot % d.page) : 0;
    float c[ITEMS][VEC], s[ITEMS][VEC];
#pragma unroll
    for (int it = 0; it < ITEMS; ++it) angles<VEC>(f[it], (double)d.pos[t], d.mscale, 1.f, c[it], s[it]);
#pragma unroll
    for (int p = 0; p < U; ++p) {
      const int h = h0 + p * hpw;
      const bool isq = h < d.Hq;
      if (CACHE && h >= d.Hq + d.Hk) {             // a value head: as it is, into its column of eight tokens
        if (h < heads && live) {
          E* o = (E*)d.vo + ((page * d.Hk + (h - d.Hq - d.Hk)) * (d.page / 8) + off / 8) * 8LL * d.D + off % 8;
#pragma unroll
          for (int it = 0; it < ITEMS; ++it) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
              if (ca[it] >= 0) from_f(a[p][it][i], o[(ca[it] + i) * 8LL]);
              if (cb[it] >= 0) from_f(b[p][it][i], o[(cb[it] + i) * 8LL]);
            }
          }
        }
        continue;
      }
      if (isq ? d.wq != nullptr : d.wk != nullptr) {
        float ss = 0.f;
#pragma unroll
        for (int it = 0; it < ITEMS; ++it)
#pragma unroll
          for (int i = 0; i < VEC; ++i) ss += a[p][it][i] * a[p][it][i] + b[p][it][i] * b[p][it][i];
        ss = sum_lanes(ss, lph);
        const float r = rsqrtf(ss * inv_d + d.eps);
#pragma unroll
        for (int it = 0; it < ITEMS; ++it)
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            a[p][it][i] *= r * (isq ? wa[0][it][i] : wa[1][it][i]);
            b[p][it][i] *= r * (isq ? wb[0][it][i] : wb[1][it][i]);
          }
      }
      if (h >= heads) continue;
      E* o;
      if (isq) o = (E*)d.qo + (t * d.Hq + h) * d.D;
      else if (CACHE) o = (E*)d.ko + ((page * d.Hk + (h - d.Hq)) * d.page + off) * d.D;
      else o = (E*)d.ko + (t * d.Hk + (h - d.Hq)) * d.D;
      if (CACHE && !isq && !live) continue;
#pragma unroll
      for (int it = 0; it < ITEMS; ++it) {
        turn<VEC, INSIDE>(a[p][it], b[p][it], c[it], s[it]);
        if (ca[it] >= 0) store<E, VEC>(o + ca[it], a[p][it]);
        if (cb[it] >= 0) store<E, VEC>(o + cb[it], b[p][it]);
      }
    }
  }
}

// ---- backward: as the forward, gradients in place of inputs; x is read again where it was normed. NORM: either of q
// and k has a weight. Weight gradients: each lane sums its own elements over its units in 32 bits, a block adds its
// lanes and waves in a fixed order into part[block], rotary_fold_kernel the blocks: no atomics, the same bits each run.
template <int TYPE, int VEC, int ITEMS, int U, bool INSIDE, bool NORM>
__global__ __launch_bounds__(NTH) void rotary_bwd_kernel(const RotDesc d, int lph, int npg) {
  typedef typename Elem<TYPE>::t E;
  const int lane = threadIdx.x & 63, hl = lane / lph, il = lane % lph, hpw = 64 / lph;
  const int heads = d.Hq + d.Hk;
  int ca[ITEMS], cb[ITEMS];
  double f[ITEMS][VEC];
  float wa[2][ITEMS][VEC], wb[2][ITEMS][VEC], da[2][ITEMS][VEC], db[2][ITEMS][VEC];
#pragma unroll
  for (int it = 0; it < ITEMS; ++it) {
    item_chunks<VEC>(il + it * lph, d.D, d.R, d.inter, ca[it], cb[it]);
    pair_freqs<VEC, INSIDE>(d, ca[it], cb[it], il + it * lph, f[it]);
    if (NORM) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const void* w = j ? d.wk : d.wq;
          wa[j][it][i] = w && ca[it] >= 0 ? load_w(w, d.wtype, ca[it] + i) : 1.f;
          wb[j][it][i] = w && cb[it] >= 0 ? load_w(w, d.wtype, cb[it] + i) : 1.f;
          da[j][it][i] = db[j][it][i] = 0.f;
        }
      }
    }
  }
  const float inv_d = 1.f / d.D;
  const long long units = d.T * npg, nw = (long long)gridDim.x * (NTH / 64);
  for (long long u = (long long)blockIdx.x * (NTH / 64) + (threadIdx.x >> 6); u < units; u += nw) {
    const long long t = u / npg;
    const int h0 = (int)(u % npg) * U * hpw + hl;
    float a[U][ITEMS][VEC], b[U][ITEMS][VEC], xa[U][ITEMS][VEC], xb[U][ITEMS][VEC];
#pragma unroll
    for (int p = 0; p < U; ++p) {
      const int h = h0 + p * hpw;
      const bool isq = h < d.Hq, on = h < heads;
      const E* g = isq ? (const E*)d.gq + t * d.gq_ts + h * d.gq_hs : (const E*)d.gk + t * d.gk_ts + (h - d.Hq) * d.gk_hs;
      const E* x = isq ? (const E*)d.q + t * d.q_ts + h * d.q_hs : (const E*)d.k + t * d.k_ts + (h - d.Hq) * d.k_hs;
      const bool nrm = NORM && on && (isq ? d.wq != nullptr : d.wk != nullptr);
#pragma unroll
      for (int it = 0; it < ITEMS; ++it) {
        load<E, VEC>(g + ca[it], (const E*)d.gq, on && ca[it] >= 0, a[p][it]);
        load<E, VEC>(g + cb[it], (const E*)d.gq, on && cb[it] >= 0, b[p][it]);
        if (NORM) {
          load<E, VEC>(x + ca[it], (const E*)d.q, nrm && ca[it] >= 0, xa[p][it]);
          load<E, VEC>(x + cb[it], (const E*)d.q, nrm && cb[it] >= 0, xb[p][it]);
        }
      }
    }
    float c[ITEMS][VEC], s[ITEMS][VEC];
#pragma unroll
    for (int it = 0; it < ITEMS; ++it) angles<VEC>(f[it], (double)d.pos[t], d.mscale, -1.f, c[it], s[it]);
#pragma unroll
    for (int p = 0; p < U; ++p) {
      const int h = h0 + p * hpw;
      const bool isq = h < d.Hq, on = h < heads;
#pragma unroll
      for (int it = 0; it < ITEMS; ++it) turn<VEC, INSIDE>(a[p][it], b[p][it], c[it], s[it]);
      if (NORM) {
        const bool nrm = on && (isq ? d.wq != nullptr : d.wk != nullptr);
        float ss = 0.f;
#pragma unroll
        for (int it = 0; it < ITEMS; ++it)
#pragma unroll
          for (int i = 0; i < VEC; ++i) ss += xa[p][it][i] * xa[p][it][i] + xb[p][it][i] * xb[p][it][i];
        ss = sum_lanes(ss, lph);
        const float r = nrm ? rsqrtf(ss * inv_d + d.eps) : 0.f;
        float hu = 0.f;
#pragma unroll
        for (int it = 0; it < ITEMS; ++it)
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            xa[p][it][i] *= r;                        // u
            xb[p][it][i] *= r;
            const float ga = a[p][it][i] * xa[p][it][i], gb = b[p][it][i] * xb[p][it][i];   // 0 without a norm
            da[0][it][i] += isq ? ga : 0.f;
            da[1][it][i] += isq ? 0.f : ga;
            db[0][it][i] += isq ? gb : 0.f;
            db[1][it][i] += isq ? 0.f : gb;
            const float va = isq ? wa[0][it][i] : wa[1][it][i], vb = isq ? wb[0][it][i] : wb[1][it][i];
            hu += ga * va + gb * vb;
            a[p][it][i] *= va;                        // h
            b[p][it][i] *= vb;
          }
        hu = sum_lanes(hu, lph) * inv_d;
        const float rr = nrm ? r : 1.f;
#pragma unroll
        for (int it = 0; it < ITEMS; ++it)
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            a[p][it][i] = rr * (a[p][it][i] - xa[p][it][i] * hu);
            b[p][it][i] = rr * (b[p][it][i] - xb[p][it][i] * hu);
          }
      }
      if (!on) continue;
      E* o = isq ? (E*)d.qo + (t * d.Hq + h) * d.D : (E*)d.ko + (t * d.Hk + (h - d.Hq)) * d.D;
#pragma unroll
      for (int it = 0; it < ITEMS; ++it) {
        if (ca[it] >= 0) store<E, VEC>(o + ca[it], a[p][it]);
        if (cb[it] >= 0) store<E, VEC>(o + cb[it], b[p][it]);
      }
    }
  }
  if (!NORM) return;
  __shared__ float red[NTH / 64][2][512];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
#pragma unroll
    for (int it = 0; it < ITEMS; ++it) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        float x = da[j][it][i], y = db[j][it][i];
        for (int o = lph; o < 64; o <<= 1) {
          x += __shfl_xor(x, o, 64);
          y += __shfl_xor(y, o, 64);
        }
        if (hl == 0 && ca[it] >= 0) red[threadIdx.x >> 6][j][ca[it] + i] = x;
        if (hl == 0 && cb[it] >= 0) red[threadIdx.x >> 6][j][cb[it] + i] = y;
      }
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < 2 * d.D; e += NTH) {
    const int j = e / d.D, i = e % d.D;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < NTH / 64; ++w) v += red[w][j][i];
    d.part[((long long)blockIdx.x * 2 + j) * d.D + i] = v;
  }
}

// weight gradients from the blocks' partials: 64 columns a block, 16 waves each over every 16th row
__global__ __launch_bounds__(1024) void rotary_fold_kernel(const RotDesc d, int nblocks) {
  __shared__ float red[16][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, e = blockIdx.x * 64 + lane;
  float v = 0.f;
  if (e < 2 * d.D)
    for (int r = w; r < nblocks; r += 16) v += d.part[(long long)r * 2 * d.D + e];
  red[w][lane] = v;
  __syncthreads();
  if (w != 0 || e >= 2 * d.D) return;
  v = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) v += red[i][lane];
  void* o = e < d.D ? d.dwq : d.dwk;
  const int i = e < d.D ? e : e - d.D;
  if (!o) return;
  if (d.dwtype == 0) ((float*)o)[i] = d.dwacc ? ((float*)o)[i] + v : v;
  else if (d.dwtype == 1) ((bf16_t*)o)[i] = f2bf(v);
  else ((__half*)o)[i] = __float2half(v);
}

bool aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }

// whether every access can take 16 bytes, and the layout's pairs fall into whole chunks
bool vec_ok(const RotDesc& d, int vec, bool bwd) {
  if (d.D % vec || d.R % (d.inter ? vec : 2 * vec)) return false;
  if (((d.q_ts | d.q_hs | d.k_ts | d.k_hs) % vec) || !aligned(d.q) || !aligned(d.k) || !aligned(d.qo) || !aligned(d.ko))
    return false;
  if (d.slots && (((d.v_ts | d.v_hs) % vec) || !aligned(d.v))) return false;
  if (bwd && (((d.gq_ts | d.gq_hs | d.gk_ts | d.gk_hs) % vec) || !aligned(d.gq) || !aligned(d.gk))) return false;
  return true;
}

int items_of(const RotDesc& d, int vec) {
  if (vec > 1 && d.inter) return (d.D / vec + 1) / 2;
  return d.R / (2 * vec) + ((d.D - d.R) / vec + 1) / 2;
}

int pow2_at_least(int n) {
  int p = 1;
  while (p < n) p <<= 1;
  return p;
}

constexpr int FWD_BLOCKS = 2048, BWD_BLOCKS = 1024;   // the backward's count also sizes its partials

template <int TYPE, int VEC, int ITEMS, int U, bool INSIDE>
int launch(const RotDesc& d, bool bwd, int lph, hipStream_t st) {
  const int heads = d.Hq + d.Hk + (d.slots ? d.Hk : 0), per = (64 / lph) * U, npg = (heads + per - 1) / per;
  const long long blocks = (d.T * npg + 3) / 4;
  if (!bwd) {
    const int grid = (int)(blocks < FWD_BLOCKS ? blocks : FWD_BLOCKS);
    if (d.slots)
      hipLaunchKernelGGL((rotary_fwd_kernel<TYPE, VEC, ITEMS, U, INSIDE, true>), dim3(grid), dim3(NTH), 0, st, d, lph, npg);
    else
      hipLaunchKernelGGL((rotary_fwd_kernel<TYPE, VEC, ITEMS, U, INSIDE, false>), dim3(grid), dim3(NTH), 0, st, d, lph, npg);
    return (int)hipGetLastError();
  }
  const int grid = (int)(blocks < BWD_BLOCKS ? blocks : BWD_BLOCKS);
  if (d.wq || d.wk) {
    hipLaunchKernelGGL((rotary_bwd_kernel<TYPE, VEC, ITEMS, U, INSIDE, true>), dim3(grid), dim3(NTH), 0, st, d, lph, npg);
    const int rc = (int)hipGetLastError();
    if (rc) return rc;
    hipLaunchKernelGGL(rotary_fold_kernel, dim3((2 * d.D + 63) / 64), dim3(1024), 0, st, d, grid);
  } else {
    hipLaunchKernelGGL((rotary_bwd_kernel<TYPE, VEC, ITEMS, U, INSIDE, false>), dim3(grid), dim3(NTH), 0, st, d, lph, npg);
  }
  return (int)hipGetLastError();
}

template <int TYPE>
int dispatch(const RotDesc& d, bool bwd, hipStream_t st) {
  constexpr int V = Elem<TYPE>::VEC;
  if (vec_ok(d, V, bwd)) {
    const int lph = pow2_at_least(items_of(d, V));
    return d.inter ? launch<TYPE, V, 1, 2, true>(d, bwd, lph, st) : launch<TYPE, V, 1, 2, false>(d, bwd, lph, st);
  }
  const int n = items_of(d, 1);
  if (n <= 64) return launch<TYPE, 1, 1, 1, false>(d, bwd, pow2_at_least(n), st);
  return launch<TYPE, 1, 4, 1, false>(d, bwd, 64, st);
}

int run(const RotDesc* d, bool bwd, hipStream_t st) {
  if (!d || d->T < 0 || d->Hq < 1 || d->Hk < 1 || d->D < 1 || d->D > 512 || d->R < 0 || d->R > d->D ||
      d->R % 2)
    return -1;
  if (d->slots && (d->page < 8 || d->page % 8 || d->nslots < 0)) return -2;
  if (d->T == 0) {                         // no tokens: the weight gradients are zero
    if (!bwd || !(d->wq || d->wk)) return 0;
    hipLaunchKernelGGL(rotary_fold_kernel, dim3((2 * d->D + 63) / 64), dim3(1024), 0, st, *d, 0);
    return (int)hipGetLastError();
  }
  switch (d->dtype) {
    case 0: return dispatch<0>(*d, bwd, st);
    case 1: return dispatch<1>(*d, bwd, st);
    case 2: return dispatch<2>(*d, bwd, st);
  }
  return -3;
}
}  // namespace

OBST_API int obst_rotary_fwd(const RotDesc* d, hipStream_t st) { return run(d, false, st); }
OBST_API int obst_rotary_bwd(const RotDesc* d, hipStream_t st) { return run(d, true, st); }
// floats of RotDesc.part
OBST_API long long obst_rotary_part(int D) { return 2LL * BWD_BLOCKS * D; }
