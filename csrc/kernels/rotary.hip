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
// product is off by 10^-2 radians, this one by three roundings of 2^-53 of the turns made, 2e-15 radians a turn: less
// than a rounding of 32 bits up to 3e7 turns (position 1.8e8 of a pair of frequency 1). sin and cos then see an argument
// within half a turn.
//
// A head's elements are cut into items of two chunks of VEC elements (16 bytes): one lane holds both members of its
// pairs, so the rotation needs no exchange between lanes. LPH lanes hold a head, a wave 64 / LPH heads of one token.
// VEC = 1 takes what 16-byte accesses cannot (odd head widths, strides or addresses).
//
// Bound by memory: every element is read once and written once. At 32768 tokens of 2 x 16 heads x 128 in bf16, normed:
// forward 88 us (537 MB, 6.1 TB/s), backward 141 us (805 MB, 5.7 TB/s) and 4 us for the weight sums.
#include <hip/hip_fp16.h>
#include "common.h"

struct RotDesc {
  const void *q, *k, *v, *gq, *gk;      // inputs [T, H, D] (strides below); output gradients (backward)
  void *qo, *ko, *vo;                   // outputs, contiguous [T, H, D]; ko / vo: the caches when slots is set
  const void *wq, *wk;                  // norm weights [D] or null
  const double* freqs;                  // [R / 2]
  const long long* pos;                 // [T]; null: nothing turns
  const int* slots;                     // [T] or null
  float* part;                          // backward: weight-gradient partials [blocks][D]
  void *dwq, *dwk;                      // backward: weight gradients
  long long q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, gq_ts, gq_hs, gk_ts, gk_hs;   // token / head strides, in elements
  long long T, nslots;
  int Hq, Hk, D, R, inter, dtype, wtype, dwtype, dwacc, page;   // types: 0 fp32, 1 bf16, 2 fp16
  float mscale, eps;
};
static_assert(sizeof(RotDesc) == 272);    // as ops/_lib.py packs it

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

typedef __attribute__((ext_vector_type(4))) uint32_t u32x4_t;

template <typename E, int VEC>
struct alignas(sizeof(E) * VEC < 16 ? sizeof(E) * VEC : 16) Chunk { E e[VEC]; };

template <bool LINES, typename E, int VEC>
__device__ __forceinline__ void store(E* p, const float* f) {
  Chunk<E, VEC> c;
#pragma unroll
  for (int i = 0; i < VEC; ++i) from_f(f[i], c.e[i]);
  if constexpr (LINES) __builtin_nontemporal_store(__builtin_bit_cast(u32x4_t, c), reinterpret_cast<u32x4_t*>(p));
  else *reinterpret_cast<Chunk<E, VEC>*>(p) = c;
}

// LINES, in the normed backward: chunks go past the caches where a head's lanes together take whole 128-byte lines
// (bf16 x 128: 165 -> 146 us for the loads, 141 with the stores). Where they take parts of lines, the caches hold the
// rest for the other half's access (fp32 x 96, half a head 1.5 lines: 26 us, 30 past the caches). The forward, at 6
// TB/s, gains nothing from loads and loses 10 % with stores past the caches.
template <bool LINES, typename E, int VEC>
__device__ __forceinline__ Chunk<E, VEC> load_once(const E* p) {
  if constexpr (LINES) {
    return __builtin_bit_cast(Chunk<E, VEC>, __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(p)));
  }
  return *reinterpret_cast<const Chunk<E, VEC>*>(p);
}

// the compiler no longer knows what a loaded chunk holds: what it derived from it is not kept
template <typename E, int VEC>
__device__ __forceinline__ void forget(Chunk<E, VEC>& c) {
  if constexpr (sizeof(Chunk<E, VEC>) == 16) {
    uint4 x = __builtin_bit_cast(uint4, c);
    asm volatile("" : "+v"(x.x), "+v"(x.y), "+v"(x.z), "+v"(x.w));
    c = __builtin_bit_cast(Chunk<E, VEC>, x);
  }
}

__device__ __forceinline__ float load_w(const void* w, int type, int i) {
  if (type == 0) return ((const float*)w)[i];
  return type == 1 ? bf2f(((const bf16_t*)w)[i]) : __half2float(((const __half*)w)[i]);
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

// the pairs of a lane's two chunks: (a[i], b[i]), or inside each chunk. Chunks that do not turn (ta, tb) stay as they
// are, whatever their neighbours hold
template <int VEC, bool INSIDE>
__device__ __forceinline__ void turn(float* a, float* b, const float* c, const float* s, bool ta, bool tb) {
  if (INSIDE) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float* v = j ? b : a;
      if (j ? tb : ta) {
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) {
          const float x = v[2 * i], y = v[2 * i + 1], cc = c[j * (VEC / 2) + i], ss = s[j * (VEC / 2) + i];
          v[2 * i] = x * cc - y * ss;
          v[2 * i + 1] = y * cc + x * ss;
        }
      }
    }
  } else if (ta) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float x = a[i], y = b[i];
      a[i] = x * c[i] - y * s[i];
      b[i] = y * c[i] + x * s[i];
    }
  }
}

// One lane's share of a head: its items' chunks, which of them exist, and where their pairs' cos and sin lie in Staged
template <int VEC, int ITEMS, bool INSIDE>
struct Lane {
  int ca[ITEMS], cb[ITEMS];              // first elements, 0 where there is no such chunk
  bool ha[ITEMS], hb[ITEMS], ta[ITEMS], tb[ITEMS];
  int fa[ITEMS], fb[ITEMS];              // first pair (INSIDE: of each chunk), 0 where the chunk does not turn

  __device__ __forceinline__ Lane(const RotDesc& d, int il, int lph) {
#pragma unroll
    for (int it = 0; it < ITEMS; ++it) {
      int a, b;
      item_chunks<VEC>(il + it * lph, d.D, d.R, d.inter, a, b);
      ha[it] = a >= 0;
      hb[it] = b >= 0;
      ca[it] = max(a, 0);
      cb[it] = max(b, 0);
      ta[it] = ha[it] && a < d.R;
      tb[it] = hb[it] && b < d.R;
      fa[it] = !ta[it] ? 0 : INSIDE ? a / 2 : VEC == 1 ? il + it * lph : a;
      fb[it] = tb[it] ? b / 2 : 0;
    }
  }
};

// Shared memory of a block: norm weights (fp32), frequencies (turns per position), and each wave's cos and sin of the
// pairs of its token, times mscale
struct Staged {
  float w[2][512];
  double f[256];
  float c[NTH / 64][256], s[NTH / 64][256];
};

// an offset of 0 that the compiler cannot see through: reads of Staged at it stay where they are written. Hoisted out
// of the loops, as it would have them, they hold 32 to 48 registers a lane and spill
__device__ __forceinline__ int here() {
  int z = 0;
  asm volatile("" : "+s"(z));
  return z;
}

__device__ __forceinline__ void stage(const RotDesc& d, Staged& s) {
  for (int i = threadIdx.x; i < d.D; i += NTH) {
    if (d.wq) s.w[0][i] = load_w(d.wq, d.wtype, i);
    if (d.wk) s.w[1][i] = load_w(d.wk, d.wtype, i);
  }
  if ((int)threadIdx.x < d.R / 2) s.f[threadIdx.x] = d.freqs[threadIdx.x] * 0.15915494309189535;
  __syncthreads();
}

// cos and sin of pos * f turns, times m and (sin) sign. The angle is reduced in 64 bits to a quarter turn r in [-1/2,
// 1/2] and its quadrant; there the Taylor polynomials of sin and cos(pi r / 2) to the 9th and 10th power are off by
// less than 2^-28
__device__ __forceinline__ void turn_of(double pos, double f, float m, float sign, float& c, float& s) {
  double t = pos * f;
  t = 4.0 * (t - rint(t));
  const double k = rint(t);
  const float r = (float)(t - k), r2 = r * r;
  const int q = (int)k;
  const float sn = r * (1.5707963267948966f + r2 * (-0.6459640975062462f + r2 * (0.07969262624616704f +
                   r2 * (-0.004681754135318688f + r2 * 0.00016044118478735982f))));
  const float cs = 1.f + r2 * (-1.2337005501361697f + r2 * (0.2536695079010480f + r2 * (-0.02086348076335296f +
                   r2 * (0.0009192602748394266f + r2 * -2.5202042373060605e-05f))));
  const float u = q & 1 ? cs : sn, v = q & 1 ? sn : cs;
  c = m * (q + 1 & 2 ? -v : v);
  s = m * sign * (q & 2 ? -u : u);
}

// those of a token, a pair a lane, through shared memory for all of the wave's heads (each lane forming those of its
// own pairs, eight times over in a wave of eight heads, took half of the forward's instructions)
__device__ __forceinline__ void turn_angles(const RotDesc& d, Staged& sh, int w, double pos, float sign) {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");      // the wave's reads of its last token's are done
  for (int i = threadIdx.x & 63; i < d.R / 2; i += 64) turn_of(pos, sh.f[i], d.mscale, sign, sh.c[w][i], sh.s[w][i]);
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}

// a lane's VEC pairs of them
template <int VEC, bool INSIDE>
__device__ __forceinline__ void read_angles(const float* t, int fa, int fb, float* o) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) o[i] = INSIDE && i >= VEC / 2 ? t[fb + i - VEC / 2] : t[fa + i];
}

template <int CTRL>
__device__ __forceinline__ float dpp_mov(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, false));
}
// sum over the lph (a power of two) lanes of a head; every lane of the wave takes part
__device__ __forceinline__ float sum_lanes(float v, int lph) {
  if (lph > 1) v += dpp_mov<0xB1>(v);    // lane ^ 1
  if (lph > 2) v += dpp_mov<0x4E>(v);    // lane ^ 2
  if (lph > 4) v += dpp_mov<0x141>(v);   // the other four of eight
  if (lph > 8) v += dpp_mov<0x140>(v);   // the other eight of sixteen
  if (lph > 16) v += __shfl_xor(v, 16, 64);
  if (lph > 32) v += __shfl_xor(v, 32, 64);
  return v;
}

// those of one lane's pairs, for rows of several tokens in a wave
template <int VEC, bool INSIDE>
__device__ __forceinline__ void own_angles(const double* f, int fa, int fb, double pos, float m, float sign, float* c,
                                           float* s) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    turn_of(pos, f[INSIDE && i >= VEC / 2 ? fb + i - VEC / 2 : fa + i], m, sign, c[i], s[i]);
  }
}

// Which row a lane has in a pass. Passes run over the heads of q, then of k: of one token, or (ROWS) over all (token,
// head) pairs of the call, where a token's heads leave most of a wave's lanes without one.
struct Row {
  long long t;
  int h;
  bool on;
};

template <bool ROWS>
__device__ __forceinline__ Row row_of(const RotDesc& d, long long t, int p, int hl, int hpw, int H) {
  if (!ROWS) {
    const int h = p * hpw + hl;
    return {t, min(h, H - 1), h < H};
  }
  const unsigned n = (unsigned)d.T * H, r = (unsigned)p * hpw + hl, c = min(r, n - 1);    // T H < 2^31
  return {c / H, (int)(c % H), r < n};
}

// Values into their columns of eight tokens: V cache [P][Hk][page / 8][D][8]. A wave takes a window of wt
// neighbouring tokens (8, or 1 where there are few) and VCH pieces of 64 * EV elements of their heads. Eight tokens
// of the step that fill one column block, slots 8 j .. 8 j + 7, are written together, 16 bytes at a time, by the
// window that holds the first of them. Tokens outside such a run (a decode step's, a run's ragged ends) write their
// elements one by one. (A window a token, with the other seven of a run idle, left all of a prompt's work to every
// eighth block, which is one of the eight dies: 127 us where windows of eight take 46, 5.9 TB/s, at 16384 tokens of
// 16 heads x 128.)
constexpr int VCH = 4;

template <typename E, int EV>
__device__ __forceinline__ void append_run(const RotDesc& d, long long t, int slot, int e0) {
  const long long page = slot / d.page;
  const int o8 = slot % d.page / 8, n = d.Hk * d.D;
  const E* v = (const E*)d.v + t * d.v_ts;
#pragma unroll 2
  for (int i = 0; i < VCH; ++i) {
    const int e = e0 + i * 64 * EV;
    if (e >= n) return;
    const int h = e / d.D, c = e % d.D;
    Chunk<E, EV> x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = *reinterpret_cast<const Chunk<E, EV>*>(v + j * d.v_ts + h * d.v_hs + c);
    E* o = (E*)d.vo + (((page * d.Hk + h) * (d.page / 8) + o8) * d.D + c) * 8;
#pragma unroll
    for (int k = 0; k < EV; ++k) {
      Chunk<E, 8> y;
#pragma unroll
      for (int j = 0; j < 8; ++j) y.e[j] = x[j].e[k];
      *reinterpret_cast<Chunk<E, 8>*>(o + 8 * k) = y;
    }
  }
}

template <typename E, int EV>
__device__ __forceinline__ void append_one(const RotDesc& d, long long t, int slot, int e0) {
  const long long page = slot / d.page;
  const int off = slot % 8, o8 = slot % d.page / 8, n = d.Hk * d.D;
  const E* v = (const E*)d.v + t * d.v_ts;
  Chunk<E, EV> x[VCH];
#pragma unroll
  for (int i = 0; i < VCH; ++i) {
    const int e = min(e0 + i * 64 * EV, n - EV);
    x[i] = *reinterpret_cast<const Chunk<E, EV>*>(v + e / d.D * d.v_hs + e % d.D);
  }
#pragma unroll
  for (int i = 0; i < VCH; ++i) {
    const int e = e0 + i * 64 * EV;
    if (e >= n) return;
    E* o = (E*)d.vo + (((page * d.Hk + e / d.D) * (d.page / 8) + o8) * d.D + e % d.D) * 8 + off;
#pragma unroll
    for (int k = 0; k < EV; ++k) o[8 * k] = x[i].e[k];
  }
}

template <typename E, int EV>
__device__ __forceinline__ void append_values(const RotDesc& d, long long unit, int nvg, int wt) {
  const int lane = threadIdx.x & 63, e0 = (int)(unit % nvg) * VCH * 64 * EV + lane * EV;
  const long long t0 = unit / nvg * wt;
  // lane i holds the slot of token t0 - 7 + i, -2 where there is none
  const long long at = t0 - 7 + lane;
  const int raw = d.slots[min(max(at, 0LL), d.T - 1)];
  const int slot = at >= 0 && at < d.T && raw >= 0 && raw < d.nslots ? raw : -2;
  // bit i: the token of lane i follows its neighbour's slot; it is the first of a whole run
  const unsigned long long next = __ballot(slot >= 0 && slot == __shfl_up(slot, 1, 64) + 1 && lane > 0);
  const unsigned long long first =
      __ballot(slot >= 0 && slot % 8 == 0 && lane < 15 && (next >> (lane + 1) & 0x7f) == 0x7f);
  for (int i = 7; i < 7 + wt; ++i) {
    const int s = __builtin_amdgcn_readlane(slot, i);
    if (s < 0) continue;
    if (first >> i & 1) append_run<E, EV>(d, t0 - 7 + i, s, e0);
    else if ((first >> (i - 7) & 0xff) == 0) append_one<E, EV>(d, t0 - 7 + i, s, e0);   // in no run
  }
}

// ---- forward. A wave's unit is U passes, of one token or (ROWS) of the call; a pass is 64 / lph heads, all of q or
// all of k. CACHE: k goes into the pages, and the blocks behind the first `rot` write the values.
template <int TYPE, int VEC, int ITEMS, int U, bool INSIDE, bool ROWS, bool CACHE, int EV>
__global__ __launch_bounds__(NTH, 4) void rotary_fwd_kernel(const RotDesc d, int lph, int pq, int pk, int rot,
                                                            int nvg, int wt) {
  typedef typename Elem<TYPE>::t E;
  __shared__ Staged sh;
  if (CACHE && (int)blockIdx.x >= rot) {
    const long long units = (d.T + wt - 1) / wt * nvg, nw = (long long)(gridDim.x - rot) * (NTH / 64);
    for (long long u = (long long)(blockIdx.x - rot) * (NTH / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
         u < units; u += nw)
      append_values<E, EV>(d, u, nvg, wt);
    return;
  }
  const int lane = threadIdx.x & 63, hl = lane / lph, il = lane % lph, hpw = 64 / lph;
  const int np = pq + pk, npg = (np + U - 1) / U;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Lane<VEC, ITEMS, INSIDE> ln(d, il, lph);
  stage(d, sh);
  const float inv_d = 1.f / d.D;
  const long long units = ROWS ? npg : d.T * npg, nw = (long long)rot * (NTH / 64);
  for (long long u = (long long)blockIdx.x * (NTH / 64) + wave; u < units; u += nw) {
    const long long t = ROWS ? 0 : u / npg;
    const int p0 = (int)(ROWS ? u : u % npg) * U;
    Chunk<E, VEC> xa[U][ITEMS], xb[U][ITEMS];
    Row row[U];
#pragma unroll
    for (int p = 0; p < U; ++p) {
      if (p0 + p >= np) break;
      const bool isq = p0 + p < pq;
      row[p] = row_of<ROWS>(d, t, p0 + p - (isq ? 0 : pq), hl, hpw, isq ? d.Hq : d.Hk);
      const long long rt = row[p].t;
      const int h = row[p].h;
      const E* x = isq ? (const E*)d.q + rt * d.q_ts + h * d.q_hs : (const E*)d.k + rt * d.k_ts + h * d.k_hs;
#pragma unroll
      for (int it = 0; it < ITEMS; ++it) {
        xa[p][it] = *reinterpret_cast<const Chunk<E, VEC>*>(x + ln.ca[it]);
        xb[p][it] = *reinterpret_cast<const Chunk<E, VEC>*>(x + ln.cb[it]);
      }
    }
    const bool still = CACHE && !d.pos;                // nothing turns
    if (!ROWS) turn_angles(d, sh, wave, still ? 0.0 : (double)d.pos[t], 1.f);
#pragma unroll
    for (int p = 0; p < U; ++p) {
      if (p0 + p >= np) break;
      const bool isq = p0 + p < pq;
      const long long rt = row[p].t;
      const int h = row[p].h;
      const int slot = CACHE && !isq ? d.slots[rt] : 0;
      const double pos = ROWS && !still ? (double)d.pos[rt] : 0.0;
      float a[ITEMS][VEC], b[ITEMS][VEC];
#pragma unroll
      for (int it = 0; it < ITEMS; ++it)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          a[it][i] = to_f(xa[p][it].e[i]);
          b[it][i] = to_f(xb[p][it].e[i]);
        }
      if (isq ? d.wq != nullptr : d.wk != nullptr) {
        const float* w = sh.w[isq ? 0 : 1] + here();
        float ss = 0.f;
#pragma unroll
        for (int it = 0; it < ITEMS; ++it) {
          float sa = 0.f, sb = 0.f;
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            sa += a[it][i] * a[it][i];
            sb += b[it][i] * b[it][i];
          }
          ss += (ln.ha[it] ? sa : 0.f) + (ln.hb[it] ? sb : 0.f);
        }
        const float r = rsqrtf(sum_lanes(ss, lph) * inv_d + d.eps);
#pragma unroll
        for (int it = 0; it < ITEMS; ++it)
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            a[it][i] *= r * w[ln.ca[it] + i];
            b[it][i] *= r * w[ln.cb[it] + i];
          }
      }
      if (!row[p].on || slot < 0 || (CACHE && slot >= d.nslots)) continue;
      E* o;
      if (isq) o = (E*)d.qo + (rt * d.Hq + h) * d.D;
      else if (CACHE) o = (E*)d.ko + (((long long)(slot / d.page) * d.Hk + h) * d.page + slot % d.page) * d.D;
      else o = (E*)d.ko + (rt * d.Hk + h) * d.D;
#pragma unroll
      for (int it = 0; it < ITEMS; ++it) {
        float c[VEC], s[VEC];
        const int z = here();
        if (ROWS) {
          own_angles<VEC, INSIDE>(sh.f + z, ln.fa[it], ln.fb[it], pos, d.mscale, 1.f, c, s);
        } else {
          read_angles<VEC, INSIDE>(sh.c[wave] + z, ln.fa[it], ln.fb[it], c);
          read_angles<VEC, INSIDE>(sh.s[wave] + z, ln.fa[it], ln.fb[it], s);
        }
        turn<VEC, INSIDE>(a[it], b[it], c, s, ln.ta[it], ln.tb[it]);
        if (ln.ha[it]) store<false, E, VEC>(o + ln.ca[it], a[it]);
        if (ln.hb[it]) store<false, E, VEC>(o + ln.cb[it], b[it]);
      }
    }
  }
}

// ---- backward: as the forward, gradients in place of inputs; x is read again where it was normed. NORM: either of q
// and k has a weight. Weight gradients: each lane sums its own elements over its units in 32 bits, a block adds its
// lanes and waves in a fixed order into part[block], rotary_fold_kernel the blocks: no atomics, the same bits each run.
// With sums to keep, a block works on one tensor (the first nbq on q): sums for both took 16 more registers a lane and
// spilled.
template <int TYPE, int VEC, int ITEMS, int U, bool INSIDE, bool ROWS, bool NORM, bool LINES>
__global__ __launch_bounds__(NTH, 4) void rotary_bwd_kernel(const RotDesc d, int lph, int pq, int pk, int nbq) {
  typedef typename Elem<TYPE>::t E;
  __shared__ Staged sh;
  const int lane = threadIdx.x & 63, hl = lane / lph, il = lane % lph, hpw = 64 / lph;
  const bool block_q = (int)blockIdx.x < nbq;
  const int pb = NORM && !block_q ? pq : 0, np = !NORM ? pq + pk : block_q ? pq : pk, npg = (np + U - 1) / U;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Lane<VEC, ITEMS, INSIDE> ln(d, il, lph);
  stage(d, sh);
  float da[ITEMS][VEC], db[ITEMS][VEC];
#pragma unroll
    for (int it = 0; it < ITEMS; ++it)
#pragma unroll
      for (int i = 0; i < VEC; ++i) da[it][i] = db[it][i] = 0.f;
  const float inv_d = 1.f / d.D;
  const int b0 = NORM && !block_q ? nbq : 0, nb = !NORM ? gridDim.x : block_q ? nbq : gridDim.x - nbq;
  const long long units = ROWS ? npg : d.T * npg, nw = (long long)nb * (NTH / 64);
  for (long long u = (long long)(blockIdx.x - b0) * (NTH / 64) + wave; u < units; u += nw) {
    const long long t = ROWS ? 0 : u / npg;
    const int p0 = (int)(ROWS ? u : u % npg) * U;
    Row row[U];
    Chunk<E, VEC> ga[U][ITEMS], gb[U][ITEMS], xa[U][ITEMS], xb[U][ITEMS];
#pragma unroll
    for (int p = 0; p < U; ++p) {
      if (p0 + p >= np) break;
      const bool isq = NORM ? block_q : p0 + p < pq;
      row[p] = row_of<ROWS>(d, t, pb + p0 + p - (isq ? 0 : pq), hl, hpw, isq ? d.Hq : d.Hk);
      const long long rt = row[p].t;
      const int h = row[p].h;
      const E* g = isq ? (const E*)d.gq + rt * d.gq_ts + h * d.gq_hs : (const E*)d.gk + rt * d.gk_ts + h * d.gk_hs;
      const E* x = isq ? (const E*)d.q + rt * d.q_ts + h * d.q_hs : (const E*)d.k + rt * d.k_ts + h * d.k_hs;
#pragma unroll
      for (int it = 0; it < ITEMS; ++it) {
        ga[p][it] = load_once<LINES, E, VEC>(g + ln.ca[it]);
        gb[p][it] = load_once<LINES, E, VEC>(g + ln.cb[it]);
        if (NORM) {
          xa[p][it] = load_once<LINES, E, VEC>(x + ln.ca[it]);
          xb[p][it] = load_once<LINES, E, VEC>(x + ln.cb[it]);
        }
      }
    }
    if (!ROWS) turn_angles(d, sh, wave, (double)d.pos[t], -1.f);
#pragma unroll
    for (int p = 0; p < U; ++p) {
      if (p0 + p >= np) break;
      const bool isq = NORM ? block_q : p0 + p < pq;
      const long long rt = row[p].t;
      const int h = row[p].h;
      const double pos = ROWS ? (double)d.pos[rt] : 0.0;
      float a[ITEMS][VEC], b[ITEMS][VEC];
#pragma unroll
      for (int it = 0; it < ITEMS; ++it) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          a[it][i] = to_f(ga[p][it].e[i]);
          b[it][i] = to_f(gb[p][it].e[i]);
        }
        float c[VEC], s[VEC];
        const int z = here();
        if (ROWS) {
          own_angles<VEC, INSIDE>(sh.f + z, ln.fa[it], ln.fb[it], pos, d.mscale, -1.f, c, s);
        } else {
          read_angles<VEC, INSIDE>(sh.c[wave] + z, ln.fa[it], ln.fb[it], c);
          read_angles<VEC, INSIDE>(sh.s[wave] + z, ln.fa[it], ln.fb[it], s);
        }
        turn<VEC, INSIDE>(a[it], b[it], c, s, ln.ta[it], ln.tb[it]);
      }
      if (NORM && (isq ? d.wq != nullptr : d.wk != nullptr)) {
        // with p = sum x^2 and e = sum g w x:  u = x r,  dx = r g w - (e r^3 / D) x,  dw += g x r
        const float* w = sh.w[isq ? 0 : 1] + here();
        float ss = 0.f, e = 0.f;
#pragma unroll
        for (int it = 0; it < ITEMS; ++it) {
          float sa = 0.f, sb = 0.f, ea = 0.f, eb = 0.f;
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            const float ya = to_f(xa[p][it].e[i]), yb = to_f(xb[p][it].e[i]);
            sa += ya * ya;
            sb += yb * yb;
            ea += a[it][i] * w[ln.ca[it] + i] * ya;
            eb += b[it][i] * w[ln.cb[it] + i] * yb;
          }
          ss += (ln.ha[it] ? sa : 0.f) + (ln.hb[it] ? sb : 0.f);
          e += (ln.ha[it] ? ea : 0.f) + (ln.hb[it] ? eb : 0.f);
        }
        ss = sum_lanes(ss, lph);
        e = sum_lanes(e, lph);
        // lanes past the last head repeat it for their loads: nothing of theirs may reach the weight sums
        const float r = rsqrtf(ss * inv_d + d.eps), rw = row[p].on ? r : 0.f, k = e * inv_d * r * r * r;
        w = sh.w[isq ? 0 : 1] + here();
#pragma unroll
        for (int it = 0; it < ITEMS; ++it) {
          forget(xa[p][it]);                          // x is widened again rather than kept in 32 bits
          forget(xb[p][it]);
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            const float ya = to_f(xa[p][it].e[i]), yb = to_f(xb[p][it].e[i]);
            da[it][i] += a[it][i] * (ya * rw);
            db[it][i] += b[it][i] * (yb * rw);
            a[it][i] = a[it][i] * (r * w[ln.ca[it] + i]) - k * ya;
            b[it][i] = b[it][i] * (r * w[ln.cb[it] + i]) - k * yb;
          }
        }
      }
      if (!row[p].on) continue;
      E* o = isq ? (E*)d.qo + (rt * d.Hq + h) * d.D : (E*)d.ko + (rt * d.Hk + h) * d.D;
#pragma unroll
      for (int it = 0; it < ITEMS; ++it) {
        if (ln.ha[it]) store<LINES, E, VEC>(o + ln.ca[it], a[it]);
        if (ln.hb[it]) store<LINES, E, VEC>(o + ln.cb[it], b[it]);
      }
    }
  }
  if (!NORM) return;
  __shared__ float red[NTH / 64][512];
#pragma unroll
  for (int it = 0; it < ITEMS; ++it) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      float x = da[it][i], y = db[it][i];
      for (int o = lph; o < 64; o <<= 1) {
        x += __shfl_xor(x, o, 64);
        y += __shfl_xor(y, o, 64);
      }
      if (hl == 0 && ln.ha[it]) red[threadIdx.x >> 6][ln.ca[it] + i] = x;
      if (hl == 0 && ln.hb[it]) red[threadIdx.x >> 6][ln.cb[it] + i] = y;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < d.D; i += NTH) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < NTH / 64; ++w) v += red[w][i];
    d.part[(long long)blockIdx.x * d.D + i] = v;
  }
}

// weight gradients from the blocks' partials, in 64 bits (up to 1024 of them): 16 columns a block, 64 rows of it side
// by side, in a fixed order
__global__ __launch_bounds__(1024) void rotary_fold_kernel(const RotDesc d, int nbq, int nb) {
  __shared__ double red[64][17];
  const int col = threadIdx.x & 15, row = threadIdx.x >> 4, e = blockIdx.x * 16 + col;
  double s = 0.0;
  if (e < 2 * d.D) {
#pragma unroll 4
    for (int r = row + (e < d.D ? 0 : nbq); r < (e < d.D ? nbq : nb); r += 64)
      s += d.part[(long long)r * d.D + (e < d.D ? e : e - d.D)];
  }
  red[row][col] = s;
  __syncthreads();
  if (threadIdx.x >= 16 || e >= 2 * d.D) return;
  s = 0.0;
#pragma unroll
  for (int i = 0; i < 64; ++i) s += red[i][col];
  const float v = (float)s;
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

// the turned queries may take the queries' own place (a wave reads all of a row before it writes it), but no other part of
// what the call reads or writes
bool out_overlaps(const RotDesc& d) {
  const size_t e = d.dtype == 0 ? 4 : 2, row = (size_t)d.Hq * d.D, n = d.qo ? e * d.T * row : 0;
  const bool own = d.qo == d.q && (d.q_hs == d.D || d.Hq == 1) && (d.q_ts == (long long)row || d.T == 1);
  auto span = [&](long long ts, int H, long long hs) { return e * ((d.T - 1) * ts + (H - 1) * hs + d.D); };
  const size_t pool = e * (size_t)d.nslots * d.Hk * d.D;
  return (!own && overlap(d.qo, n, d.q, span(d.q_ts, d.Hq, d.q_hs))) ||
         overlap(d.qo, n, d.k, span(d.k_ts, d.Hk, d.k_hs)) || overlap(d.qo, n, d.v, span(d.v_ts, d.Hk, d.v_hs)) ||
         overlap(d.qo, n, d.ko, pool) || overlap(d.qo, n, d.vo, pool) || overlap(d.qo, n, d.pos, 8 * d.T) ||
         overlap(d.qo, n, d.slots, 4 * d.T);
}

// four blocks a CU; the backward's count also sizes its partials
constexpr int FWD_BLOCKS = 1024, BWD_BLOCKS = 1024;

// passes of a token, or (ROWS) of the call
template <bool ROWS>
struct Passes {
  int pq, pk;
  Passes(const RotDesc& d, int lph) : pq(of(d, d.Hq, 64 / lph)), pk(of(d, d.Hk, 64 / lph)) {}
  static int of(const RotDesc& d, int H, int hpw) { return (int)(((ROWS ? d.T * H : H) + hpw - 1) / hpw); }
  long long units(const RotDesc& d, int U) const { return (ROWS ? 1 : d.T) * ((pq + pk + U - 1) / U); }
  static int blocks(long long units, int most) {
    const long long b = (units + 3) / 4;
    return (int)(b < most ? b : most);
  }
};

template <int TYPE, int VEC, int ITEMS, int U, bool INSIDE, bool ROWS>
int forward(const RotDesc& d, int lph, hipStream_t st) {
  const Passes<ROWS> p(d, lph);
  const int grid = p.blocks(p.units(d, U), FWD_BLOCKS);
  if (!d.slots) {
    hipLaunchKernelGGL((rotary_fwd_kernel<TYPE, VEC, ITEMS, U, INSIDE, ROWS, false, 1>), dim3(grid), dim3(NTH), 0, st,
                       d, lph, p.pq, p.pk, grid, 0, 0);
    return (int)hipGetLastError();
  }
  constexpr int EV = VEC == 1 ? 1 : 2;                     // VEC > 1: D and the strides are even
  const int nvg = (d.Hk * d.D + VCH * 64 * EV - 1) / (VCH * 64 * EV), wt = d.T < 1024 ? 1 : 8;
  const int vgrid = p.blocks((d.T + wt - 1) / wt * nvg, FWD_BLOCKS);
  hipLaunchKernelGGL((rotary_fwd_kernel<TYPE, VEC, ITEMS, U, INSIDE, ROWS, true, EV>), dim3(grid + vgrid), dim3(NTH), 0,
                     st, d, lph, p.pq, p.pk, grid, nvg, wt);
  return (int)hipGetLastError();
}

template <int TYPE, int VEC, int ITEMS, int U, bool INSIDE, bool ROWS>
int backward(const RotDesc& d, int lph, hipStream_t st) {
  const Passes<ROWS> p(d, lph);
  const int grid = p.blocks(p.units(d, U), BWD_BLOCKS);
  hipLaunchKernelGGL((rotary_bwd_kernel<TYPE, VEC, ITEMS, U, INSIDE, ROWS, false, false>), dim3(grid), dim3(NTH), 0, st,
                     d, lph, p.pq, p.pk, 0);
  return (int)hipGetLastError();
}

template <int TYPE, int VEC, int ITEMS, bool INSIDE, bool ROWS, bool LINES>
int backward_normed(const RotDesc& d, int lph, hipStream_t st) {
  const Passes<ROWS> p(d, lph);
  // blocks for q and for k, as many as their units ask for
  const long long n = ROWS ? 1 : d.T, bq = (n * p.pq + 3) / 4, bk = (n * p.pk + 3) / 4;
  int nq = (int)bq, nk = (int)bk;
  if (bq + bk > BWD_BLOCKS) {
    nq = (int)((long long)BWD_BLOCKS * p.pq / (p.pq + p.pk));
    nq = nq < 1 ? 1 : nq > BWD_BLOCKS - 1 ? BWD_BLOCKS - 1 : nq;
    nk = BWD_BLOCKS - nq;
  }
  hipLaunchKernelGGL((rotary_bwd_kernel<TYPE, VEC, ITEMS, 1, INSIDE, ROWS, true, LINES>), dim3(nq + nk), dim3(NTH), 0, st,
                     d, lph, p.pq, p.pk, nq);
  const int rc = (int)hipGetLastError();
  if (rc) return rc;
  hipLaunchKernelGGL(rotary_fold_kernel, dim3((2 * d.D + 15) / 16), dim3(1024), 0, st, d, nq, nq + nk);
  return (int)hipGetLastError();
}

// Passes a unit. Four share one token's angles and keep four rows of loads in flight (two where the rows are several
// tokens': registers); under 1024 tokens one each spreads them over more waves. The normed backward takes one: a
// second pass' loads and the sums leave it three waves a SIMD (199 us where one pass took 164 at the time, 32768
// tokens of 2 x 16 heads x 128 in bf16).
template <int TYPE, int VEC, bool INSIDE, bool ROWS>
int by_tokens(const RotDesc& d, bool bwd, int lph, hipStream_t st) {
  constexpr int MANY = ROWS ? 2 : 4;
  const bool few = d.T < 1024;
  if (!bwd)
    return few ? forward<TYPE, VEC, 1, 1, INSIDE, ROWS>(d, lph, st)
               : forward<TYPE, VEC, 1, MANY, INSIDE, ROWS>(d, lph, st);
  if (d.wq || d.wk)
    return items_of(d, VEC) * 16 % 128 == 0 ? backward_normed<TYPE, VEC, 1, INSIDE, ROWS, true>(d, lph, st)
                                            : backward_normed<TYPE, VEC, 1, INSIDE, ROWS, false>(d, lph, st);
  return few ? backward<TYPE, VEC, 1, 1, INSIDE, ROWS>(d, lph, st)
             : backward<TYPE, VEC, 1, MANY, INSIDE, ROWS>(d, lph, st);
}

template <int TYPE, int ITEMS>
int by_element(const RotDesc& d, bool bwd, int lph, hipStream_t st) {
  if (!bwd) return forward<TYPE, 1, ITEMS, 1, false, false>(d, lph, st);
  return d.wq || d.wk ? backward_normed<TYPE, 1, ITEMS, false, false, false>(d, lph, st)
                      : backward<TYPE, 1, ITEMS, 1, false, false>(d, lph, st);
}

template <int TYPE>
int dispatch(const RotDesc& d, bool bwd, hipStream_t st) {
  constexpr int V = Elem<TYPE>::VEC;
  if (vec_ok(d, V, bwd)) {
    const int lph = pow2_at_least(items_of(d, V));
    // Rows of several tokens in a wave where one token's heads fill at most half of it. 65536 tokens normed in bf16,
    // forward + backward, rows against tokens: 1 + 1 heads x 32 17 + 19 against 52 + 99 us, 8 + 8 x 32 34 + 56
    // against 53 + 101; at 12 + 12 x 64 (three quarters of a wave), 32768 tokens, 48 + 76 against 40 + 68
    const int most = d.Hq > d.Hk ? d.Hq : d.Hk;
    if (most * lph <= 32 && d.T * most < 1LL << 31)
      return d.inter ? by_tokens<TYPE, V, true, true>(d, bwd, lph, st)
                     : by_tokens<TYPE, V, false, true>(d, bwd, lph, st);
    return d.inter ? by_tokens<TYPE, V, true, false>(d, bwd, lph, st)
                   : by_tokens<TYPE, V, false, false>(d, bwd, lph, st);
  }
  const int n = items_of(d, 1);
  return n <= 64 ? by_element<TYPE, 1>(d, bwd, pow2_at_least(n), st) : by_element<TYPE, 4>(d, bwd, 64, st);
}

int run(const RotDesc* d, bool bwd, hipStream_t st) {
  if (!d || d->T < 0 || d->Hq < (d->slots ? 0 : 1) || d->Hk < 1 || d->D < 1 || d->D > 512 || d->R < 0 || d->R > d->D ||
      d->R % 2 || (d->T > 0 && !d->pos && (d->R || !d->slots)))
    return -1;
  if (d->slots && (d->page < 8 || d->page % 8 || d->nslots < 0 || !aligned(d->vo))) return -2;
  if (d->T == 0) {                         // no tokens: the weight gradients are zero
    if (!bwd || !(d->wq || d->wk)) return 0;
    hipLaunchKernelGGL(rotary_fold_kernel, dim3((2 * d->D + 15) / 16), dim3(1024), 0, st, *d, 0, 0);
    return (int)hipGetLastError();
  }
  if (d->slots && out_overlaps(*d)) return -4;
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
OBST_API long long obst_rotary_part(int D) { return (long long)BWD_BLOCKS * D; }
