// Selective scan: a diagonal recurrence with an input-dependent step per channel,
//
//   dt' = softplus(dt + bias)  (or dt + bias);   a_tn = exp(dt'_t A_n);   h_tn = a_tn h_{t-1,n} + dt'_t u_t B_tn
//   y_t = sum_n C_tn h_tn + D u_t
//   g_tn = C_tn dy_t + r_{t+1,n},  r_tn = a_tn g_tn  (r behind the last step: the gradient of the last state);  q_tn = r_tn h_{t-1,n}
//   ddt' = sum_n A_n q_n + u sum_n g_n B_n;  du = dt' sum_n g_n B_n + D dy;  dA_n = sum_t dt' q_n;
//   dB_n = sum_channels g_n dt' u;  dC_n = sum_channels dy h_n;  dD = sum dy u;  dbias = sum ddt
//
// for every channel d (u, dt, A[d], D, bias of its own; B_t and C_t shared by all channels). Bound by the exponentials
// (one per step, channel and state; 16 a clock and SM) and, backward, by the issue of the products around them; the
// tensors themselves are read and written once.
//
// Layout: 4 states a lane, G = NP / 4 lanes a channel (NP: the states padded to 8, 16, 32 or 64), CT channels a lane, so
// that h stays in registers along time and a warp holds 32 * 4 * CT states. Time runs in tiles of 16 steps, whose
// rows a warp fetches two tiles ahead by asynchronous copies; it makes the steps (dt', dt' u) of its channels once a
// tile and reads them, and B and C as they came, from shared memory. A warp goes on by itself (no block barrier), and the
// exponentials of a few steps run ahead of the chain through h.
// Sequences with too few channels to fill the GPU are cut into segments: one launch computes every segment's state
// from zero and its total step, the next starts each segment from the combination of those before it.
// Backward: the forward pass leaves h at every tile's start; a tile's states are computed again from there into shared
// memory and walked through in reverse. Sums over channels and states are made by halving exchanges (n values over n
// lanes cost n - 1 shuffles and leave one sum in each lane). States, sums and gradients are fp32; sums over channel
// blocks, segments and sequences are made from partial sums in a fixed order (no atomics: two runs give the same bits).
// Exponentials are the hardware's (2 units in the last place) with their mean error taken out (`decay`): the gradient of A over 2048
// steps is off by 0.95e-6 of its norm, as with exact ones in fp32 (0.9e-6), which would take a third more time.
//
// Measured (bf16 rows, 16 states): a prompt of 8192 x 4096 362 us, of 6 x 777 x 1000 with 64 states (fp16, lengths drawn) 107 to 134 us; forward
// 4 x 2048 x 2048 159 us, backward 470 us. With enough warps a pass runs at 0.64 to 0.78 of the exponentials' rate; the backward
// kernel issues ~190 instructions for 8 states of a lane and step, and at two warps a scheduler is busy 54 % of the time.
#pragma once
#include "bdh_kernels.h"
#include "device_once.h"
#include "pair_math.cuh"

#include <cmath>
#include <type_traits>

namespace bdh {
namespace {

constexpr int LT = 16;                 // steps per tile
constexpr int FWD_WARPS = 2;           // independent warps of a block, forward and sweeps
constexpr int BWD_WARPS = 4;           // warps of a block that add their sums over channels up, backward
constexpr int FWD_BLOCKS = 6;          // blocks an SM that leave a thread the registers to run ahead (measured: 4 to 8 within 3 %;
                                       // left to itself the compiler takes 96 and spills: 20 % slower on few warps)
constexpr int BWD_BLOCKS = 2;
constexpr int STEP_THREADS = 128;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LOG2E_LO = 1.925963033500e-08f;      // log2(e) - LOG2E
constexpr float LN2 = 0.6931471805599453f;

struct ScanArgs {
  BdhScanDesc d;
  Lengths len;
  int tiles, per_seg, segs;            // tiles per sequence, per segment; segments
  int parts;                           // warps (forward) or blocks (backward) across the channels
  const float* seg_state;              // [B][segs][D][NP]: states of the segments from zero (forward or reverse)
  const float* seg_dt;                 // [B][segs][D]: their total steps
};

__device__ __forceinline__ void load4(const float* p, f2& x, f2& y) {
  const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(p);
  x = v.x;
  y = v.y;
}

// exp(dt A), A2 = A log2(e). The hardware's exponential 2^x is low by 0.5 to 2.6 10^-8 of itself on average (measured, by ranges of x
// between -0.3 and -10^-5), which a state that keeps its past for 1 / |x| steps adds up. EVEN, added within the product's one
// rounding, makes that -1.5 to 0.6 10^-8, nowhere further from 0 than it was. 2^0 stays 1 (it is up to 6 10^-8).
constexpr float EVEN = 1.5e-8f;
__device__ __forceinline__ f2 decay(float dt, f2 A2) { return ex2x2(fma1(dt, A2, both(EVEN))); }

// exp(-|x|), to about 2^-22 of itself: the rounding of |x| log2(e) is put back as a factor 1 + its residual ln(2).
__device__ __forceinline__ f2 exp_minus_abs(f2 x) {
  float a, b;
  unpack2(x, a, b);
  const f2 m = pack2(-fminf(fabsf(a), 120.f), -fminf(fabsf(b), 120.f));
  const f2 y = mul2(m, both(LOG2E));
  const f2 lo = fma2(m, both(LOG2E_LO), fma2(m, both(LOG2E), mul2(y, both(-1.f))));
  const f2 t = ex2x2(y);
  return fma2(t, mul2(lo, both(LN2)), t);
}

// softplus(x) = max(x, 0) + log1p(exp(-|x|)) for two steps at once. log1p(t) / t on [0, 1] is the polynomial of degree 9
// through its values at the Chebyshev nodes (the nearest singularity, t = -1, makes the error fall by 3 + 2 sqrt(2) a degree): off
// by at most 1.5e-8 of itself with its coefficients in 32 bits, so the result is off by the 32-bit rounding of the sums.
__device__ __forceinline__ f2 softplus2(f2 x) {
  constexpr float P[10] = {1.0f, -0.49999892711639404f, 0.33329710364341736f, -0.24951615929603577f, 0.1966327428817749f,
                           -0.1526966691017151f, 0.10543623566627502f, -0.056373611092567444f, 0.019542526453733444f,
                           -0.0031760570127516985f};
  const f2 t = exp_minus_abs(x);
  f2 p = both(P[9]);
#pragma unroll
  for (int i = 8; i >= 0; --i) p = fma2(p, t, both(P[i]));
  float a, b, ma, mb;
  unpack2(x, a, b);
  asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(ma) : "f"(a));
  asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(mb) : "f"(b));
  return fma2(p, t, pack2(ma, mb));
}
// its derivative, 1 / (1 + exp(-x)); the quick division is off by 2 units in the last place
__device__ __forceinline__ f2 sigmoid2(f2 x) {
  float a, b, ta, tb;
  unpack2(x, a, b);
  unpack2(exp_minus_abs(x), ta, tb);
  return pack2(__fdividef(a < 0.f ? ta : 1.f, 1.f + ta), __fdividef(b < 0.f ? tb : 1.f, 1.f + tb));
}

// Sums of v[0..NV) over the lanes that differ in the bits FIRST .. FIRST * LANES / 2 of the lane number: the number of
// values halves with every exchange while there is more than one. Leaves max(1, NV / LANES) sums; the first of them is
// that of value `at`; `once` marks one lane of those that hold the same.
template <int NV, int LANES, int FIRST>
__device__ __forceinline__ void sum_over(float (&v)[NV], int lane, int& at, bool& once) {
  at = 0;
  once = true;
  int n = NV;
#pragma unroll
  for (int o = LANES * FIRST / 2; o >= FIRST; o >>= 1) {
    const bool up = lane & o;
    if (n > 1) {
      n >>= 1;
#pragma unroll
      for (int i = 0; i < NV / 2; ++i) {
        if (i >= n) break;
        const float keep = up ? v[i + n] : v[i], send = up ? v[i] : v[i + n];
        v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
      }
      at += up ? n : 0;
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
      once = once && !up;
    }
  }
}

// A warp's part of a tile: 16 steps of CW channels; for loading and storing, lane l has the step l / 2 and the first or
// second half of the channels (and of the states of B and C).
template <typename T, int G, int CT>
struct Shape {
  static constexpr int NP = 4 * G;
  static constexpr int LANES = 32 / G;                 // channel lanes
  static constexpr int CW = LANES * CT;                // channels of a warp
  static constexpr int E = CW / 2;                     // elements of a lane
  static constexpr int V = E < 16 / static_cast<int>(sizeof(T)) ? E : 16 / static_cast<int>(sizeof(T));
  static constexpr int NV = E / V;                     // its packs
  static constexpr int NB = NP / 8;                    // packs of 4 states of B (or C) of a lane
};

template <typename T, int V, bool VEC>
__device__ __forceinline__ Pack<T, V> load_row(const T* p, int c, int D) {
  Pack<T, V> r;
  if constexpr (VEC) {
    if (c < D) r.load(p + c); else r.zero();
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) r.e[i] = c + i < D ? p[c + i] : elem_from_float<T>(0.f);
  }
  return r;
}
template <typename T, int V, bool VEC>
__device__ __forceinline__ void store_row(T* p, int c, int D, const Pack<T, V>& r) {
  if constexpr (VEC) {
    if (c < D) r.store(p + c);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (c + i < D) p[c + i] = r.e[i];
  }
}

// The rows of one tile on their way from memory (what lies behind `len` reads as 0), in registers: the bits as they were
// loaded, since taking elements out of them right behind the load would wait for it.
template <typename T, int G, int CT, bool VEC, bool DY>
struct Tile {
  using S = Shape<T, G, CT>;
  using Raw = typename Pack<T, S::V>::Raw;
  using Raw4 = typename Pack<T, 4>::Raw;
  Raw ru[S::NV], rdt[S::NV], rdy[DY ? S::NV : 1];
  Raw4 rB[S::NB], rC[S::NB];

  template <int V>
  static __device__ __forceinline__ typename Pack<T, V>::Raw fetch(const T* p, int c, int D) {
    const Pack<T, V> r = load_row<T, V, VEC>(p, c, D);
    return *reinterpret_cast<const typename Pack<T, V>::Raw*>(&r);
  }
  template <int V>
  static __device__ __forceinline__ Pack<T, V> bits(const typename Pack<T, V>::Raw& r) {
    Pack<T, V> p;
    *reinterpret_cast<typename Pack<T, V>::Raw*>(&p) = r;
    return p;
  }
  __device__ __forceinline__ void load(const BdhScanDesc& d, int b, int c0, int t0, int len) {
    const int lane = threadIdx.x & 31, t = t0 + lane / 2, c = c0 + (lane & 1) * S::E, n = (lane & 1) * (S::NP / 2);
    const bool in = t < len;
    const int D = in ? d.D : 0, N = in ? d.N : 0;
#pragma unroll
    for (int i = 0; i < S::NV; ++i) {
      ru[i] = fetch<S::V>(static_cast<const T*>(d.u) + b * d.u_sb + t * d.u_st, c + i * S::V, D);
      rdt[i] = fetch<S::V>(static_cast<const T*>(d.dt) + b * d.dt_sb + t * d.dt_st, c + i * S::V, D);
      if constexpr (DY) rdy[i] = fetch<S::V>(static_cast<const T*>(d.dy) + b * d.dy_sb + t * d.dy_st, c + i * S::V, D);
    }
#pragma unroll
    for (int i = 0; i < S::NB; ++i) {
      rB[i] = fetch<4>(static_cast<const T*>(d.B_) + b * d.b_sb + t * d.b_st, n + 4 * i, N);
      rC[i] = fetch<4>(static_cast<const T*>(d.C_) + b * d.c_sb + t * d.c_st, n + 4 * i, N);
    }
  }
  __device__ __forceinline__ Pack<T, S::V> u(int i) const { return bits<S::V>(ru[i]); }
  __device__ __forceinline__ Pack<T, S::V> dt(int i) const { return bits<S::V>(rdt[i]); }
  __device__ __forceinline__ Pack<T, S::V> dy(int i) const { return bits<S::V>(rdy[i]); }
  __device__ __forceinline__ void put_bc(T* B, T* C) const {
    const int at = (threadIdx.x & 31) * (S::NP / 2);
#pragma unroll
    for (int i = 0; i < S::NB; ++i) {
      *reinterpret_cast<Raw4*>(B + at + 4 * i) = rB[i];
      *reinterpret_cast<Raw4*>(C + at + 4 * i) = rC[i];
    }
  }
};

// The same in shared memory, fetched by asynchronous copies RING - 1 tiles ahead: a warp alone on its scheduler takes less
// time for a tile than one load from memory. Every lane reads back only what it copied itself.
constexpr int RING = 3;

template <typename T, int G, int CT, bool VEC, bool DY>
struct Ring {
  using S = Shape<T, G, CT>;
  struct alignas(16) Stage {
    T u[LT * S::CW], dt[LT * S::CW], dy[DY ? LT * S::CW : 8];
    T B[LT * S::NP], C[LT * S::NP];
  } stage[RING];

  template <int V>
  static __device__ __forceinline__ void fetch(T* to, const T* base, long long at, int c, int D) {
    constexpr int BYTES = V * static_cast<int>(sizeof(T));
    if constexpr (VEC && BYTES >= 4) {
      copy_async<BYTES>(to, c < D ? base + at + c : base, c < D);
    } else {
      const Pack<T, V> r = load_row<T, V, VEC>(base + at, c, D);
      r.store(to);
    }
  }
  // always closes a group, so that the groups count the tiles; nothing is copied past the segment's `end`
  template <bool WANT_B, bool WANT_C>
  __device__ __forceinline__ void load(const BdhScanDesc& d, int tile, int end, int b, int c0, int len) {
    const int lane = threadIdx.x & 31, t = tile * LT + lane / 2, c = c0 + (lane & 1) * S::E, n = (lane & 1) * (S::NP / 2);
    if (tile >= 0 && tile < end) {
      Stage& s = stage[tile % RING];
      const int D = t < len ? d.D : 0, N = t < len ? d.N : 0;
#pragma unroll
      for (int i = 0; i < S::NV; ++i) {
        const int at = lane * S::E + i * S::V;
        fetch<S::V>(s.u + at, static_cast<const T*>(d.u), b * d.u_sb + t * d.u_st, c + i * S::V, D);
        fetch<S::V>(s.dt + at, static_cast<const T*>(d.dt), b * d.dt_sb + t * d.dt_st, c + i * S::V, D);
        if constexpr (DY) fetch<S::V>(s.dy + at, static_cast<const T*>(d.dy), b * d.dy_sb + t * d.dy_st, c + i * S::V, D);
      }
#pragma unroll
      for (int i = 0; i < S::NB; ++i) {
        const int at = lane * (S::NP / 2) + 4 * i;
        if constexpr (WANT_B) fetch<4>(s.B + at, static_cast<const T*>(d.B_), b * d.b_sb + t * d.b_st, n + 4 * i, N);
        if constexpr (WANT_C) fetch<4>(s.C + at, static_cast<const T*>(d.C_), b * d.c_sb + t * d.c_st, n + 4 * i, N);
      }
    }
    copy_close();
  }
  struct View {
    const Stage& s;
    template <int V>
    static __device__ __forceinline__ Pack<T, V> get(const T* p) {
      Pack<T, V> r;
      r.load(p);
      return r;
    }
    __device__ __forceinline__ int lane() const { return threadIdx.x & 31; }
    __device__ __forceinline__ Pack<T, S::V> u(int i) const { return get<S::V>(s.u + lane() * S::E + i * S::V); }
    __device__ __forceinline__ Pack<T, S::V> dt(int i) const { return get<S::V>(s.dt + lane() * S::E + i * S::V); }
    __device__ __forceinline__ Pack<T, S::V> dy(int i) const { return get<S::V>(s.dy + lane() * S::E + i * S::V); }
  };
  __device__ __forceinline__ View at(int tile) const { return View{stage[tile % RING]}; }
};

// What a warp's compute loop reads. Rows are padded by 16 bytes, so that eight lanes that store four rows meet no bank twice.
// (B and C are read as they came: made fp32 beside this they cost more shared memory and stores than the conversions,
// 16 states 5 %, 64 states 2.7 times.)
template <int G, int CT, bool DY>
struct alignas(16) WarpMem {
  static constexpr int NP = 4 * G, CW = 32 / G * CT;
  float2 step[LT][CW + 2];                             // dt', dt' u
  float dy[DY ? LT : 1][CW + 4];
  float bias[CW], skip[CW];

  static constexpr int ZEROS = CW;                     // the columns behind the channels, which stay 0
  __device__ __forceinline__ void params(const BdhScanDesc& d, int c0) {
    if (const int t = threadIdx.x & 31; t < LT) {
      step[t][CW] = step[t][CW + 1] = make_float2(0.f, 0.f);
      if constexpr (DY) dy[t][CW] = dy[t][CW + 1] = 0.f;
    }
    for (int i = threadIdx.x & 31; i < CW; i += 32) {
      bias[i] = (d.dt_bias && c0 + i < d.D) ? d.dt_bias[c0 + i] : 0.f;
      skip[i] = (d.skip && c0 + i < d.D) ? d.skip[c0 + i] : 0.f;
    }
  }
  // Rows behind `len` get dt' = 0: the states stay as they are. (Channels behind D need nothing: their u, dy and A
  // read as 0.)
  template <typename T, typename Source>
  __device__ __forceinline__ void put(const BdhScanDesc& d, const Source& x, int t0, int len) {
    using S = Shape<T, G, CT>;
    const int lane = threadIdx.x & 31, t = lane / 2, c = (lane & 1) * S::E;
    const f2 keep = t0 + t < len ? ~f2{0} : f2{0};       // (bits, not a factor: the bias alone may be infinite)
    float dt[S::E + 1], uu[S::E + 1];
    dt[S::E] = uu[S::E] = 0.f;
#pragma unroll
    for (int i = 0; i < S::NV; ++i) {
      const Pack<T, S::V> pd = x.dt(i), pu = x.u(i);
#pragma unroll
      for (int j = 0; j < S::V; ++j) {
        dt[i * S::V + j] = pd[j] + bias[c + i * S::V + j];
        uu[i * S::V + j] = pu[j];
      }
    }
#pragma unroll
    for (int j = 0; j < S::E; j += 2) {
      f2 s = pack2(dt[j], dt[j + 1]);
      if (d.softplus) s = softplus2(s);
      s &= keep;
      float s0, s1, v0, v1;
      unpack2(s, s0, s1);
      unpack2(mul2(s, pack2(uu[j], uu[j + 1])), v0, v1);
      if constexpr (S::E > 1)
        *reinterpret_cast<float4*>(&step[t][c + j]) = make_float4(s0, v0, s1, v1);
      else
        step[t][c] = make_float2(s0, v0);
    }
    if constexpr (DY) {
#pragma unroll
      for (int i = 0; i < S::NV; ++i) {
        const Pack<T, S::V> p = x.dy(i);
#pragma unroll
        for (int j = 0; j < S::V; ++j) dy[t][c + i * S::V + j] = p[j];
      }
    }
  }
  __device__ __forceinline__ void steps(int t, int cl, float (&dt)[CT], float (&du)[CT]) const {
    if constexpr (CT == 2) {
      const float4 v = *reinterpret_cast<const float4*>(&step[t][cl]);
      dt[0] = v.x; du[0] = v.y;
      dt[1] = v.z; du[1] = v.w;
    } else {
      const float2 v = step[t][cl];
      dt[0] = v.x;
      du[0] = v.y;
    }
  }
  __device__ __forceinline__ void dys(int t, int cl, float (&g)[CT]) const {
    if constexpr (CT == 2) {
      const float2 v = *reinterpret_cast<const float2*>(&dy[t][cl]);
      g[0] = v.x;
      g[1] = v.y;
    } else {
      g[0] = dy[t][cl];
    }
  }
};

// This lane's 4 states (n0 ..) of channel c in a [.., D, N] tensor
__device__ __forceinline__ void load_state(const float* p, int c, int n0, const BdhScanDesc& d, f2 (&h)[2]) {
  float v[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = (p != nullptr && c < d.D && n0 + j < d.N) ? p[static_cast<long long>(c) * d.N + n0 + j] : 0.f;
  h[0] = pack2(v[0], v[1]);
  h[1] = pack2(v[2], v[3]);
}
__device__ __forceinline__ void store_state(float* p, int c, int n0, const BdhScanDesc& d, const f2 (&h)[2]) {
  float v[4];
  unpack2(h[0], v[0], v[1]);
  unpack2(h[1], v[2], v[3]);
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (c < d.D && n0 + j < d.N) p[static_cast<long long>(c) * d.N + n0 + j] = v[j];
}

// States that N is padded with have to stay 0 whatever their channel's step, which may be infinite, and 0 * inf is not 0.
// Lanes of padding alone read the step (and dy) of a column of zeros behind the warp's channels, which costs nothing; a lane that has
// both kinds (N not a multiple of 4) clears the others' bits (3 % of a pass).
enum { PACKS, ELEMENTS, MIXED };                       // rows in packs of 16 bytes; element by element; so, with such lanes
struct Real {
  f2 m[2];                             // all bits of this lane's states below N
  __device__ __forceinline__ Real(int n0, int N) {
    unsigned v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = n0 + j < N ? 0xffffffffu : 0u;
    m[0] = static_cast<f2>(v[1]) << 32 | v[0];
    m[1] = static_cast<f2>(v[3]) << 32 | v[2];
  }
  template <int FIT>
  __device__ __forceinline__ f2 keep(f2 x, int j) const { return FIT == MIXED ? x & m[j] : x; }
};

// A2 = A log2(e); 0 for padding
template <int CT>
__device__ __forceinline__ void load_a(const BdhScanDesc& d, int c, int n0, f2 (&A2)[CT][2]) {
#pragma unroll
  for (int k = 0; k < CT; ++k) {
    load_state(d.A, c + k, n0, d, A2[k]);
    A2[k][0] = mul2(A2[k][0], both(LOG2E));
    A2[k][1] = mul2(A2[k][1], both(LOG2E));
  }
}

// h exp(x), x in units of ln 2, for a whole segment's x: A and the steps may have any sign, so the factor alone may be past 2^128
// where the product is not. It is applied in two halves, and a state of 0 (nothing came in yet) or an infinite one stays what it
// is, as it does step by step.
__device__ __forceinline__ float grown(float h, float x) {
  const float half = ex2(0.5f * x);
  return h + h == h ? h : h * half * half;             // (0 and the infinities are their own doubles)
}
__device__ __forceinline__ f2 grown2(f2 h, f2 x) {
  float h0, h1, x0, x1;
  unpack2(h, h0, h1);
  unpack2(x, x0, x1);
  return pack2(grown(h0, x0), grown(h1, x1));
}

// The state a segment starts from: `h` (the sequence's own) carried through the segments before it, in order; in reverse
// through those behind it.
template <int CT, int NP>
__device__ __forceinline__ void carry(const ScanArgs& a, int b, int from, int to, int by, int c, int n0, const f2 (&A2)[CT][2], f2 (&h)[CT][2]) {
  const Real real(n0, a.d.N);
  constexpr int AT_ONCE = 4;                           // segments whose loads go out together: the chain through h waits once for them
  for (int left = (to - from) * by, s = from; left > 0; left -= AT_ONCE, s += AT_ONCE * by) {
    float dt[AT_ONCE][CT];
    f2 in[AT_ONCE][CT][2];
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i)
#pragma unroll
      for (int k = 0; k < CT; ++k) {
        dt[i][k] = 0.f;
        in[i][k][0] = in[i][k][1] = both(0.f);
        if (i < left && c + k < a.d.D) {
          const long long at = (static_cast<long long>(b) * a.segs + s + i * by) * a.d.D + c + k;
          dt[i][k] = a.seg_dt[at];
          load4(a.seg_state + at * NP + n0, in[i][k][0], in[i][k][1]);
        }
      }
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i)
#pragma unroll
      for (int k = 0; k < CT; ++k)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          h[k][j] = real.keep<MIXED>(add2(grown2(h[k][j], mul2(both(dt[i][k]), A2[k][j])), in[i][k][j]), j);
  }
}

// The factors of a few steps, made ahead of the chain through h: its loads must not stand behind the stores of the steps
// before, which the compiler cannot tell from them.
template <int G, int CT, bool WANT_C>
struct Steps {
  static constexpr int N = 4 / CT;
  f2 e[N][CT][2], in[N][CT][2], k[WANT_C ? N : 1][2];
  template <typename Mem, typename Rows>
  __device__ __forceinline__ void make(const Mem& sh, const Rows& rows, int t, int cl, int n0, const f2 (&A2)[CT][2]) {
#pragma unroll
    for (int s = 0; s < N; ++s) {
      float dt[CT], du[CT];
      f2 b[2];
      sh.steps(t + s, cl, dt, du);
      rows.B(t + s, n0, b);
      if constexpr (WANT_C) rows.C(t + s, n0, k[s]);
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        e[s][c][0] = decay(dt[c], A2[c][0]);
        e[s][c][1] = decay(dt[c], A2[c][1]);
        in[s][c][0] = mul1(du[c], b[0]);
        in[s][c][1] = mul1(du[c], b[1]);
      }
    }
  }
};

// This lane's states of B and C at a step of rows [LT][NP]
template <typename T, int NP>
struct RowsOf {
  const T *b, *c;
  static __device__ __forceinline__ void get(const T* p, f2 (&f)[2]) { Pairs<T, 4>::get(*reinterpret_cast<const typename Pack<T, 4>::Raw*>(p), f); }
  __device__ __forceinline__ void B(int t, int n0, f2 (&f)[2]) const { get(b + t * NP + n0, f); }
  __device__ __forceinline__ void C(int t, int n0, f2 (&f)[2]) const { get(c + t * NP + n0, f); }
};

struct Where {
  int part, b, seg;                    // channels, sequence, segment
};
__device__ __forceinline__ Where where(const ScanArgs& a, long long unit) {
  Where w;
  w.part = static_cast<int>(unit % a.parts);
  const int bs = static_cast<int>(unit / a.parts);
  w.b = bs / a.segs;
  w.seg = bs - w.b * a.segs;
  return w;
}

// ---- forward -----------------------------------------------------------------------------------------
// Each warp on its own. The partial sums over a lane's 4 states go through shared memory: a channel's G lanes are
// added up where the outputs are written, which costs a store a step instead of a chain of exchanges.
template <typename T, int G, int CT, bool VEC>
struct FwdMem {
  WarpMem<G, CT, false> in;
  alignas(16) T zeros[Shape<T, G, CT>::E];             // as wide as a lane's channels
  alignas(16) float part[LT][CT * 32 + 4];
  Ring<T, G, CT, VEC, false> ring;
};

template <typename T, int G, int CT, int FIT>
__global__ void __launch_bounds__(32 * FWD_WARPS, FWD_BLOCKS) selective_scan_fwd_kernel(const ScanArgs a, long long units, float* marks) {
  constexpr bool VEC = FIT == PACKS;
  using S = Shape<T, G, CT>;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  const int lane = threadIdx.x & 31;
  const long long unit = static_cast<long long>(blockIdx.x) * FWD_WARPS + (threadIdx.x >> 5);
  if (unit >= units) return;
  FwdMem<T, G, CT, VEC>& sh = reinterpret_cast<FwdMem<T, G, CT, VEC>*>(smem_raw)[threadIdx.x >> 5];
  const BdhScanDesc& d = a.d;
  const Where w = where(a, unit);
  const int n0 = lane % G * 4, cl = lane / G * CT, c0 = w.part * S::CW, c = c0 + cl;
  const int len = a.len.get(w.b, d.T);
  const int first = w.seg * a.per_seg, last = min(first + a.per_seg, a.tiles), end = min(last, (len + LT - 1) / LT);
#pragma unroll
  for (int i = 0; i < RING - 1; ++i) sh.ring.template load<true, true>(d, first + i, end, w.b, c0, len);
  const Real real(n0, d.N);
  const int cs = n0 < d.N ? cl : sh.in.ZEROS;          // where this lane reads its steps
  f2 A2[CT][2], h[CT][2];
  load_a<CT>(d, c, n0, A2);
#pragma unroll
  for (int k = 0; k < CT; ++k)
    load_state(d.h0 ? d.h0 + static_cast<long long>(w.b) * d.D * d.N : nullptr, c + k, n0, d, h[k]);
  carry<CT, S::NP>(a, w.b, 0, w.seg, 1, c, n0, A2, h);
  sh.in.params(d, c0);
  for (int i = lane; i < S::E; i += 32) sh.zeros[i] = elem_from_float<T>(0.f);
  __syncwarp();
  const int row = lane / 2, col = (lane & 1) * S::E;
  for (int tile = first; tile < last; ++tile) {
    const int t0 = tile * LT;
    if (tile < end) {
      copy_wait<RING - 2>();
      sh.in.template put<T>(d, sh.ring.at(tile), t0, len);
      __syncwarp();
      const RowsOf<T, S::NP> bc{sh.ring.at(tile).s.B, sh.ring.at(tile).s.C};
      sh.ring.template load<true, true>(d, tile + RING - 1, end, w.b, c0, len);
      if (marks != nullptr)
#pragma unroll
        for (int k = 0; k < CT; ++k)
          if (c + k < d.D)
            *reinterpret_cast<ulonglong2*>(marks + ((static_cast<long long>(w.b) * a.tiles + tile) * d.D + c + k) * S::NP + n0) =
                make_ulonglong2(h[k][0], h[k][1]);
      using Group = Steps<G, CT, true>;
      Group now, next;
      now.make(sh.in, bc, 0, cs, n0, A2);
#pragma unroll
      for (int s0 = 0; s0 < LT; s0 += Group::N) {
        if (s0 + Group::N < LT) next.make(sh.in, bc, s0 + Group::N, cs, n0, A2);
#pragma unroll
        for (int s = 0; s < Group::N; ++s)
#pragma unroll
          for (int k = 0; k < CT; ++k) {
            h[k][0] = real.template keep<FIT>(fma2(now.e[s][k][0], h[k][0], now.in[s][k][0]), 0);
            h[k][1] = real.template keep<FIT>(fma2(now.e[s][k][1], h[k][1], now.in[s][k][1]), 1);
            sh.part[s0 + s][k * 32 + lane] = sum2(fma2(now.k[s][1], h[k][1], mul2(now.k[s][0], h[k][0])));
          }
        now = next;
      }
      __syncwarp();
    }
    if (t0 + row < d.T) {
      T* y = static_cast<T*>(d.y) + (static_cast<long long>(w.b) * d.T + t0 + row) * d.D;
      const bool in = t0 + row < len;
      const T* skip_u = d.skip != nullptr ? sh.ring.at(tile).s.u + lane * S::E : sh.zeros;
#pragma unroll
      for (int i = 0; i < S::NV; ++i) {
        Pack<T, S::V> o, u;                            // (without a skip u is 0 here: 0 times an infinite u is not)
        u.load(skip_u + i * S::V);
#pragma unroll
        for (int j = 0; j < S::V; ++j) {
          const int cc = col + i * S::V + j;
          float v = 0.f;
          if (in) {
            const float* p = &sh.part[row][cc % CT * 32 + cc / CT * G];
            if constexpr (G == 2) {
              const float2 q = *reinterpret_cast<const float2*>(p);
              v = q.x + q.y;
            } else {
#pragma unroll
              for (int g = 0; g < G; g += 4) {
                const float4 q = *reinterpret_cast<const float4*>(p + g);
                v += (q.x + q.y) + (q.z + q.w);
              }
            }
            v = fmaf(sh.in.skip[cc], u[j], v);
          }
          o.set(j, v);
        }
        store_row<T, S::V, VEC>(y, c0 + col + i * S::V, d.D, o);
      }
    }
  }
  if (w.seg == a.segs - 1)
#pragma unroll
    for (int k = 0; k < CT; ++k) store_state(d.hT + static_cast<long long>(w.b) * d.D * d.N, c + k, n0, d, h[k]);
}

// States of the segments from zero: h_t = a_t h_{t-1} + dt' u B_t, or in reverse r_t = a_t (r_{t+1} + dy_t C_t); and the
// sum of the segment's steps. Each warp on its own.
template <typename T, int G, int CT, bool VEC, bool REV>
struct SweepMem {
  WarpMem<G, CT, REV> in;
  Ring<T, G, CT, VEC, REV> ring;
};

template <typename T, int G, int CT, int FIT, bool REV>
__global__ void __launch_bounds__(32 * FWD_WARPS, FWD_BLOCKS) selective_scan_sweep_kernel(const ScanArgs a, long long units, float* seg_state, float* seg_dt) {
  constexpr bool VEC = FIT == PACKS;
  using S = Shape<T, G, CT>;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  const int lane = threadIdx.x & 31;
  const long long unit = static_cast<long long>(blockIdx.x) * FWD_WARPS + (threadIdx.x >> 5);
  if (unit >= units) return;
  SweepMem<T, G, CT, VEC, REV>& sh = reinterpret_cast<SweepMem<T, G, CT, VEC, REV>*>(smem_raw)[threadIdx.x >> 5];
  const BdhScanDesc& d = a.d;
  const Where w = where(a, unit);
  const int n0 = lane % G * 4, cl = lane / G * CT, c0 = w.part * S::CW, c = c0 + cl;
  const int len = a.len.get(w.b, d.T);
  const int first = w.seg * a.per_seg, end = min(min(first + a.per_seg, a.tiles), (len + LT - 1) / LT);
  const int n = end - first;
  // the i-th tile of the walk; the copies run ahead in the same order
  const auto tile_of = [&](int i) { return REV ? end - 1 - i : first + i; };
#pragma unroll
  for (int i = 0; i < RING - 1; ++i) sh.ring.template load<!REV, REV>(d, i < n ? tile_of(i) : -1, end, w.b, c0, len);
  const Real real(n0, d.N);
  const int cs = n0 < d.N ? cl : sh.in.ZEROS;
  f2 A2[CT][2], h[CT][2];
  float total[CT];
  load_a<CT>(d, c, n0, A2);
#pragma unroll
  for (int k = 0; k < CT; ++k) {
    h[k][0] = h[k][1] = both(0.f);
    total[k] = 0.f;
  }
  sh.in.params(d, c0);
  __syncwarp();
  for (int i = 0; i < n; ++i) {
    const int tile = tile_of(i);
    copy_wait<RING - 2>();
    sh.in.template put<T>(d, sh.ring.at(tile), tile * LT, len);
    __syncwarp();
    const RowsOf<T, S::NP> bc{sh.ring.at(tile).s.B, sh.ring.at(tile).s.C};
    sh.ring.template load<!REV, REV>(d, i + RING - 1 < n ? tile_of(i + RING - 1) : -1, end, w.b, c0, len);
    constexpr int GS = 8 / CT;
#pragma unroll
    for (int s0 = 0; s0 < LT; s0 += GS) {
      f2 e[GS][CT][2], in[GS][CT][2];
#pragma unroll
      for (int s = 0; s < GS; ++s) {
        const int t = REV ? LT - 1 - s0 - s : s0 + s;
        float dt[CT], du[CT];
        f2 b[2];
        sh.in.steps(t, cs, dt, du);
        if constexpr (REV) {
          bc.C(t, n0, b);
          sh.in.dys(t, cs, du);
        } else {
          bc.B(t, n0, b);
        }
#pragma unroll
        for (int k = 0; k < CT; ++k) {
          e[s][k][0] = decay(dt[k], A2[k][0]);
          e[s][k][1] = decay(dt[k], A2[k][1]);
          in[s][k][0] = mul1(du[k], b[0]);
          in[s][k][1] = mul1(du[k], b[1]);
          total[k] += dt[k];
        }
      }
#pragma unroll
      for (int s = 0; s < GS; ++s)
#pragma unroll
        for (int k = 0; k < CT; ++k)
#pragma unroll
          for (int j = 0; j < 2; ++j)
            h[k][j] = real.template keep<FIT>(
                REV ? mul2(e[s][k][j], add2(h[k][j], in[s][k][j])) : fma2(e[s][k][j], h[k][j], in[s][k][j]), j);
    }
    __syncwarp();
  }
#pragma unroll
  for (int k = 0; k < CT; ++k)
    if (c + k < d.D) {
      const long long at = (static_cast<long long>(w.b) * a.segs + w.seg) * d.D + c + k;
      *reinterpret_cast<ulonglong2*>(seg_state + at * S::NP + n0) = make_ulonglong2(h[k][0], h[k][1]);
      if (n0 == 0) seg_dt[at] = total[k];
    }
}

// ---- backward ----------------------------------------------------------------------------------------
struct ScanGrads {
  const float* marks;                  // [B][tiles][D][NP]: h at the start of every tile
  float* bc;                           // [channel blocks][B][T][2 NP]: partial dB | dC
  float* da;                           // [B][segs][D][NP]: partial dA
  float* per_channel;                  // [2][B][segs][D]: partial dD, dbias
};

template <typename T, int G, int CT>
struct BwdMem {
  static constexpr int NP = 4 * G, CW = 32 / G * CT;
  struct PerWarp {
    WarpMem<G, CT, true> in;
    alignas(16) T B[LT * NP], C[LT * NP];
    float2 out[LT][CW + 2];            // sum g B, sum A2 q
    ulonglong2 h[LT][CT][32];          // h_{t-1}, each lane its own
    __device__ __forceinline__ RowsOf<T, NP> bc() const { return {B, C}; }
  } warp[BWD_WARPS];
  alignas(16) float bc[BWD_WARPS][LT][2 * NP];     // the warps' sums over their channels
  alignas(16) float last[BWD_WARPS][NP];           // dC of a sequence's last row, where rows of its tile are behind it
};

// What a step of the reverse walk reads
template <typename T, int G, int CT>
struct BwdStep {
  float dt[CT], du[CT], gy[CT];
  f2 b[2], c[2];
  ulonglong2 h[CT];
  __device__ __forceinline__ void load(const typename BwdMem<T, G, CT>::PerWarp& sh, int t, int lane, int cl, int n0) {
    sh.in.steps(t, cl, dt, du);
    sh.in.dys(t, cl, gy);
    sh.bc().B(t, n0, b);
    sh.bc().C(t, n0, c);
#pragma unroll
    for (int k = 0; k < CT; ++k) h[k] = sh.h[t][k][lane];
  }
};

template <typename T, int G, int CT, int FIT>
__global__ void __launch_bounds__(32 * BWD_WARPS, BWD_BLOCKS) selective_scan_bwd_kernel(const ScanArgs a, const ScanGrads o) {
  constexpr bool VEC = FIT == PACKS;
  using S = Shape<T, G, CT>;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  BwdMem<T, G, CT>& all = *reinterpret_cast<BwdMem<T, G, CT>*>(smem_raw);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  typename BwdMem<T, G, CT>::PerWarp& sh = all.warp[warp];
  const BdhScanDesc& d = a.d;
  const Where w = where(a, blockIdx.x);
  const int n0 = lane % G * 4, cl = lane / G * CT, c0 = (w.part * BWD_WARPS + warp) * S::CW, c = c0 + cl;
  const int len = a.len.get(w.b, d.T);
  const Real real(n0, d.N);
  const int cs = n0 < d.N ? cl : sh.in.ZEROS;
  f2 A2[CT][2], r[CT][2], da[CT][2];
  load_a<CT>(d, c, n0, A2);
#pragma unroll
  for (int k = 0; k < CT; ++k) {
    load_state(d.dhT ? d.dhT + static_cast<long long>(w.b) * d.D * d.N : nullptr, c + k, n0, d, r[k]);
    da[k][0] = da[k][1] = both(0.f);
  }
  carry<CT, S::NP>(a, w.b, a.segs - 1, w.seg, -1, c, n0, A2, r);
  sh.in.params(d, c0);
  float sum_skip[S::E], sum_bias[S::E];                // of this lane's channels, over its rows
#pragma unroll
  for (int j = 0; j < S::E; ++j) sum_skip[j] = sum_bias[j] = 0.f;
  const int first = w.seg * a.per_seg, last = min(first + a.per_seg, a.tiles);
  const int row = lane / 2, col = (lane & 1) * S::E;
  const unsigned skip_bits = d.skip != nullptr ? ~0u : 0u;     // (without a skip dy, which may be infinite, has no part in du)
  Tile<T, G, CT, VEC, true> x;
  x.load(d, w.b, c0, (last - 1) * LT, len);
  f2 mark[CT][2];                                      // the next tile's first state, fetched with its rows
  const auto load_marks = [&](int tile) {
#pragma unroll
    for (int k = 0; k < CT; ++k) {
      mark[k][0] = mark[k][1] = both(0.f);
      if (c + k < d.D && tile * LT < len)
        load4(o.marks + ((static_cast<long long>(w.b) * a.tiles + tile) * d.D + c + k) * S::NP + n0, mark[k][0], mark[k][1]);
    }
  };
  load_marks(last - 1);
  __syncwarp();
  for (int tile = last - 1; tile >= first; --tile) {
    const int t0 = tile * LT;
    const bool any = t0 < len;                         // (the same for the whole block)
    const int rows = min(LT, len - t0);                // of the sequence
    Pack<T, S::V> u[S::NV], dt_raw[S::NV], dy[S::NV];
#pragma unroll
    for (int i = 0; i < S::NV; ++i) {
      u[i] = x.u(i);
      dt_raw[i] = x.dt(i);
      dy[i] = x.dy(i);
    }
    if (any) {
      f2 h[CT][2], dat[CT][2];
      sh.in.template put<T>(d, x, t0, len);
      x.put_bc(sh.B, sh.C);
#pragma unroll
      for (int k = 0; k < CT; ++k) {
        h[k][0] = mark[k][0];
        h[k][1] = mark[k][1];
        dat[k][0] = dat[k][1] = both(0.f);
      }
      __syncwarp();
      if (tile > first) {
        x.load(d, w.b, c0, t0 - LT, len);
        load_marks(tile - 1);
      }
      using Group = Steps<G, CT, false>;
      const RowsOf<T, S::NP> bc = sh.bc();
      Group now, next;
      now.make(sh.in, bc, 0, cs, n0, A2);
#pragma unroll
      for (int s0 = 0; s0 < LT; s0 += Group::N) {
        if (s0 + Group::N < LT) next.make(sh.in, bc, s0 + Group::N, cs, n0, A2);
#pragma unroll
        for (int s = 0; s < Group::N; ++s)
#pragma unroll
          for (int k = 0; k < CT; ++k) {
            sh.h[s0 + s][k][lane] = make_ulonglong2(h[k][0], h[k][1]);
            h[k][0] = real.template keep<FIT>(fma2(now.e[s][k][0], h[k][0], now.in[s][k][0]), 0);
            h[k][1] = real.template keep<FIT>(fma2(now.e[s][k][1], h[k][1], now.in[s][k][1]), 1);
          }
        now = next;
      }
      if (rows < LT) {
        // Rows behind the sequence multiply the state, which may be infinite, by their zeros: they get a state of 0. The last
        // row's dC, which the walk makes of the state behind it, is made here.
        float gy[CT], cv[4];
        sh.in.dys(rows - 1, cs, gy);
        f2 sc0 = mul1(gy[0], h[0][0]), sc1 = mul1(gy[0], h[0][1]);
#pragma unroll
        for (int k = 1; k < CT; ++k) {
          sc0 = fma1(gy[k], h[k][0], sc0);
          sc1 = fma1(gy[k], h[k][1], sc1);
        }
        unpack2(sc0, cv[0], cv[1]);
        unpack2(sc1, cv[2], cv[3]);
        int at;
        bool once;
        sum_over<4, S::LANES, G>(cv, lane, at, once);
        constexpr int CLEFT = 4 / S::LANES > 1 ? 4 / S::LANES : 1;
        if (once)
#pragma unroll
          for (int i = 0; i < CLEFT; ++i) all.last[warp][n0 + at + i] = cv[i];
#pragma unroll 1
        for (int t = rows; t < LT; ++t)
#pragma unroll
          for (int k = 0; k < CT; ++k) sh.h[t][k][lane] = make_ulonglong2(0, 0);
      }
      BwdStep<T, G, CT> at_t, before;
      at_t.load(sh, LT - 1, lane, cs, n0);
#pragma unroll 4
      for (int t = LT - 1; t >= 0; --t) {
        before.load(sh, t > 0 ? t - 1 : 0, lane, cs, n0);              // ahead of this step's stores
        f2 sb0, sb1, sc0, sc1;
        float nv[2 * CT];
#pragma unroll
        for (int k = 0; k < CT; ++k) {
          const float dt = at_t.dt[k], du = at_t.du[k], gy = at_t.gy[k];
          const f2 g0 = real.template keep<FIT>(fma1(gy, at_t.c[0], r[k][0]), 0), g1 = real.template keep<FIT>(fma1(gy, at_t.c[1], r[k][1]), 1);
          const f2 e0 = decay(dt, A2[k][0]), e1 = decay(dt, A2[k][1]);
          if (k == 0) {
            sb0 = mul1(du, g0); sb1 = mul1(du, g1);
            sc0 = mul1(gy, h[k][0]); sc1 = mul1(gy, h[k][1]);
          } else {
            sb0 = fma1(du, g0, sb0); sb1 = fma1(du, g1, sb1);
            sc0 = fma1(gy, h[k][0], sc0); sc1 = fma1(gy, h[k][1], sc1);
          }
          r[k][0] = real.template keep<FIT>(mul2(e0, g0), 0);
          r[k][1] = real.template keep<FIT>(mul2(e1, g1), 1);
          h[k][0] = at_t.h[k].x;
          h[k][1] = at_t.h[k].y;
          const f2 q0 = mul2(r[k][0], h[k][0]), q1 = mul2(r[k][1], h[k][1]);
          dat[k][0] = fma1(dt, q0, dat[k][0]);
          dat[k][1] = fma1(dt, q1, dat[k][1]);
          nv[2 * k] = sum2(fma2(g1, at_t.b[1], mul2(g0, at_t.b[0])));
          nv[2 * k + 1] = sum2(fma2(A2[k][1], q1, mul2(A2[k][0], q0)));
        }
        int at;
        bool once;
        sum_over<2 * CT, G, 1>(nv, lane, at, once);
        constexpr int NLEFT = 2 * CT / G > 1 ? 2 * CT / G : 1;
        if (once)
#pragma unroll
          for (int i = 0; i < NLEFT; ++i) reinterpret_cast<float*>(&sh.out[t][cl])[at + i] = nv[i];
        float cv[8];                                   // dB of the 4 states, then dC
        unpack2(sb0, cv[0], cv[1]);
        unpack2(sb1, cv[2], cv[3]);
        unpack2(sc0, cv[4], cv[5]);
        unpack2(sc1, cv[6], cv[7]);
        sum_over<8, S::LANES, G>(cv, lane, at, once);
        constexpr int CLEFT = 8 / S::LANES > 1 ? 8 / S::LANES : 1;
        if (once)
#pragma unroll
          for (int i = 0; i < CLEFT; ++i) all.bc[warp][t][(at + i) / 4 * S::NP + n0 + (at + i) % 4] = cv[i];
        at_t = before;
      }
      if (rows < LT) {
        __syncwarp();
        for (int i = lane; i < S::NP; i += 32) all.bc[warp][rows - 1][S::NP + i] = all.last[warp][i];
      }
#pragma unroll
      for (int k = 0; k < CT; ++k) {                   // sums of tiles: a chain of 16, then one of the tiles
        da[k][0] = add2(da[k][0], dat[k][0]);
        da[k][1] = add2(da[k][1], dat[k][1]);
      }
    } else if (tile > first) {
      x.load(d, w.b, c0, t0 - LT, len);
      load_marks(tile - 1);
    }
    __syncthreads();
    if (t0 + row < d.T) {
      const bool in = t0 + row < len;
      const long long at = (static_cast<long long>(w.b) * d.T + t0 + row) * d.D;
#pragma unroll
      for (int i = 0; i < S::NV; ++i) {
        Pack<T, S::V> pu, pd;
        float raw[S::V + 1], dd[S::V + 1];
        raw[S::V] = dd[S::V] = 0.f;
#pragma unroll
        for (int j = 0; j < S::V; ++j) {
          const int cc = col + i * S::V + j;
          raw[j] = dt_raw[i][j] + sh.in.bias[cc];
          float du = 0.f;
          dd[j] = 0.f;
          if (in) {
            const float2 s = sh.out[row][cc];
            du = fmaf(sh.in.step[row][cc].x, s.x, sh.in.skip[cc] * __uint_as_float(__float_as_uint(dy[i][j]) & skip_bits));
            dd[j] = fmaf(u[i][j], s.x, LN2 * s.y);
            sum_skip[i * S::V + j] = fmaf(dy[i][j], u[i][j], sum_skip[i * S::V + j]);
          }
          pu.set(j, du);
        }
        if (d.softplus && in)
#pragma unroll
          for (int j = 0; j < S::V; j += 2) {
            float s0, s1;
            unpack2(sigmoid2(pack2(raw[j], raw[j + 1])), s0, s1);
            dd[j] *= s0;
            dd[j + 1] *= s1;
          }
#pragma unroll
        for (int j = 0; j < S::V; ++j) {
          pd.set(j, dd[j]);
          sum_bias[i * S::V + j] += dd[j];
        }
        store_row<T, S::V, VEC>(static_cast<T*>(d.du) + at, c0 + col + i * S::V, d.D, pu);
        store_row<T, S::V, VEC>(static_cast<T*>(d.ddt) + at, c0 + col + i * S::V, d.D, pd);
      }
    }
    for (int i = threadIdx.x; i < LT * S::NP / 2; i += 32 * BWD_WARPS) {
      const int t = i / (S::NP / 2), n = i % (S::NP / 2) * 4;
      if (t0 + t >= d.T) break;
      float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
      if (t < rows)
#pragma unroll
        for (int k = 0; k < BWD_WARPS; ++k) {
          const float4 q = *reinterpret_cast<const float4*>(&all.bc[k][t][n]);
          s.x += q.x; s.y += q.y; s.z += q.z; s.w += q.w;
        }
      *reinterpret_cast<float4*>(o.bc + ((static_cast<long long>(w.part) * d.B + w.b) * d.T + t0 + t) * (2 * S::NP) + n) = s;
    }
    __syncthreads();
  }
  const long long seg = static_cast<long long>(w.b) * a.segs + w.seg;
#pragma unroll
  for (int k = 0; k < CT; ++k) {
    if (c + k < d.D) *reinterpret_cast<ulonglong2*>(o.da + (seg * d.D + c + k) * S::NP + n0) = make_ulonglong2(da[k][0], da[k][1]);
    if (w.seg == 0 && d.dh0 != nullptr) store_state(d.dh0 + static_cast<long long>(w.b) * d.D * d.N, c + k, n0, d, r[k]);
  }
  // the 16 lanes of a warp that share channels add their sums up
#pragma unroll
  for (int j = 0; j < S::E; ++j) {
#pragma unroll
    for (int off = 16; off > 1; off >>= 1) {
      sum_skip[j] += __shfl_xor_sync(0xffffffffu, sum_skip[j], off);
      sum_bias[j] += __shfl_xor_sync(0xffffffffu, sum_bias[j], off);
    }
    const int cc = c0 + col + j;
    if (lane < 2 && cc < d.D) {
      o.per_channel[seg * d.D + cc] = sum_skip[j];
      o.per_channel[(static_cast<long long>(d.B) * a.segs + seg) * d.D + cc] = sum_bias[j];
    }
  }
}

// dB, dC: sums over the channel blocks, in order
template <typename T>
__global__ void __launch_bounds__(256) selective_scan_bc_kernel(const float* part, int blocks, long long rows, int NP, int N, T* dB, T* dC) {
  const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x, all = rows * 2 * NP;
  if (i >= all) return;
  const int n = static_cast<int>(i % (2 * NP));
  if (n % NP >= N) return;
  float s = 0.f;
#pragma unroll 8
  for (int k = 0; k < blocks; ++k) s += part[k * all + i];
  (n >= NP ? dC : dB)[i / (2 * NP) * N + n % NP] = elem_from_float<T>(s);
}

// dA, dD, dbias: sums over sequences and segments, in order
__global__ void __launch_bounds__(256) selective_scan_params_kernel(const float* da, const float* per_channel, int parts, int D, int NP, int N,
                                                                    float* dA, float* dD, float* dbias) {
  const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x, na = static_cast<long long>(D) * NP;
  float s = 0.f;
  if (i < na) {
#pragma unroll 8
    for (int k = 0; k < parts; ++k) s += da[k * na + i];
    const int n = static_cast<int>(i % NP);
    if (n < N) dA[i / NP * N + n] = s;
  } else if (i < na + 2 * D) {
    const long long j = i - na, what = j / D;
    for (int k = 0; k < parts; ++k) s += per_channel[(what * parts + k) * D + j % D];
    float* p = what ? dbias : dD;
    if (p != nullptr) p[j % D] = s;
  }
}

// ---- one token ---------------------------------------------------------------------------------------
// Bound by the states: 4 B N D read and written per stream. A lane group takes R streams of one channel: A, bias and
// skip are read once, and each lane makes the steps (a softplus each) of its share of the streams for the others.
template <typename T, int G, int R>
__global__ void __launch_bounds__(STEP_THREADS) selective_scan_step_kernel(const BdhScanDesc d, const float* h, long long h_sb, float* out,
                                                                           long long out_sb, const unsigned char* active, int vec) {
  constexpr int OWN = (R + G - 1) / G;                 // streams whose steps this lane makes
  const int lane = threadIdx.x & 31, ng = lane % G, n0 = 4 * ng;
  const long long i = (static_cast<long long>(blockIdx.x) * STEP_THREADS + threadIdx.x) / G;
  const int c = static_cast<int>(i % d.D);
  const long long b0 = i / d.D * R;
  const bool live = b0 < d.B;
  const long long at = static_cast<long long>(c) * d.N + n0;
  float v[R][4], a[4], y[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const float* p = h + (b0 + r) * h_sb + at;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[r][j] = 0.f;
    if (!live || b0 + r >= d.B) continue;
    if (vec) {
      if (n0 < d.N) *reinterpret_cast<float4*>(v[r]) = *reinterpret_cast<const float4*>(p);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n0 + j < d.N) v[r][j] = p[j];
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) a[j] = live && n0 + j < d.N ? d.A[at + j] * LOG2E : 0.f;
  const float bias = live && d.dt_bias ? d.dt_bias[c] : 0.f, skip = live && d.skip ? d.skip[c] : 0.f;
  float step[OWN], input[OWN];
#pragma unroll
  for (int k = 0; k < OWN; ++k) {
    const long long b = b0 + k * G + ng;
    const bool on = live && k * G + ng < R && b < d.B && (active == nullptr || active[b] != 0);
    input[k] = on ? elem_to_float<T>(static_cast<const T*>(d.u)[b * d.u_sb + c]) : 0.f;
    step[k] = on ? elem_to_float<T>(static_cast<const T*>(d.dt)[b * d.dt_sb + c]) + bias : 0.f;
    float same;
    if (d.softplus) unpack2(softplus2(both(step[k])), step[k], same);
    if (!on) step[k] = 0.f;
  }
  const int first = lane - ng;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const long long b = b0 + r;
    const float dt = __shfl_sync(0xffffffffu, step[r / G], first + r % G), u = __shfl_sync(0xffffffffu, input[r / G], first + r % G);
    const bool on = live && b < d.B && (active == nullptr || active[b] != 0);
    float sum = 0.f;
    if (on && n0 < d.N) {
      const T* pb = static_cast<const T*>(d.B_) + b * d.b_sb + n0;
      const T* pc = static_cast<const T*>(d.C_) + b * d.c_sb + n0;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n0 + j < d.N) {
          v[r][j] = fmaf(ex2(fmaf(dt, a[j], EVEN)), v[r][j], dt * u * elem_to_float<T>(pb[j]));
          sum = fmaf(elem_to_float<T>(pc[j]), v[r][j], sum);
        }
    }
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    y[r] = !on ? 0.f : d.skip ? fmaf(skip, u, sum) : sum;
    if (!live || b >= d.B) continue;
    float* p = out + b * out_sb + at;
    if (on || p != h + b * h_sb + at) {
      if (vec) {
        if (n0 < d.N) *reinterpret_cast<float4*>(p) = *reinterpret_cast<const float4*>(v[r]);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n0 + j < d.N) p[j] = v[r][j];
      }
    }
    if (ng == r % G) static_cast<T*>(d.y)[b * d.D + c] = elem_from_float<T>(y[r]);
  }
}

// ---- host --------------------------------------------------------------------------------------------
bool multiple(const void* p, long long bytes) { return reinterpret_cast<unsigned long long>(p) % bytes == 0; }

int checked(const BdhScanDesc& d) {
  if (d.dtype < 0 || d.dtype > 2 || d.B < 0 || d.T < 0 || d.D < 1 || d.N < 1 || d.N > 64) return BDH_ERR_ARGUMENT;
  return BDH_OK;
}

int lanes_for(int N) { return N <= 8 ? 2 : N <= 16 ? 4 : N <= 32 ? 8 : 16; }

struct Plan {
  int G, CT, parts, tiles, per_seg, segs;
};

Plan plan(const BdhScanDesc& d, int CT, int warps, long long segs) {
  Plan p;
  p.G = lanes_for(d.N);
  p.CT = CT;
  const int cb = warps * 32 / p.G * CT;
  p.parts = (d.D + cb - 1) / cb;
  p.tiles = (d.T + LT - 1) / LT;
  if (segs > p.tiles) segs = p.tiles > 0 ? p.tiles : 1;
  p.per_seg = static_cast<int>((p.tiles + segs - 1) / segs);
  if (p.per_seg < 1) p.per_seg = 1;
  p.segs = p.tiles > 0 ? (p.tiles + p.per_seg - 1) / p.per_seg : 1;
  return p;
}

constexpr int MOST_SEGS = 64;          // so that combining the segments stays cheap beside them

// One or two channels a lane (two: fewer reads of B and C a channel; one: twice the warps), and how many segments
// (which cost the exponentials a second time), by a model of the time of a tile: what a warp alone on its scheduler
// takes and what a busy scheduler (592 of them) takes for one, joined as the root of the sum of squares; and what the
// segments before each segment cost it, which grows with their number squared.
// Measured for 16 states (clocks): one channel 1600 and 1230, two 2350 and 1650; a sweep is 0.8 of a pass. The same figures choose for 8,
// 32 and 64 states, where a lane does the same work on as many states and only the sum over a channel's lanes differs.
Plan fwd_plan(const BdhScanDesc& d) {
  Plan best = plan(d, 2, 1, 1);
  double least = 0;
  for (int CT = 1; CT <= 2; ++CT)
    for (int segs = 1; segs <= MOST_SEGS; segs += segs < 8 ? 1 : 4) {
      const Plan p = plan(d, CT, 1, segs);
      const double alone = CT == 2 ? 2350 : 1600, busy = (CT == 2 ? 1650 : 1230) * (static_cast<double>(d.B) * p.segs * p.parts / 592);
      const double carry = 5000 + 150.0 * p.segs + 55.0 * p.segs * p.segs * d.B * p.parts / 592;
      const double t = p.per_seg * sqrt(alone * alone + busy * busy) * (p.segs > 1 ? 1.8 : 1) + (p.segs > 1 ? carry : 0);
      if (least == 0 || t < least) {
        least = t;
        best = p;
      }
    }
  return best;
}

// Two blocks fit an SM, so blocks run in rounds of 296 (one alone on its SM takes 0.7 of the time of two); a sweep, which
// segments need, is a quarter of the pass.
Plan bwd_plan(const BdhScanDesc& d) {
  Plan best = plan(d, 2, BWD_WARPS, 1);
  double least = 0;
  for (int segs = 1; segs <= MOST_SEGS; ++segs) {
    const Plan p = plan(d, 2, BWD_WARPS, segs);
    const long long blocks = static_cast<long long>(d.B) * p.segs * p.parts;
    const double rounds = blocks <= 148 ? 0.7 : static_cast<double>((blocks + 295) / 296);
    const double carry = 1 + 0.042 * p.segs * p.segs * d.B * p.parts / 296;
    const double t = rounds * (p.per_seg + 0.5) * (p.segs > 1 ? 1.25 : 1) + (p.segs > 1 ? carry : 0);
    if (least == 0 || t < least) {
      least = t;
      best = p;
    }
  }
  return best;
}

long long round4(long long n) { return (n + 3) / 4 * 4; }          // pieces of the scratch start on 16 bytes

long long seg_floats(const BdhScanDesc& d, const Plan& p) {
  return p.segs > 1 ? round4(static_cast<long long>(d.B) * p.segs * d.D * (4 * p.G + 1)) : 0;
}
long long bc_floats(const BdhScanDesc& d, const Plan& p) { return static_cast<long long>(p.parts) * d.B * d.T * 8 * p.G; }
long long da_floats(const BdhScanDesc& d, const Plan& p) { return static_cast<long long>(d.B) * p.segs * d.D * 4 * p.G; }

ScanArgs args_for(const BdhScanDesc& d, const Plan& p, const float* seg) {
  ScanArgs a;
  a.d = d;
  a.len = Lengths{d.lengths, d.lengths64};
  a.tiles = p.tiles; a.per_seg = p.per_seg; a.segs = p.segs; a.parts = p.parts;
  a.seg_state = seg;
  a.seg_dt = seg ? seg + static_cast<long long>(d.B) * p.segs * d.D * (4 * p.G) : nullptr;
  return a;
}

// Can rows be moved in packs of 16 bytes, and those of B and C in packs of 4 states?
bool packs_fit(const BdhScanDesc& d, int size) {
  const int V = 16 / size;
  if (d.D % V || d.N % 4) return false;
  for (const void* q : {d.u, d.dt, d.dy, static_cast<const void*>(d.y), static_cast<const void*>(d.du), static_cast<const void*>(d.ddt)})
    if (!multiple(q, 16)) return false;
  for (long long s : {d.u_sb, d.u_st, d.dt_sb, d.dt_st, d.dy_sb, d.dy_st})
    if (s % V) return false;
  if (!multiple(d.B_, 4 * size) || !multiple(d.C_, 4 * size)) return false;
  for (long long s : {d.b_sb, d.b_st, d.c_sb, d.c_st})
    if (s % 4) return false;
  return true;
}

int launched() { return cudaGetLastError() == cudaSuccess ? BDH_OK : BDH_ERR_LAUNCH; }

template <typename K>
int allow_smem(PerDeviceOnce& once, K kernel, int bytes) {
  return once.run([&] {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) == cudaSuccess ? BDH_OK : BDH_ERR_LAUNCH;
  });
}

template <typename T, int G, int CT, int FIT, bool REV>
int sweep_launch(const ScanArgs& a, const Plan& p, float* seg, cudaStream_t s) {
  // (a sweep's warps: those of the pass that it serves, whose segments it shares)
  ScanArgs sw = a;
  sw.parts = (a.d.D + Shape<T, G, CT>::CW - 1) / Shape<T, G, CT>::CW;
  const long long units = static_cast<long long>(a.d.B) * p.segs * sw.parts, grid = (units + FWD_WARPS - 1) / FWD_WARPS;
  if (grid > 0x7fffffffLL) return BDH_ERR_TOO_LARGE;
  auto kernel = selective_scan_sweep_kernel<T, G, CT, FIT, REV>;
  constexpr int smem = FWD_WARPS * sizeof(SweepMem<T, G, CT, FIT == PACKS, REV>);
  static PerDeviceOnce once;
  if (const int rc = allow_smem(once, kernel, smem)) return rc;
  kernel<<<static_cast<unsigned>(grid), 32 * FWD_WARPS, smem, s>>>(sw, units, seg, const_cast<float*>(a.seg_dt));
  return launched();
}

template <typename T, int G, int CT, int FIT>
int fwd_launch(const BdhScanDesc& d, const Plan& p, float* marks, float* seg, cudaStream_t s) {
  const ScanArgs a = args_for(d, p, p.segs > 1 ? seg : nullptr);
  if (p.segs > 1)
    if (const int rc = sweep_launch<T, G, CT, FIT, false>(a, p, seg, s)) return rc;
  const long long units = static_cast<long long>(d.B) * p.segs * p.parts, grid = (units + FWD_WARPS - 1) / FWD_WARPS;
  if (grid > 0x7fffffffLL) return BDH_ERR_TOO_LARGE;
  auto kernel = selective_scan_fwd_kernel<T, G, CT, FIT>;
  constexpr int smem = FWD_WARPS * sizeof(FwdMem<T, G, CT, FIT == PACKS>);
  static PerDeviceOnce once;
  if (const int rc = allow_smem(once, kernel, smem)) return rc;
  kernel<<<static_cast<unsigned>(grid), 32 * FWD_WARPS, smem, s>>>(a, units, marks);
  return launched();
}

struct BwdOut {
  float *dA, *dD, *dbias;
  void *dB, *dC;
};

template <typename T, int G, int FIT>
int bwd_launch(const BdhScanDesc& d, const Plan& p, const ScanGrads& o, float* seg, const BwdOut& out, cudaStream_t s) {
  constexpr int CT = 2;
  const ScanArgs a = args_for(d, p, p.segs > 1 ? seg : nullptr);
  if (p.segs > 1)
    if (const int rc = sweep_launch<T, G, CT, FIT, true>(a, p, seg, s)) return rc;
  const long long grid = static_cast<long long>(d.B) * p.segs * p.parts;
  if (grid > 0x7fffffffLL) return BDH_ERR_TOO_LARGE;
  auto kernel = selective_scan_bwd_kernel<T, G, CT, FIT>;
  constexpr int smem = sizeof(BwdMem<T, G, CT>);
  static PerDeviceOnce once;
  if (const int rc = allow_smem(once, kernel, smem)) return rc;
  kernel<<<static_cast<unsigned>(grid), 32 * BWD_WARPS, smem, s>>>(a, o);
  if (launched() != BDH_OK) return BDH_ERR_LAUNCH;
  const int NP = 4 * G;
  const long long rows = static_cast<long long>(d.B) * d.T;
  if ((rows * 2 * NP + 255) / 256 > 0x7fffffffLL) return BDH_ERR_TOO_LARGE;
  selective_scan_bc_kernel<T><<<static_cast<unsigned>((rows * 2 * NP + 255) / 256), 256, 0, s>>>(o.bc, p.parts, rows, NP, d.N,
                                                                                              static_cast<T*>(out.dB), static_cast<T*>(out.dC));
  if (launched() != BDH_OK) return BDH_ERR_LAUNCH;
  const long long n = static_cast<long long>(d.D) * (NP + 2);
  selective_scan_params_kernel<<<static_cast<unsigned>((n + 255) / 256), 256, 0, s>>>(o.da, o.per_channel, d.B * p.segs, d.D, NP, d.N, out.dA,
                                                                                   out.dD, out.dbias);
  return launched();
}

template <typename F>
int by_fit(const BdhScanDesc& d, int size, const F& f) {
  if (packs_fit(d, size)) return f(std::integral_constant<int, PACKS>{});
  return d.N % 4 ? f(std::integral_constant<int, MIXED>{}) : f(std::integral_constant<int, ELEMENTS>{});
}

template <typename F>
int by_lanes(int G, const F& f) {
  switch (G) {
    case 2: return f(std::integral_constant<int, 2>{});
    case 4: return f(std::integral_constant<int, 4>{});
    case 8: return f(std::integral_constant<int, 8>{});
  }
  return f(std::integral_constant<int, 16>{});
}
}  // namespace

// Of one row type each: compiled in a file of their own (selective_scan_f32.cu, _f16.cu, _bf16.cu).
template <typename T>
int selective_scan_fwd_of(const BdhScanDesc& d, float* marks, float* scratch, cudaStream_t s) {
  const Plan p = fwd_plan(d);
  if (p.segs > 1 && scratch == nullptr) return BDH_ERR_ARGUMENT;
  return by_lanes(p.G, [&](auto g) {
    return by_fit(d, sizeof(T), [&](auto fit) {
      constexpr int G = decltype(g)::value, FIT = decltype(fit)::value;
      return p.CT == 2 ? fwd_launch<T, G, 2, FIT>(d, p, marks, scratch, s) : fwd_launch<T, G, 1, FIT>(d, p, marks, scratch, s);
    });
  });
}

template <typename T>
int selective_scan_bwd_of(const BdhScanDesc& d, const float* marks, float* scratch, float* dA, float* dD, float* dbias, void* dB, void* dC,
                          cudaStream_t s) {
  const Plan p = bwd_plan(d);
  ScanGrads o;
  float* seg = scratch;
  o.marks = marks;
  o.bc = seg + seg_floats(d, p);
  o.da = o.bc + bc_floats(d, p);
  o.per_channel = o.da + da_floats(d, p);
  const BwdOut out{dA, dD, dbias, dB, dC};
  return by_lanes(p.G, [&](auto g) {
    return by_fit(d, sizeof(T), [&](auto fit) { return bwd_launch<T, decltype(g)::value, decltype(fit)::value>(d, p, o, seg, out, s); });
  });
}

// One token. Bound by the states: 8 B N D bytes a stream.
template <typename T>
int selective_scan_step_of(const BdhScanDesc& d, const float* h, long long h_sb, float* out, long long out_sb, const unsigned char* active,
                           cudaStream_t s) {
  const int vec4 = d.N % 4 == 0 && h_sb % 4 == 0 && out_sb % 4 == 0 && multiple(h, 16) && multiple(out, 16);
  return by_lanes(lanes_for(d.N), [&](auto g) {
    constexpr int G = decltype(g)::value;
    const auto launch = [&](auto kernel, int R) {
      const long long blocks = (static_cast<long long>((d.B + R - 1) / R) * d.D * G + STEP_THREADS - 1) / STEP_THREADS;
      if (blocks > 0x7fffffffLL) return static_cast<int>(BDH_ERR_TOO_LARGE);
      kernel<<<static_cast<unsigned>(blocks), STEP_THREADS, 0, s>>>(d, h, h_sb, out, out_sb, active, vec4);
      return launched();
    };
    // four streams a lane group while that still gives every SM a few blocks
    if (static_cast<long long>(d.B) * d.D * G >= 4LL * 148 * 4 * STEP_THREADS) return launch(selective_scan_step_kernel<T, G, 4>, 4);
    return launch(selective_scan_step_kernel<T, G, 1>, 1);
  });
}

#define BDH_SCAN_OF(EXTERN, T)                                                                                                          \
  EXTERN template int selective_scan_fwd_of<T>(const BdhScanDesc&, float*, float*, cudaStream_t);                                       \
  EXTERN template int selective_scan_bwd_of<T>(const BdhScanDesc&, const float*, float*, float*, float*, float*, void*, void*,         \
                                               cudaStream_t);                                                                           \
  EXTERN template int selective_scan_step_of<T>(const BdhScanDesc&, const float*, long long, float*, long long, const unsigned char*,   \
                                                cudaStream_t);

}  // namespace bdh
