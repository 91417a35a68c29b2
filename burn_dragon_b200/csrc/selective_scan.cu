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
// that h stays in registers along time and a warp holds 32 * 4 * CT states. Sums over states go over the G lanes, sums
// over channels over the 32 / G others, both by halving exchanges (n values over n lanes cost n - 1 shuffles and leave
// one sum in each lane). Time runs in tiles of 16 steps: a block fetches the next tile into registers while it works on
// the present one, whose steps (dt', dt' u) and rows of B and C lie in shared memory as fp32.
// Long sequences with too few channels to fill the GPU are cut into segments: one launch computes every segment's
// state from zero and its total step, the next starts each segment from the combination of those before it.
// Backward: the forward pass leaves h at every tile's start; a tile's states are computed again from there into shared
// memory and walked through in reverse. States, sums and gradients are fp32; sums over channel blocks, segments
// and sequences are made from partial sums in a fixed order (no atomics: two runs give the same bits).
#include "bdh_kernels.h"
#include "element_io.cuh"

#include <type_traits>

namespace bdh {
namespace {

constexpr int LT = 16;                 // steps per tile
constexpr int WARPS = 4;
constexpr int NT = 32 * WARPS;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

struct ScanArgs {
  BdhScanDesc d;
  Lengths len;
  int tiles, per_seg, segs;            // tiles per sequence, per segment; segments
  int vec, vec_bc;                     // rows can be moved in 16-byte packs; rows of B and C in packs of 4
  const float* seg_state;              // [B][segs][D][NP]: states of the segments from zero (forward or reverse)
  const float* seg_dt;                 // [B][segs][D]: their total steps
};

// ---- two fp32 operations in one instruction ------------------------------------------------------------
using f2 = unsigned long long;
__device__ __forceinline__ f2 pack2(float x, float y) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void unpack2(f2 v, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
  f2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
  f2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ f2 ex2x2(f2 v) {
  float x, y;
  unpack2(v, x, y);
  return pack2(ex2(x), ex2(y));
}
__device__ __forceinline__ float sum2(f2 v) {
  float x, y;
  unpack2(v, x, y);
  return x + y;
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

__device__ __forceinline__ float step_of(float raw, int softplus) { return softplus ? (raw > 20.f ? raw : log1pf(expf(raw))) : raw; }
__device__ __forceinline__ float step_slope(float raw, int softplus) { return softplus && raw <= 20.f ? sigmoid_f32(raw) : 1.f; }

// V adjacent channels of one row; channels behind D read as 0
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_row(const T* p, int c, int D, int vec) {
  Pack<T, V> r;
  if (vec) {
    if (c < D) r.load(p + c); else r.zero();
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) r.e[i] = c + i < D ? p[c + i] : elem_from_float<T>(0.f);
  }
  return r;
}
template <typename T, int V>
__device__ __forceinline__ void store_row(T* p, int c, int D, int vec, const Pack<T, V>& r) {
  if (vec) {
    if (c < D) r.store(p + c);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (c + i < D) p[c + i] = r.e[i];
  }
}

template <typename T, int G, int CT>
struct Shape {
  static constexpr int NP = 4 * G;
  static constexpr int LANES = 32 / G;                 // channel lanes of a warp
  static constexpr int CB = WARPS * LANES * CT;        // channels of a block
  static constexpr int V = 16 / sizeof(T);
  static constexpr int ROWV = CB / V;                  // packs of a row of the tile
  static constexpr int NVEC = (LT * ROWV + NT - 1) / NT;
  static constexpr int BCV = LT * G;                   // packs of 4 of a tile of B (or C)
  static constexpr int NBC = (2 * BCV + NT - 1) / NT;
  static_assert(ROWV >= 1 && NT % ROWV == 0, "a thread keeps its channels from pack to pack");
};

// One tile of the three row tensors and of B and C on its way from memory
template <typename T, int G, int CT, bool DY>
struct Tile {
  using S = Shape<T, G, CT>;
  Pack<T, S::V> u[S::NVEC], dt[S::NVEC], dy[DY ? S::NVEC : 1];
  Pack<T, 4> bc[S::NBC];

  // rows t0 .. t0 + LT that are not before `len`; what lies behind reads as 0
  __device__ __forceinline__ void load(const ScanArgs& a, int b, int c0, int t0, int len) {
    const BdhScanDesc& d = a.d;
#pragma unroll
    for (int i = 0; i < S::NVEC; ++i) {
      const int v = threadIdx.x + i * NT, t = t0 + v / S::ROWV, c = c0 + (v % S::ROWV) * S::V;
      if (v < LT * S::ROWV && t < len) {
        u[i] = load_row<T, S::V>(static_cast<const T*>(d.u) + b * d.u_sb + t * d.u_st, c, d.D, a.vec);
        dt[i] = load_row<T, S::V>(static_cast<const T*>(d.dt) + b * d.dt_sb + t * d.dt_st, c, d.D, a.vec);
        if constexpr (DY) dy[i] = load_row<T, S::V>(static_cast<const T*>(d.dy) + b * d.dy_sb + t * d.dy_st, c, d.D, a.vec);
      } else {
        u[i].zero();
        dt[i].zero();
        if constexpr (DY) dy[i].zero();
      }
    }
#pragma unroll
    for (int i = 0; i < S::NBC; ++i) {
      const int v = threadIdx.x + i * NT, w = v % S::BCV, t = t0 + w / G;
      if (v < 2 * S::BCV && t < len) {
        const bool is_c = v >= S::BCV;
        const T* p = is_c ? static_cast<const T*>(d.C_) + b * d.c_sb + t * d.c_st : static_cast<const T*>(d.B_) + b * d.b_sb + t * d.b_st;
        bc[i] = load_row<T, 4>(p, (w % G) * 4, d.N, a.vec_bc);
      } else {
        bc[i].zero();
      }
    }
  }
};

// What a tile's compute loop reads
template <typename T, int G, int CT, bool DY>
struct Shared {
  using S = Shape<T, G, CT>;
  float2 step[LT][S::CB];              // dt', dt' u
  float dy[DY ? LT : 1][DY ? S::CB : 4];
  float B[LT][S::NP], C[LT][S::NP];
  float bias[S::CB], skip[S::CB];

  __device__ __forceinline__ void params(const ScanArgs& a, int c0) {
    for (int i = threadIdx.x; i < S::CB; i += NT) {
      bias[i] = (a.d.dt_bias && c0 + i < a.d.D) ? a.d.dt_bias[c0 + i] : 0.f;
      skip[i] = (a.d.skip && c0 + i < a.d.D) ? a.d.skip[c0 + i] : 0.f;
    }
  }
  // channels behind D and rows behind `len` get dt' = 0: their states stay as they are
  __device__ __forceinline__ void put(const ScanArgs& a, const Tile<T, G, CT, DY>& x, int c0, int t0, int len) {
#pragma unroll
    for (int i = 0; i < S::NVEC; ++i) {
      const int v = threadIdx.x + i * NT, t = v / S::ROWV, c = (v % S::ROWV) * S::V;
      if (v >= LT * S::ROWV) break;
#pragma unroll
      for (int j = 0; j < S::V; ++j) {
        const bool in = t0 + t < len && c0 + c + j < a.d.D;
        const float s = in ? step_of(x.dt[i][j] + bias[c + j], a.d.softplus) : 0.f;
        step[t][c + j] = make_float2(s, in ? s * x.u[i][j] : 0.f);
        if constexpr (DY) dy[t][c + j] = x.dy[i][j];
      }
    }
#pragma unroll
    for (int i = 0; i < S::NBC; ++i) {
      const int v = threadIdx.x + i * NT, w = v % S::BCV;
      if (v >= 2 * S::BCV) break;
      float* p = v >= S::BCV ? &C[w / G][(w % G) * 4] : &B[w / G][(w % G) * 4];
#pragma unroll
      for (int j = 0; j < 4; ++j) p[j] = x.bc[i][j];
    }
  }
};

__device__ __forceinline__ void load4(const float* p, f2& x, f2& y) {
  const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(p);
  x = v.x;
  y = v.y;
}

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

template <int G, int CT>
struct Place {                         // which states of which channels a lane holds
  int lane, ng, cl, n0;
  __device__ __forceinline__ Place() {
    lane = threadIdx.x & 31;
    ng = lane % G;
    cl = ((threadIdx.x >> 5) * (32 / G) + lane / G) * CT;              // first channel, in the block
    n0 = 4 * ng;
  }
};

// A2 = A log2(e); 0 for padding
template <int CT>
__device__ __forceinline__ void load_a(const BdhScanDesc& d, int c, int n0, f2 (&A2)[CT][2]) {
#pragma unroll
  for (int k = 0; k < CT; ++k) {
    load_state(d.A, c + k, n0, d, A2[k]);
    const f2 s = pack2(LOG2E, LOG2E);
    A2[k][0] = mul2(A2[k][0], s);
    A2[k][1] = mul2(A2[k][1], s);
  }
}

// The state a segment starts from: `h` (the sequence's own) carried through the segments before it, in order; in reverse
// through those behind it.
template <int CT, int NP>
__device__ __forceinline__ void carry(const ScanArgs& a, int b, int from, int to, int by, int c, int n0, const f2 (&A2)[CT][2], f2 (&h)[CT][2]) {
  for (int s = from; s != to; s += by) {
#pragma unroll
    for (int k = 0; k < CT; ++k) {
      if (c + k >= a.d.D) continue;
      const long long at = (static_cast<long long>(b) * a.segs + s) * a.d.D + c + k;
      const float dt = a.seg_dt[at];
      const f2 dt2 = pack2(dt, dt);
      f2 s0, s1;
      load4(a.seg_state + at * NP + n0, s0, s1);
      h[k][0] = fma2(ex2x2(mul2(dt2, A2[k][0])), h[k][0], s0);
      h[k][1] = fma2(ex2x2(mul2(dt2, A2[k][1])), h[k][1], s1);
    }
  }
}

template <int CT>
__device__ __forceinline__ void load_steps(const float2* p, f2 (&dt)[CT], f2 (&du)[CT]) {
  if constexpr (CT == 2) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    dt[0] = pack2(v.x, v.x); du[0] = pack2(v.y, v.y);
    dt[1] = pack2(v.z, v.z); du[1] = pack2(v.w, v.w);
  } else {
    dt[0] = pack2(p->x, p->x);
    du[0] = pack2(p->y, p->y);
  }
}

struct Where {
  int cb, b, seg;
};
__device__ __forceinline__ Where where(const ScanArgs& a, int blocks) {
  Where w;
  w.cb = blockIdx.x % blocks;
  const int bs = blockIdx.x / blocks;
  w.b = bs / a.segs;
  w.seg = bs % a.segs;
  return w;
}

// ---- forward -----------------------------------------------------------------------------------------
template <typename T, int G, int CT>
__global__ void __launch_bounds__(NT) selective_scan_fwd_kernel(const ScanArgs a, int blocks, float* marks) {
  using S = Shape<T, G, CT>;
  __shared__ __align__(16) Shared<T, G, CT, false> sh;
  __shared__ float ys[LT][S::CB];
  const BdhScanDesc& d = a.d;
  const Where w = where(a, blocks);
  const Place<G, CT> me;
  const int c0 = w.cb * S::CB, c = c0 + me.cl;
  const int len = a.len.get(w.b, d.T);
  f2 A2[CT][2], h[CT][2];
  load_a<CT>(d, c, me.n0, A2);
#pragma unroll
  for (int k = 0; k < CT; ++k)
    load_state(d.h0 ? d.h0 + static_cast<long long>(w.b) * d.D * d.N : nullptr, c + k, me.n0, d, h[k]);
  carry<CT, S::NP>(a, w.b, 0, w.seg, 1, c, me.n0, A2, h);
  sh.params(a, c0);
  const int first = w.seg * a.per_seg, last = min(first + a.per_seg, a.tiles);
  Tile<T, G, CT, false> x;
  x.load(a, w.b, c0, first * LT, len);
  __syncthreads();
  for (int tile = first; tile < last; ++tile) {
    const int t0 = tile * LT;
    const bool any = t0 < len;                           // (the same for the whole block)
    if (any) sh.put(a, x, c0, t0, len);
    Pack<T, S::V> ut[S::NVEC];
#pragma unroll
    for (int i = 0; i < S::NVEC; ++i) ut[i] = x.u[i];
    __syncthreads();
    if (tile + 1 < last) x.load(a, w.b, c0, t0 + LT, len);
    if (any) {
      if (marks != nullptr)
#pragma unroll
        for (int k = 0; k < CT; ++k)
          if (c + k < d.D)
            *reinterpret_cast<ulonglong2*>(marks + ((static_cast<long long>(w.b) * a.tiles + tile) * d.D + c + k) * S::NP + me.n0) =
                make_ulonglong2(h[k][0], h[k][1]);
#pragma unroll
      for (int t4 = 0; t4 < LT; t4 += 4) {
        float v[4 * CT];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          const int t = t4 + s;
          f2 dt[CT], du[CT], b0, b1, k0, k1;
          load_steps<CT>(&sh.step[t][me.cl], dt, du);
          load4(&sh.B[t][me.n0], b0, b1);
          load4(&sh.C[t][me.n0], k0, k1);
#pragma unroll
          for (int k = 0; k < CT; ++k) {
            h[k][0] = fma2(ex2x2(mul2(dt[k], A2[k][0])), h[k][0], mul2(du[k], b0));
            h[k][1] = fma2(ex2x2(mul2(dt[k], A2[k][1])), h[k][1], mul2(du[k], b1));
            v[s * CT + k] = sum2(fma2(k1, h[k][1], mul2(k0, h[k][0])));
          }
        }
        int at;
        bool once;
        sum_over<4 * CT, G, 1>(v, me.lane, at, once);
        constexpr int LEFT = 4 * CT / G > 1 ? 4 * CT / G : 1;
        if (once)
#pragma unroll
          for (int i = 0; i < LEFT; ++i) ys[t4 + (at + i) / CT][me.cl + (at + i) % CT] = v[i];
      }
    }
    __syncthreads();
    if (d.y != nullptr) {
#pragma unroll
      for (int i = 0; i < S::NVEC; ++i) {
        const int v = threadIdx.x + i * NT, t = v / S::ROWV, cc = (v % S::ROWV) * S::V;
        if (v >= LT * S::ROWV || t0 + t >= d.T) break;
        Pack<T, S::V> o;
#pragma unroll
        for (int j = 0; j < S::V; ++j) o.set(j, t0 + t < len ? fmaf(sh.skip[cc + j], ut[i][j], ys[t][cc + j]) : 0.f);
        store_row<T, S::V>(static_cast<T*>(d.y) + (static_cast<long long>(w.b) * d.T + t0 + t) * d.D, c0 + cc, d.D, a.vec, o);
      }
    }
  }
  if (w.seg == a.segs - 1)
#pragma unroll
    for (int k = 0; k < CT; ++k) store_state(d.hT + static_cast<long long>(w.b) * d.D * d.N, c + k, me.n0, d, h[k]);
}

// States of the segments from zero: h_t = a_t h_{t-1} + dt' u B_t, or in reverse r_t = a_t (r_{t+1} + dy_t C_t); and the
// sum of the segment's steps.
template <typename T, int G, int CT, bool REV>
__global__ void __launch_bounds__(NT) selective_scan_sweep_kernel(const ScanArgs a, int blocks, float* seg_state, float* seg_dt) {
  using S = Shape<T, G, CT>;
  __shared__ __align__(16) Shared<T, G, CT, REV> sh;
  const BdhScanDesc& d = a.d;
  const Where w = where(a, blocks);
  const Place<G, CT> me;
  const int c0 = w.cb * S::CB, c = c0 + me.cl;
  const int len = a.len.get(w.b, d.T);
  f2 A2[CT][2], h[CT][2];
  float total[CT];
  load_a<CT>(d, c, me.n0, A2);
#pragma unroll
  for (int k = 0; k < CT; ++k) {
    h[k][0] = h[k][1] = pack2(0.f, 0.f);
    total[k] = 0.f;
  }
  sh.params(a, c0);
  const int first = w.seg * a.per_seg, end = min(min(first + a.per_seg, a.tiles), (len + LT - 1) / LT);
  const int n = end - first;
  Tile<T, G, CT, REV> x;
  if (n > 0) x.load(a, w.b, c0, (REV ? end - 1 : first) * LT, len);
  __syncthreads();
  for (int i = 0; i < n; ++i) {
    const int t0 = (REV ? end - 1 - i : first + i) * LT;
    sh.put(a, x, c0, t0, len);
    __syncthreads();
    if (i + 1 < n) x.load(a, w.b, c0, REV ? t0 - LT : t0 + LT, len);
#pragma unroll
    for (int s = 0; s < LT; ++s) {
      const int t = REV ? LT - 1 - s : s;
      f2 dt[CT], du[CT], b0, b1;
      load_steps<CT>(&sh.step[t][me.cl], dt, du);
      load4(REV ? &sh.C[t][me.n0] : &sh.B[t][me.n0], b0, b1);
#pragma unroll
      for (int k = 0; k < CT; ++k) {
        float one, same;
        unpack2(dt[k], one, same);
        total[k] += one;
        const f2 e0 = ex2x2(mul2(dt[k], A2[k][0])), e1 = ex2x2(mul2(dt[k], A2[k][1]));
        if constexpr (REV) {
          const float g = sh.dy[t][me.cl + k];
          const f2 g2 = pack2(g, g);
          h[k][0] = mul2(e0, fma2(g2, b0, h[k][0]));
          h[k][1] = mul2(e1, fma2(g2, b1, h[k][1]));
        } else {
          h[k][0] = fma2(e0, h[k][0], mul2(du[k], b0));
          h[k][1] = fma2(e1, h[k][1], mul2(du[k], b1));
        }
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int k = 0; k < CT; ++k)
    if (c + k < d.D) {
      const long long at = (static_cast<long long>(w.b) * a.segs + w.seg) * d.D + c + k;
      *reinterpret_cast<ulonglong2*>(seg_state + at * S::NP + me.n0) = make_ulonglong2(h[k][0], h[k][1]);
      if (me.ng == 0) seg_dt[at] = total[k];
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
struct BwdShared {
  using S = Shape<T, G, CT>;
  Shared<T, G, CT, true> in;
  float2 out[LT][S::CB];               // sum g B, log2(e) sum A q
  float bc[WARPS][LT][2 * S::NP];      // the warps' sums over their channels
  ulonglong2 h[LT][CT][NT];            // h_{t-1}, each lane its own
};

template <typename T, int G, int CT>
__global__ void __launch_bounds__(NT) selective_scan_bwd_kernel(const ScanArgs a, int blocks, const ScanGrads o) {
  using S = Shape<T, G, CT>;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  BwdShared<T, G, CT>& sh = *reinterpret_cast<BwdShared<T, G, CT>*>(smem_raw);
  const BdhScanDesc& d = a.d;
  const Where w = where(a, blocks);
  const Place<G, CT> me;
  const int warp = threadIdx.x >> 5;
  const int c0 = w.cb * S::CB, c = c0 + me.cl;
  const int len = a.len.get(w.b, d.T);
  f2 A2[CT][2], r[CT][2], da[CT][2];
  load_a<CT>(d, c, me.n0, A2);
#pragma unroll
  for (int k = 0; k < CT; ++k) {
    load_state(d.dhT ? d.dhT + static_cast<long long>(w.b) * d.D * d.N : nullptr, c + k, me.n0, d, r[k]);
    da[k][0] = da[k][1] = pack2(0.f, 0.f);
  }
  carry<CT, S::NP>(a, w.b, a.segs - 1, w.seg, -1, c, me.n0, A2, r);
  sh.in.params(a, c0);
  float sum_skip[S::V], sum_bias[S::V];                  // this thread's channels: the same in every pack
#pragma unroll
  for (int j = 0; j < S::V; ++j) sum_skip[j] = sum_bias[j] = 0.f;
  const int first = w.seg * a.per_seg, last = min(first + a.per_seg, a.tiles);
  Tile<T, G, CT, true> x;
  x.load(a, w.b, c0, (last - 1) * LT, len);
  __syncthreads();
  for (int tile = last - 1; tile >= first; --tile) {
    const int t0 = tile * LT;
    const bool any = t0 < len;
    f2 h[CT][2];
    Tile<T, G, CT, true> now = x;
    if (any) {
      sh.in.put(a, x, c0, t0, len);
#pragma unroll
      for (int k = 0; k < CT; ++k) {
        h[k][0] = h[k][1] = pack2(0.f, 0.f);
        if (c + k < d.D)
          load4(o.marks + ((static_cast<long long>(w.b) * a.tiles + tile) * d.D + c + k) * S::NP + me.n0, h[k][0], h[k][1]);
      }
    }
    __syncthreads();
    if (tile > first) x.load(a, w.b, c0, t0 - LT, len);
    if (any) {
#pragma unroll
      for (int t = 0; t < LT; ++t) {
        f2 dt[CT], du[CT], b0, b1;
        load_steps<CT>(&sh.in.step[t][me.cl], dt, du);
        load4(&sh.in.B[t][me.n0], b0, b1);
#pragma unroll
        for (int k = 0; k < CT; ++k) {
          sh.h[t][k][threadIdx.x] = make_ulonglong2(h[k][0], h[k][1]);
          h[k][0] = fma2(ex2x2(mul2(dt[k], A2[k][0])), h[k][0], mul2(du[k], b0));
          h[k][1] = fma2(ex2x2(mul2(dt[k], A2[k][1])), h[k][1], mul2(du[k], b1));
        }
      }
#pragma unroll 4
      for (int t = LT - 1; t >= 0; --t) {
        f2 dt[CT], du[CT], b0, b1, k0, k1;
        load_steps<CT>(&sh.in.step[t][me.cl], dt, du);
        load4(&sh.in.B[t][me.n0], b0, b1);
        load4(&sh.in.C[t][me.n0], k0, k1);
        f2 sb0, sb1, sc0, sc1;
        float nv[2 * CT];
#pragma unroll
        for (int k = 0; k < CT; ++k) {
          const float gy = sh.in.dy[t][me.cl + k];
          const f2 gy2 = pack2(gy, gy);
          const f2 g0 = fma2(gy2, k0, r[k][0]), g1 = fma2(gy2, k1, r[k][1]);
          const ulonglong2 hp = sh.h[t][k][threadIdx.x];
          if (k == 0) {
            sb0 = mul2(g0, du[k]); sb1 = mul2(g1, du[k]);
            sc0 = mul2(gy2, h[k][0]); sc1 = mul2(gy2, h[k][1]);
          } else {
            sb0 = fma2(g0, du[k], sb0); sb1 = fma2(g1, du[k], sb1);
            sc0 = fma2(gy2, h[k][0], sc0); sc1 = fma2(gy2, h[k][1], sc1);
          }
          r[k][0] = mul2(ex2x2(mul2(dt[k], A2[k][0])), g0);
          r[k][1] = mul2(ex2x2(mul2(dt[k], A2[k][1])), g1);
          const f2 q0 = mul2(r[k][0], hp.x), q1 = mul2(r[k][1], hp.y);
          da[k][0] = fma2(dt[k], q0, da[k][0]);
          da[k][1] = fma2(dt[k], q1, da[k][1]);
          nv[2 * k] = sum2(fma2(g1, b1, mul2(g0, b0)));
          nv[2 * k + 1] = sum2(fma2(A2[k][1], q1, mul2(A2[k][0], q0)));
          h[k][0] = hp.x;
          h[k][1] = hp.y;
        }
        int at;
        bool once;
        sum_over<2 * CT, G, 1>(nv, me.lane, at, once);
        constexpr int NLEFT = 2 * CT / G > 1 ? 2 * CT / G : 1;
        if (once)
#pragma unroll
          for (int i = 0; i < NLEFT; ++i) reinterpret_cast<float*>(&sh.out[t][me.cl])[at + i] = nv[i];
        float cv[8];                                     // dB of the 4 states, then dC
        unpack2(sb0, cv[0], cv[1]);
        unpack2(sb1, cv[2], cv[3]);
        unpack2(sc0, cv[4], cv[5]);
        unpack2(sc1, cv[6], cv[7]);
        sum_over<8, S::LANES, G>(cv, me.lane, at, once);
        constexpr int CLEFT = 8 / S::LANES > 1 ? 8 / S::LANES : 1;
        if (once)
#pragma unroll
          for (int i = 0; i < CLEFT; ++i) sh.bc[warp][t][(at + i) / 4 * S::NP + me.n0 + (at + i) % 4] = cv[i];
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < S::NVEC; ++i) {
      const int v = threadIdx.x + i * NT, t = v / S::ROWV, cc = (v % S::ROWV) * S::V;
      if (v >= LT * S::ROWV || t0 + t >= d.T) break;
      const bool in = t0 + t < len;
      Pack<T, S::V> pu, pd;
#pragma unroll
      for (int j = 0; j < S::V; ++j) {
        float du = 0.f, dd = 0.f;
        if (in) {
          const float2 s = sh.out[t][cc + j];
          const float gy = now.dy[i][j], uu = now.u[i][j];
          du = fmaf(sh.in.step[t][cc + j].x, s.x, sh.in.skip[cc + j] * gy);
          dd = fmaf(uu, s.x, LN2 * s.y) * step_slope(now.dt[i][j] + sh.in.bias[cc + j], d.softplus);
          sum_skip[j] = fmaf(gy, uu, sum_skip[j]);
          sum_bias[j] += dd;
        }
        pu.set(j, du);
        pd.set(j, dd);
      }
      const long long at = (static_cast<long long>(w.b) * d.T + t0 + t) * d.D;
      store_row<T, S::V>(static_cast<T*>(d.du) + at, c0 + cc, d.D, a.vec, pu);
      store_row<T, S::V>(static_cast<T*>(d.ddt) + at, c0 + cc, d.D, a.vec, pd);
    }
    for (int i = threadIdx.x; i < LT * 2 * S::NP; i += NT) {
      const int t = i / (2 * S::NP), n = i % (2 * S::NP);
      if (t0 + t >= d.T) break;
      float s = 0.f;
      if (any)
#pragma unroll
        for (int k = 0; k < WARPS; ++k) s += sh.bc[k][t][n];
      o.bc[((static_cast<long long>(w.cb) * d.B + w.b) * d.T + t0 + t) * (2 * S::NP) + n] = s;
    }
    __syncthreads();
  }
  const long long seg = static_cast<long long>(w.b) * a.segs + w.seg;
#pragma unroll
  for (int k = 0; k < CT; ++k) {
    if (c + k < d.D) *reinterpret_cast<ulonglong2*>(o.da + (seg * d.D + c + k) * S::NP + me.n0) = make_ulonglong2(da[k][0], da[k][1]);
    if (w.seg == 0 && d.dh0 != nullptr) store_state(d.dh0 + static_cast<long long>(w.b) * d.D * d.N, c + k, me.n0, d, r[k]);
  }
  // the threads that share channels add their sums up, in order
  float* buf = reinterpret_cast<float*>(smem_raw);       // [2][NT][V]
#pragma unroll
  for (int j = 0; j < S::V; ++j) {
    buf[threadIdx.x * S::V + j] = sum_skip[j];
    buf[(NT + threadIdx.x) * S::V + j] = sum_bias[j];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * S::CB; i += NT) {
    const int what = i / S::CB, cc = i % S::CB;
    float s = 0.f;
    for (int k = cc / S::V; k < NT; k += S::ROWV) s += buf[(what * NT + k) * S::V + cc % S::V];
    if (c0 + cc < d.D) o.per_channel[(static_cast<long long>(what) * d.B * a.segs + seg) * d.D + c0 + cc] = s;
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
// Bound by the states: 4 B N D read and written per stream.
template <typename T, int G>
__global__ void __launch_bounds__(NT) selective_scan_step_kernel(const BdhScanDesc d, const float* h, long long h_sb, float* out, long long out_sb,
                                                                 const unsigned char* active, int vec4) {
  const int lane = threadIdx.x & 31, ng = lane % G, n0 = 4 * ng;
  const long long i = (static_cast<long long>(blockIdx.x) * NT + threadIdx.x) / G;
  const int b = static_cast<int>(i / d.D), c = static_cast<int>(i % d.D);
  const bool live = b < d.B, on = live && (active == nullptr || active[b] != 0);
  float v[4] = {0.f, 0.f, 0.f, 0.f}, y = 0.f, u = 0.f;
  const long long at = static_cast<long long>(c) * d.N + n0;
  if (live) {
    const float* hp = h + b * h_sb + at;
    if (vec4 && n0 < d.N) {
      const float4 t = *reinterpret_cast<const float4*>(hp);
      v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = n0 + j < d.N ? hp[j] : 0.f;
    }
    if (on) {
      u = elem_to_float<T>(static_cast<const T*>(d.u)[b * d.u_sb + c]);
      const float raw = elem_to_float<T>(static_cast<const T*>(d.dt)[b * d.dt_sb + c]) + (d.dt_bias ? d.dt_bias[c] : 0.f);
      const float dt = step_of(raw, d.softplus), du = dt * u;
      const T* bp = static_cast<const T*>(d.B_) + b * d.b_sb + n0;
      const T* cp = static_cast<const T*>(d.C_) + b * d.c_sb + n0;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n0 + j < d.N) {
          v[j] = fmaf(ex2(dt * (d.A[at + j] * LOG2E)), v[j], du * elem_to_float<T>(bp[j]));
          y = fmaf(elem_to_float<T>(cp[j]), v[j], y);
        }
    }
  }
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
  if (!live) return;
  float* op = out + b * out_sb + at;
  if (on || op != h + b * h_sb + at) {
    if (vec4 && n0 < d.N) {
      *reinterpret_cast<float4*>(op) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n0 + j < d.N) op[j] = v[j];
    }
  }
  if (ng == 0)
    static_cast<T*>(d.y)[static_cast<long long>(b) * d.D + c] = elem_from_float<T>(on ? fmaf(d.skip ? d.skip[c] : 0.f, u, y) : 0.f);
}

// ---- host --------------------------------------------------------------------------------------------
bool multiple(const void* p, long long bytes) { return reinterpret_cast<unsigned long long>(p) % bytes == 0; }

int checked(const BdhScanDesc& d) {
  if (d.dtype < 0 || d.dtype > 2 || d.B < 0 || d.T < 0 || d.D < 1 || d.N < 1 || d.N > 64) return BDH_ERR_ARGUMENT;
  return BDH_OK;
}

int lanes_for(int N) { return N <= 8 ? 2 : N <= 16 ? 4 : N <= 32 ? 8 : 16; }

// Channels a lane. Two halve the reads of B and C from shared memory; one gives twice the warps.
int channels_for(const BdhScanDesc& d) {
  const int cb = WARPS * 32 / lanes_for(d.N) * 2;
  const long long blocks = static_cast<long long>(d.B) * ((d.D + cb - 1) / cb);
  return blocks >= 2 * 148 ? 2 : 1;
}

struct Plan {
  int G, CT, CB, blocks, tiles, per_seg, segs;
};

// `blocks_wanted`: below it the sequence is cut (at most 64 ways, so that combining the pieces stays cheap)
Plan plan(const BdhScanDesc& d, int CT, int blocks_wanted) {
  Plan p;
  p.G = lanes_for(d.N);
  p.CT = CT;
  p.CB = WARPS * 32 / p.G * CT;
  p.blocks = (d.D + p.CB - 1) / p.CB;
  p.tiles = (d.T + LT - 1) / LT;
  const long long have = static_cast<long long>(d.B) * p.blocks;
  long long segs = have >= blocks_wanted ? 1 : (blocks_wanted + have - 1) / have;
  if (segs > 64) segs = 64;
  if (segs > p.tiles) segs = p.tiles > 0 ? p.tiles : 1;
  p.per_seg = static_cast<int>((p.tiles + segs - 1) / segs);
  if (p.per_seg < 1) p.per_seg = 1;
  p.segs = p.tiles > 0 ? (p.tiles + p.per_seg - 1) / p.per_seg : 1;
  return p;
}

Plan fwd_plan(const BdhScanDesc& d) {
  const int CT = channels_for(d);
  Plan p = plan(d, CT, 1);
  // cutting costs the exponentials a second time: worth it from a third of the GPU down
  if (static_cast<long long>(d.B) * p.blocks < 50) p = plan(d, CT, 148);
  return p;
}
Plan bwd_plan(const BdhScanDesc& d) { return plan(d, 2, 2 * 148); }

long long round4(long long n) { return (n + 3) / 4 * 4; }          // pieces of the scratch start on 16 bytes

long long seg_floats(const BdhScanDesc& d, const Plan& p) {
  return p.segs > 1 ? round4(static_cast<long long>(d.B) * p.segs * d.D * (4 * p.G + 1)) : 0;
}
long long bc_floats(const BdhScanDesc& d, const Plan& p) { return static_cast<long long>(p.blocks) * d.B * d.T * 8 * p.G; }
long long da_floats(const BdhScanDesc& d, const Plan& p) { return static_cast<long long>(d.B) * p.segs * d.D * 4 * p.G; }

ScanArgs args_for(const BdhScanDesc& d, const Plan& p, int size, const float* seg) {
  ScanArgs a;
  a.d = d;
  a.len = Lengths{d.lengths, d.lengths64};
  a.tiles = p.tiles; a.per_seg = p.per_seg; a.segs = p.segs;
  const int V = 16 / size;
  a.vec = d.D % V == 0;
  for (const void* q : {d.u, d.dt, d.dy, static_cast<const void*>(d.y), static_cast<const void*>(d.du), static_cast<const void*>(d.ddt)})
    a.vec = a.vec && multiple(q, 16);
  for (long long s : {d.u_sb, d.u_st, d.dt_sb, d.dt_st, d.dy_sb, d.dy_st}) a.vec = a.vec && s % V == 0;
  a.vec_bc = d.N % 4 == 0 && multiple(d.B_, 4 * size) && multiple(d.C_, 4 * size);
  for (long long s : {d.b_sb, d.b_st, d.c_sb, d.c_st}) a.vec_bc = a.vec_bc && s % 4 == 0;
  a.seg_state = seg;
  a.seg_dt = seg ? seg + static_cast<long long>(d.B) * p.segs * d.D * (4 * p.G) : nullptr;
  return a;
}

int launched() { return cudaGetLastError() == cudaSuccess ? BDH_OK : BDH_ERR_LAUNCH; }

long long grid_of(const BdhScanDesc& d, const Plan& p) { return static_cast<long long>(d.B) * p.segs * p.blocks; }

template <typename T, int G, int CT>
int fwd_launch(const BdhScanDesc& d, const Plan& p, float* marks, float* seg, cudaStream_t s) {
  const long long grid = grid_of(d, p);
  if (grid > 0x7fffffffLL) return BDH_ERR_TOO_LARGE;
  const ScanArgs a = args_for(d, p, sizeof(T), p.segs > 1 ? seg : nullptr);
  if (p.segs > 1) {
    selective_scan_sweep_kernel<T, G, CT, false><<<static_cast<unsigned>(grid), NT, 0, s>>>(a, p.blocks, seg, const_cast<float*>(a.seg_dt));
    if (launched() != BDH_OK) return BDH_ERR_LAUNCH;
  }
  selective_scan_fwd_kernel<T, G, CT><<<static_cast<unsigned>(grid), NT, 0, s>>>(a, p.blocks, marks);
  return launched();
}

template <typename T, int G, int CT>
int bwd_launch(const BdhScanDesc& d, const Plan& p, const ScanGrads& o, float* seg, float* dA, float* dD, float* dbias, void* dB, void* dC,
               cudaStream_t s) {
  const long long grid = grid_of(d, p);
  if (grid > 0x7fffffffLL) return BDH_ERR_TOO_LARGE;
  const ScanArgs a = args_for(d, p, sizeof(T), p.segs > 1 ? seg : nullptr);
  if (p.segs > 1) {
    selective_scan_sweep_kernel<T, G, CT, true><<<static_cast<unsigned>(grid), NT, 0, s>>>(a, p.blocks, seg, const_cast<float*>(a.seg_dt));
    if (launched() != BDH_OK) return BDH_ERR_LAUNCH;
  }
  auto kernel = selective_scan_bwd_kernel<T, G, CT>;
  const int smem = sizeof(BwdShared<T, G, CT>);
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return BDH_ERR_LAUNCH;
  kernel<<<static_cast<unsigned>(grid), NT, smem, s>>>(a, p.blocks, o);
  if (launched() != BDH_OK) return BDH_ERR_LAUNCH;
  const int NP = 4 * G;
  const long long rows = static_cast<long long>(d.B) * d.T;
  if ((rows * 2 * NP + 255) / 256 > 0x7fffffffLL) return BDH_ERR_TOO_LARGE;
  selective_scan_bc_kernel<T><<<static_cast<unsigned>((rows * 2 * NP + 255) / 256), 256, 0, s>>>(o.bc, p.blocks, rows, NP, d.N,
                                                                                              static_cast<T*>(dB), static_cast<T*>(dC));
  if (launched() != BDH_OK) return BDH_ERR_LAUNCH;
  const long long n = static_cast<long long>(d.D) * (NP + 2);
  selective_scan_params_kernel<<<static_cast<unsigned>((n + 255) / 256), 256, 0, s>>>(o.da, o.per_channel, d.B * p.segs, d.D, NP, d.N, dA, dD,
                                                                                   dbias);
  return launched();
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
template <typename F>
int by_type(int dtype, const F& f) {
  switch (dtype) {
    case BDH_F32: return f(float{});
    case BDH_F16: return f(__half{});
  }
  return f(__nv_bfloat16{});
}

}  // namespace
}  // namespace bdh

using namespace bdh;

extern "C" void bdh_selective_scan_sizes(const BdhScanDesc* d, long long* marks, long long* fwd_scratch, long long* bwd_scratch) {
  *marks = *fwd_scratch = *bwd_scratch = 0;
  if (checked(*d) != BDH_OK) return;
  const Plan f = fwd_plan(*d), b = bwd_plan(*d);
  const long long NP = 4 * f.G;
  *marks = static_cast<long long>(d->B) * f.tiles * d->D * NP;
  *fwd_scratch = seg_floats(*d, f);
  *bwd_scratch = seg_floats(*d, b) + bc_floats(*d, b) + da_floats(*d, b) + static_cast<long long>(d->B) * b.segs * d->D * 2;
}

extern "C" int bdh_selective_scan_fwd(const BdhScanDesc* d, float* marks, float* scratch, cudaStream_t s) {
  if (const int rc = checked(*d)) return rc;
  if (d->B == 0) return BDH_OK;
  if (d->T == 0) return BDH_ERR_ARGUMENT;
  const Plan p = fwd_plan(*d);
  if (p.segs > 1 && scratch == nullptr) return BDH_ERR_ARGUMENT;
  return by_type(d->dtype, [&](auto t) {
    return by_lanes(p.G, [&](auto g) {
      using T = decltype(t);
      constexpr int G = decltype(g)::value;
      return p.CT == 2 ? fwd_launch<T, G, 2>(*d, p, marks, scratch, s) : fwd_launch<T, G, 1>(*d, p, marks, scratch, s);
    });
  });
}

extern "C" int bdh_selective_scan_bwd(const BdhScanDesc* d, const float* marks, float* scratch, float* dA, float* dD, float* dbias, void* dB,
                                      void* dC, cudaStream_t s) {
  if (const int rc = checked(*d)) return rc;
  if (d->B == 0 || d->T == 0) return BDH_ERR_ARGUMENT;
  const Plan p = bwd_plan(*d);
  ScanGrads o;
  float* seg = scratch;
  o.marks = marks;
  o.bc = seg + seg_floats(*d, p);
  o.da = o.bc + bc_floats(*d, p);
  o.per_channel = o.da + da_floats(*d, p);
  return by_type(d->dtype, [&](auto t) {
    return by_lanes(p.G, [&](auto g) { return bwd_launch<decltype(t), decltype(g)::value, 2>(*d, p, o, seg, dA, dD, dbias, dB, dC, s); });
  });
}

extern "C" int bdh_selective_scan_step(const BdhScanDesc* d, const float* h, long long h_sb, float* out, long long out_sb,
                                       const unsigned char* active, cudaStream_t s) {
  if (const int rc = checked(*d)) return rc;
  if (d->B == 0) return BDH_OK;
  const int vec4 = d->N % 4 == 0 && h_sb % 4 == 0 && out_sb % 4 == 0 && multiple(h, 16) && multiple(out, 16);
  return by_type(d->dtype, [&](auto t) {
    return by_lanes(lanes_for(d->N), [&](auto g) {
      constexpr int G = decltype(g)::value;
      const long long blocks = (static_cast<long long>(d->B) * d->D * G + NT - 1) / NT;
      if (blocks > 0x7fffffffLL) return static_cast<int>(BDH_ERR_TOO_LARGE);
      selective_scan_step_kernel<decltype(t), G><<<static_cast<unsigned>(blocks), NT, 0, s>>>(*d, h, h_sb, out, out_sb, active, vec4);
      return launched();
    });
  });
}
