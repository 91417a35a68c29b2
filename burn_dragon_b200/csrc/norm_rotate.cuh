// RMS norm of every query and key head and its rotation, in one pass and in both directions:
//
//   r = 1 / sqrt(mean x^2 + eps);  v = x r w + b;  (o_2i, o_2i+1) = R(angle_i) (v_2i, v_2i+1) for the first P pairs
//   dv = R^T do;  db = sum dv;  dw = sum dv x r;  dx = r (w dv - x r mean(w dv x r));
//   d angle_i = sum over heads of v_2i dv_2i+1 - v_2i+1 dv_2i                     (a rotation keeps this cross product)
//
// The angle of a token's pair is given, or 2 pi frac(position * freq) with the product in 64 bits (a position of 10^6
// leaves 4 of 24 bits of the fraction in 32). Bound by memory: ~9 (forward) or ~13 operations an element against one
// tensor in and one out (two in, one out). G lanes hold one head's row, so x is read once. A thread stays with its
// token slot and its columns and goes through heads: sines and cosines are made once per token and block (one for
// each pair and head would cost more than the rest of the row) and stay in registers over the heads; a row's slot is
// refilled from the next token as soon as it has been unpacked, so that loads are always on their way. Heads come in
// groups of hr rows, each of q or of k alone, so that a weight's gradient stays in registers over all rows that share
// it. Sums are fp32, in a fixed order.
//
// Measured, 4 x 4096 tokens, 32 + 8 heads of 128, bf16: forward 89 us (0.58 of the copy rate), backward 158 us (0.49). The pairs' turns
// and conversions issue about 20 instructions a pair of elements, with a scheduler busy 60 and 49 % of the time: at five and
// three warps each they wait for the results of their own arithmetic and of shared memory. 64 tokens alone: 5 us.
#pragma once
#include "bdh_kernels.h"
#include "pair_math.cuh"

#include <cfloat>
#include <type_traits>

namespace bdh {
namespace {

constexpr int NT = 128;
// Blocks an SM: as many as run at once, in one round over the tokens. Registers for five and three (4 x 4096 tokens, 32 + 8 heads
// of 128, bf16, in one run: forward 87 us, backward 156 us; for four and two 90 and 191 us, for six and four, which spill, 125 and
// 203 us; two rounds of blocks 89 and 171 us). Rows of several packs a lane need more.
constexpr int FWD_BLOCKS = 5, BWD_BLOCKS = 3;

struct NormArgs {
  BdhNormRotateDesc d;
  Lengths len;
  int tokens;                // B * T
  int G, hr, TS;             // lanes per row; heads per group; tokens at once (TS * hr * G <= NT)
  int q_groups, groups, per_block, slices;     // groups of q; of q and k; of a block (blockIdx.y: the slice)
  float per_column;          // 1 / Dh
};

// This thread's place, and its rows of the token group that starts at `first`
template <typename T, int V, bool VEC, int NV>
struct Place {
  using Raw = typename Pack<T, V>::Raw;
  static constexpr int N = V / 2;
  int lane, ts, hl, g0, ng;  // lane of the row; token slot; head within a group; the slice's groups
  bool slot_ok;

  __device__ __forceinline__ Place(const NormArgs& a) {
    lane = threadIdx.x % a.G;
    const int slot = threadIdx.x / a.G;
    ts = slot / a.hr;
    hl = slot - ts * a.hr;
    slot_ok = ts < a.TS;
    g0 = blockIdx.y * a.per_block;
    ng = min(a.per_block, a.groups - g0);
  }
  __device__ __forceinline__ int column(const NormArgs& a, int n) const { return (n * a.G + lane) * V; }
  __device__ __forceinline__ bool key(const NormArgs& a, int u) const { return g0 + u >= a.q_groups; }
  // first head of the u-th group, in its tensor (the same for the block), and whether this thread has a row of it
  __device__ __forceinline__ int first_head(const NormArgs& a, int u) const { return (g0 + u - (key(a, u) ? a.q_groups : 0)) * a.hr; }
  __device__ __forceinline__ bool has(const NormArgs& a, int u) const {
    return slot_ok && u < ng && first_head(a, u) + hl < (key(a, u) ? a.d.Hk : a.d.Hq);
  }
};

// A token's rows: where this thread's first one lies in a strided input, and in a dense [tokens, heads, Dh] tensor; the
// u-th group's is as many heads on.
template <typename T, typename P>
struct Rows {
  const T *q, *k;
  long long q_dense, k_dense;
  __device__ __forceinline__ Rows(const NormArgs& a, const P& me, int b, int t) {
    const BdhNormRotateDesc& d = a.d;
    const long long at = static_cast<long long>(b) * d.T + t;
    q = static_cast<const T*>(d.q) + b * d.q_sb + t * d.q_st + me.hl * d.q_sh;
    k = static_cast<const T*>(d.k) + b * d.k_sb + t * d.k_st + me.hl * d.k_sh;
    q_dense = (at * d.Hq + me.hl) * d.Dh;
    k_dense = (at * d.Hk + me.hl) * d.Dh;
  }
  __device__ __forceinline__ const T* in(const NormArgs& a, const P& me, int u) const {
    const long long h = me.first_head(a, u);
    return me.key(a, u) ? k + h * a.d.k_sh : q + h * a.d.q_sh;
  }
  __device__ __forceinline__ long long dense(const NormArgs& a, const P& me, int u) const {
    return (me.key(a, u) ? k_dense : q_dense) + static_cast<long long>(me.first_head(a, u)) * a.d.Dh;
  }
};

struct Token {
  int b, t;
  bool live, in;             // it exists; it is not behind its sequence's length
};
__device__ __forceinline__ Token token_at(const NormArgs& a, long long i) {
  Token k;
  k.live = i < a.tokens;
  const int at = k.live ? static_cast<int>(i) : 0;
  k.b = at / a.d.T;
  k.t = at - k.b * a.d.T;
  k.in = k.live && k.t < a.len.get(k.b, a.d.T);
  return k;
}

// V elements from column c on, as they lie in memory; columns behind Dh read as 0
template <typename T, int V, bool VEC>
__device__ __forceinline__ typename Pack<T, V>::Raw load_cols(const T* p, int c, int Dh) {
  Pack<T, V> k;
  if constexpr (VEC) {
    if (c < Dh) return *reinterpret_cast<const typename Pack<T, V>::Raw*>(p + c);
    k.zero();
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) k.e[i] = c + i < Dh ? p[c + i] : elem_from_float<T>(0.f);
  }
  return *reinterpret_cast<const typename Pack<T, V>::Raw*>(&k);
}
template <typename T, int V, bool VEC>
__device__ __forceinline__ void store_cols(T* p, int c, int Dh, const f2 (&f)[V / 2]) {
  const typename Pack<T, V>::Raw raw = Pairs<T, V>::put(f);
  if constexpr (VEC) {
    if (c < Dh) *reinterpret_cast<typename Pack<T, V>::Raw*>(p + c) = raw;
  } else {
    const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (c + i < Dh) p[c + i] = e[i];
  }
}

__device__ __forceinline__ float group_sum(float v, int G) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    if (o < G) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// 1 / sqrt(x). The quick root takes a subnormal x for 0. With a normal eps there is none; SUB: there may be (2 % of a pass).
template <bool SUB>
__device__ __forceinline__ float rsqrt_of(float x) {
  if constexpr (SUB) return rsqrtf(x);
  float r;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// cs[s][i] = (cos, sin) of pair i of token first + s
__device__ __forceinline__ void fill_angles(const NormArgs& a, float2* cs, long long first) {
  const BdhNormRotateDesc& d = a.d;
  for (int item = threadIdx.x; item < a.TS * d.P; item += NT) {
    const int slot = item / d.P, i = item - slot * d.P;
    const Token k = token_at(a, first + slot);
    if (k.in) {                                                 // (an angle behind a length may be anything; no row uses it)
      float sn, c;
      if (d.angles != nullptr) {
        sincosf(d.angles[k.b * d.ang_sb + k.t * d.ang_st + i], &sn, &c);
      } else {
        const long long at = k.b * d.pos_sb + k.t * d.pos_st;
        const long long pos = d.positions == nullptr ? d.pos0 + k.t
                              : d.positions64 ? static_cast<const long long*>(d.positions)[at]
                                              : static_cast<long long>(static_cast<const int*>(d.positions)[at]);
        const double turns = static_cast<double>(pos) * static_cast<double>(d.freqs[2 * i]);
        sincospif(2.f * static_cast<float>(turns - floor(turns)), &sn, &c);
      }
      cs[item] = make_float2(c, sn);
    }
  }
}

// Weights and biases of a block's rows in shared memory: one row of Dh (padded to the lanes' columns) for each of q and k,
// or for each of the slice's heads
struct Weights {
  float *w, *b;
  int pitch, per_head;
  // packs of 4 columns of all lanes lie together, so that the lanes' loads of 16 bytes meet no bank twice
  template <int V>
  static __device__ __forceinline__ int place(int c, int G) {
    const int n = c / (G * V), lane = c / V % G, i = c % V;
    return (n * V + i / 4 * 4) * G + lane * 4 + i % 4;
  }
  template <int V>
  static __device__ __forceinline__ void load(const float* p, int row, int n, int lane, int G, f2 (&f)[V / 2]) {
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(p + row + (n * V + i) * G + lane * 4);
      f[i / 2] = v.x;
      f[i / 2 + 1] = v.y;
    }
  }
  template <int V>
  __device__ __forceinline__ void fill(const NormArgs& a, float* at, int pitch_, int rows, int g0) {
    const BdhNormRotateDesc& d = a.d;
    pitch = pitch_;
    per_head = d.per_head;
    w = at;
    b = at + rows * pitch;
    for (int i = threadIdx.x; i < rows * pitch; i += NT) {
      const int row = i / pitch, c = i - row * pitch;
      const bool key = per_head ? g0 + row / a.hr >= a.q_groups : row == 1;
      const int head = per_head ? (g0 + row / a.hr - (key ? a.q_groups : 0)) * a.hr + row % a.hr : 0;
      const bool ok = c < d.Dh && (!per_head || head < (key ? d.Hk : d.Hq));
      const float* pw = key ? d.k_weight : d.q_weight;
      const float* pb = key ? d.k_bias : d.q_bias;
      const int to = row * pitch + place<V>(c, a.G);
      w[to] = ok && pw != nullptr ? pw[static_cast<long long>(head) * d.Dh + c] : 1.f;
      b[to] = ok && pb != nullptr ? pb[static_cast<long long>(head) * d.Dh + c] : 0.f;
    }
  }
  __device__ __forceinline__ int row(const NormArgs& a, int u, int hl, bool key) const { return per_head ? u * a.hr + hl : key; }
};

// (x, y) turned by (cos, sin) = e
__device__ __forceinline__ f2 turn(f2 v, float2 e) {
  float x, y;
  unpack2(v, x, y);
  return pack2(x * e.x - y * e.y, fmaf(y, e.x, x * e.y));
}

template <typename T, int V, bool VEC, int NV, int U, bool SUB>
__global__ void __launch_bounds__(NT, NV == 1 ? FWD_BLOCKS : 2) norm_rotate_fwd_kernel(const NormArgs a, int w_rows) {
  using P = Place<T, V, VEC, NV>;
  using Raw = typename P::Raw;
  constexpr int N = P::N;
  extern __shared__ __align__(16) float smem[];
  const BdhNormRotateDesc& d = a.d;
  const P me(a);
  Weights wt;
  const int pitch = a.G * V * NV;
  wt.template fill<V>(a, smem, pitch, w_rows, me.g0);
  float2* cs = reinterpret_cast<float2*>(smem + 2 * w_rows * pitch);         // two sets: the tokens' now, and the next ones'
  const int cs_set = a.TS * d.P;
  Raw raw[U][NV];
  const auto load = [&](const Token& k, const Rows<T, P>& r, int u) {
    const int Dh = k.in && me.has(a, u) ? d.Dh : 0;
    const T* p = r.in(a, me, u);
#pragma unroll
    for (int n = 0; n < NV; ++n) raw[u][n] = load_cols<T, V, VEC>(p, me.column(a, n), Dh);
  };
  const long long stride = static_cast<long long>(gridDim.x) * a.TS;
  long long first = static_cast<long long>(blockIdx.x) * a.TS;
  Token now = token_at(a, first + me.ts);
  Rows<T, P> rows(a, me, now.b, now.t);
#pragma unroll
  for (int u = 0; u < U; ++u) load(now, rows, u);
  fill_angles(a, cs, first);
  __syncthreads();
  int set = 0;
  for (; first < a.tokens; first += stride) {
    const Token next = token_at(a, first + stride + me.ts);
    const Rows<T, P> next_rows(a, me, next.b, next.t);
    const float eps = now.in ? d.eps : 1.f;                     // (behind a length the row is 0, and d.eps may be)
    float2 e[NV][N];                                            // (0, 0) for a token behind its length: its rows become 0
#pragma unroll
    for (int n = 0; n < NV; ++n)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int pair = me.column(a, n) / 2 + i;
        e[n][i] = make_float2(now.in ? 1.f : 0.f, 0.f);
        if (now.in && me.slot_ok && pair < d.P) e[n][i] = cs[set * cs_set + me.ts * d.P + pair];
      }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u >= me.ng) break;                                    // (the same for the block)
      f2 x[NV][N], ss = both(0.f);
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        Pairs<T, V>::get(raw[u][n], x[n]);
#pragma unroll
        for (int i = 0; i < N; ++i) ss = fma2(x[n][i], x[n][i], ss);
      }
      load(next, next_rows, u);
      const float rs = rsqrt_of<SUB>(fmaf(group_sum(sum2(ss), a.G), a.per_column, eps));
      if (!now.live || !me.has(a, u)) continue;
      const bool key = me.key(a, u);
      T* o = static_cast<T*>(key ? d.k_out : d.q_out) + rows.dense(a, me, u);
      const int wrow = wt.row(a, u, me.hl, key) * pitch;
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        f2 w[N], b[N];
        wt.load<V>(wt.w, wrow, n, me.lane, a.G, w);
        wt.load<V>(wt.b, wrow, n, me.lane, a.G, b);
#pragma unroll
        for (int i = 0; i < N; ++i) x[n][i] = turn(fma2(mul2(x[n][i], both(rs)), w[i], b[i]), e[n][i]);
        store_cols<T, V, VEC>(o, me.column(a, n), d.Dh, x[n]);
      }
    }
    if (first + stride < a.tokens) fill_angles(a, cs + (set ^ 1) * cs_set, first + stride);
    __syncthreads();
    set ^= 1;
    now = next;
    rows = next_rows;
  }
}

// Shared memory: weights; two sets of angles; then (dang) the rows' cross products, or (at the end) the rows' sums for the
// weights. PER_HEAD: a sum for each of the thread's heads; else one for q and one for k. partial: [2 (weight, bias)]
// [lines][width], see norm_rotate_params_kernel.
template <typename T, int V, bool VEC, int NV, int U, bool PER_HEAD, bool BIAS, bool SUB>
__global__ void __launch_bounds__(NT, NV == 1 ? BWD_BLOCKS : 2) norm_rotate_bwd_kernel(const NormArgs a, int w_rows, float* partial, float* dang) {
  using P = Place<T, V, VEC, NV>;
  using Raw = typename P::Raw;
  constexpr int N = P::N, SUMS = PER_HEAD ? U : 2;
  extern __shared__ __align__(16) float smem[];
  const BdhNormRotateDesc& d = a.d;
  const P me(a);
  Weights wt;
  const int pitch = a.G * V * NV;
  wt.template fill<V>(a, smem, pitch, w_rows, me.g0);
  float2* cs = reinterpret_cast<float2*>(smem + 2 * w_rows * pitch);
  const int cs_set = a.TS * d.P, rows = a.TS * a.hr, slot = me.ts * a.hr + me.hl;
  float* rowbuf = reinterpret_cast<float*>(cs + 2 * cs_set);
  Raw rx[U][NV], rg[U][NV];
  const auto load = [&](const Token& k, const Rows<T, P>& r, int u) {
    const int Dh = k.in && me.has(a, u) ? d.Dh : 0;
    const T* p = r.in(a, me, u);
    const T* g = static_cast<const T*>(me.key(a, u) ? d.dk_out : d.dq_out) + r.dense(a, me, u);
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      rx[u][n] = load_cols<T, V, VEC>(p, me.column(a, n), Dh);
      rg[u][n] = load_cols<T, V, VEC>(g, me.column(a, n), Dh);
    }
  };
  f2 gw[SUMS][NV][N], gb[BIAS ? SUMS : 1][NV][N];
#pragma unroll
  for (int k = 0; k < SUMS; ++k)
#pragma unroll
    for (int n = 0; n < NV; ++n)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        gw[k][n][i] = both(0.f);
        if (BIAS) gb[BIAS ? k : 0][n][i] = both(0.f);
      }
  const long long stride = static_cast<long long>(gridDim.x) * a.TS;
  long long first = static_cast<long long>(blockIdx.x) * a.TS;
  Token now = token_at(a, first + me.ts);
  Rows<T, P> at(a, me, now.b, now.t);
#pragma unroll
  for (int u = 0; u < U; ++u) load(now, at, u);
  fill_angles(a, cs, first);
  __syncthreads();
  int set = 0;
  for (; first < a.tokens; first += stride) {
    const Token next = token_at(a, first + stride + me.ts);
    const Rows<T, P> next_at(a, me, next.b, next.t);
    const float eps = now.in ? d.eps : 1.f;
    float2 e[NV][N];
    float cross[NV][N];
#pragma unroll
    for (int n = 0; n < NV; ++n)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int pair = me.column(a, n) / 2 + i;
        e[n][i] = make_float2(1.f, 0.f);
        if (now.in && me.slot_ok && pair < d.P) e[n][i] = cs[set * cs_set + me.ts * d.P + pair];
        cross[n][i] = 0.f;
      }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u >= me.ng) break;                                    // (the same for the block)
      const bool key = me.key(a, u);
      const int wrow = wt.row(a, u, me.hl, key) * pitch;
      f2 x[NV][N], g[NV][N], w[NV][N], ss = both(0.f), dot = both(0.f);
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        Pairs<T, V>::get(rx[u][n], x[n]);
        Pairs<T, V>::get(rg[u][n], g[n]);
        wt.load<V>(wt.w, wrow, n, me.lane, a.G, w[n]);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          g[n][i] = turn(g[n][i], make_float2(e[n][i].x, -e[n][i].y));       // dv = R^T do
          ss = fma2(x[n][i], x[n][i], ss);
          dot = fma2(mul2(g[n][i], w[n][i]), x[n][i], dot);
        }
      }
      load(next, next_at, u);
      const float rs = rsqrt_of<SUB>(fmaf(group_sum(sum2(ss), a.G), a.per_column, eps));
      const float m = group_sum(sum2(dot), a.G) * a.per_column * rs * rs;            // mean(w dv x r) r, per element of x
      if (!now.live || !me.has(a, u)) continue;
      T* o = static_cast<T*>(key ? d.dk : d.dq) + at.dense(a, me, u);
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        f2 out[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const f2 hat = mul2(x[n][i], both(rs));
          out[i] = mul2(both(rs), fma2(x[n][i], both(-m), mul2(g[n][i], w[n][i])));
          const f2 gh = mul2(g[n][i], hat);
          if constexpr (PER_HEAD) {
            gw[u][n][i] = add2(gw[u][n][i], gh);
            if (BIAS) gb[BIAS ? u : 0][n][i] = add2(gb[BIAS ? u : 0][n][i], g[n][i]);
          } else if (key) {
            gw[1][n][i] = add2(gw[1][n][i], gh);
            if (BIAS) gb[BIAS ? 1 : 0][n][i] = add2(gb[BIAS ? 1 : 0][n][i], g[n][i]);
          } else {
            gw[0][n][i] = add2(gw[0][n][i], gh);
            if (BIAS) gb[0][n][i] = add2(gb[0][n][i], g[n][i]);
          }
        }
        if (dang != nullptr) {                                  // (behind a length x and dv are 0)
          f2 b[N];
          wt.load<V>(wt.b, wrow, n, me.lane, a.G, b);
#pragma unroll
          for (int i = 0; i < N; ++i) {
            float v0, v1, g0, g1;
            unpack2(fma2(mul2(x[n][i], both(rs)), w[n][i], b[i]), v0, v1);
            unpack2(g[n][i], g0, g1);
            cross[n][i] += v0 * g1 - v1 * g0;
          }
        }
        store_cols<T, V, VEC>(o, me.column(a, n), d.Dh, out);
      }
    }
    if (dang != nullptr) {
#pragma unroll
      for (int n = 0; n < NV; ++n)
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int pair = me.column(a, n) / 2 + i;
          if (me.slot_ok && pair < d.P) rowbuf[slot * d.P + pair] = cross[n][i];
        }
    }
    if (first + stride < a.tokens) fill_angles(a, cs + (set ^ 1) * cs_set, first + stride);
    __syncthreads();
    if (dang != nullptr) {
      for (int i = threadIdx.x; i < cs_set; i += NT) {
        const int s = i / d.P, pair = i - s * d.P;
        if (first + s >= a.tokens) break;
        float sum = 0.f;
        for (int h = 0; h < a.hr; ++h) sum += rowbuf[(s * a.hr + h) * d.P + pair];
        dang[(static_cast<long long>(blockIdx.y) * a.tokens + first + s) * d.P + pair] = sum;
      }
      __syncthreads();
    }
    set ^= 1;
    now = next;
    at = next_at;
  }
  if (partial == nullptr) return;
  // the block's sums, over its token slots: of each head, or (one weight for all heads) of q's and of k's rows
  const int width = d.per_head ? (d.Hq + d.Hk) * d.Dh : 2 * d.Dh;
  const long long lines = static_cast<long long>(gridDim.x) * (d.per_head ? 1 : gridDim.y);
  const long long line = d.per_head ? blockIdx.x : static_cast<long long>(blockIdx.x) * gridDim.y + blockIdx.y;
  float* buf = smem;                                            // [rows][Dh]
#pragma unroll
  for (int what = 0; what < (BIAS ? 2 : 1); ++what) {
    float* out = partial + (what * lines + line) * width;
#pragma unroll
    for (int k = 0; k < SUMS; ++k) {
      if (PER_HEAD && k >= me.ng) break;
      __syncthreads();
#pragma unroll
      for (int n = 0; n < NV; ++n)
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int c = me.column(a, n) + 2 * i;
          float lo, hi;
          unpack2(BIAS && what ? gb[BIAS ? k : 0][n][i] : gw[k][n][i], lo, hi);
          if (me.slot_ok && c < d.Dh) {
            buf[slot * d.Dh + c] = lo;
            buf[slot * d.Dh + c + 1] = hi;
          }
        }
      __syncthreads();
      if constexpr (PER_HEAD) {
        const bool key = me.key(a, k);
        const int h0 = (me.g0 + k - (key ? a.q_groups : 0)) * a.hr, n_heads = min(a.hr, (key ? d.Hk : d.Hq) - h0);
        for (int i = threadIdx.x; i < n_heads * d.Dh; i += NT) {
          float sum = 0.f;
          for (int s = 0; s < a.TS; ++s) sum += buf[s * a.hr * d.Dh + i];
          out[static_cast<long long>((key ? d.Hq : 0) + h0) * d.Dh + i] = sum;
        }
      } else {
        for (int c = threadIdx.x; c < d.Dh; c += NT) {
          float sum = 0.f;
          for (int s = 0; s < rows; ++s) sum += buf[s * d.Dh + c];
          out[k * d.Dh + c] = sum;
        }
      }
    }
  }
}

// Column sums of partial[what][lines][width]: the first q_width columns are q's, the others k's. Block: 32 columns x 16
// line sets, each added up in order, then the 16 in order.
__global__ void __launch_bounds__(512) norm_rotate_params_kernel(const float* partial, long long lines, int width, int q_width, float* dqw,
                                                                 float* dkw, float* dqb, float* dkb) {
  __shared__ float part[16][33];
  const int c = blockIdx.x * 32 + threadIdx.x;
  const float* p = partial + blockIdx.y * lines * width;
  float sum = 0.f;
  if (c < width) {
#pragma unroll 4
    for (long long l = threadIdx.y; l < lines; l += 16) sum += p[l * width + c];
  }
  part[threadIdx.y][threadIdx.x] = sum;
  __syncthreads();
  if (threadIdx.y != 0 || c >= width) return;
  sum = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) sum += part[i][threadIdx.x];
  float* q = blockIdx.y ? dqb : dqw;
  float* k = blockIdx.y ? dkb : dkw;
  if (c < q_width) {
    if (q) q[c] = sum;
  } else if (k) {
    k[c - q_width] = sum;
  }
}

// d angles = sum over the slices of heads, in order
__global__ void __launch_bounds__(256) norm_rotate_angles_kernel(const float* parts, float* dang, long long n, int slices) {
  const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= n) return;
  float sum = 0.f;
  for (int s = 0; s < slices; ++s) sum += parts[s * n + i];
  dang[i] = sum;
}

bool multiple(const void* p, long long bytes) { return reinterpret_cast<unsigned long long>(p) % bytes == 0; }

bool packs_fit(const BdhNormRotateDesc& d, int v, int size) {
  for (const void* p : {d.q, d.k, static_cast<const void*>(d.q_out), static_cast<const void*>(d.k_out), d.dq_out, d.dk_out,
                        static_cast<const void*>(d.dq), static_cast<const void*>(d.dk)})
    if (!multiple(p, static_cast<long long>(v) * size)) return false;
  for (long long s : {d.q_sb, d.q_st, d.q_sh, d.k_sb, d.k_st, d.k_sh})
    if (s % v) return false;
  return d.Dh % v == 0;
}

int checked(const BdhNormRotateDesc& d) {
  if (d.dtype < 0 || d.dtype > 2 || d.B < 0 || d.T < 0 || d.Hq < 1 || d.Hk < 0 || d.Dh < 2 || d.Dh % 2 || d.Dh > 512 || d.P < 0 ||
      2 * d.P > d.Dh)
    return BDH_ERR_ARGUMENT;
  if (d.P > 0 && d.angles == nullptr && d.freqs == nullptr) return BDH_ERR_ARGUMENT;
  if (static_cast<long long>(d.B) * d.T > (1 << 30) || d.Hq + static_cast<long long>(d.Hk) > 65535) return BDH_ERR_TOO_LARGE;
  return BDH_OK;
}

NormArgs args_for(const BdhNormRotateDesc& d, int v, int nv, int groups_a_block) {
  NormArgs a;
  a.d = d;
  a.len = Lengths{d.lengths, d.lengths64};
  a.tokens = d.B * d.T;
  a.per_column = 1.f / d.Dh;
  a.G = 1;
  while (a.G * v * nv < d.Dh) a.G *= 2;
  const int rows = NT / a.G, most = d.Hq > d.Hk ? d.Hq : d.Hk;
  a.hr = most < rows ? most : rows;
  a.TS = rows / a.hr;
  a.q_groups = (d.Hq + a.hr - 1) / a.hr;
  a.groups = a.q_groups + (d.Hk + a.hr - 1) / a.hr;
  a.slices = (a.groups + groups_a_block - 1) / groups_a_block;
  a.per_block = (a.groups + a.slices - 1) / a.slices;
  return a;
}

bool subnormal(const BdhNormRotateDesc& d) { return !(d.eps >= FLT_MIN); }      // may mean x^2 + eps be?

int launched() { return cudaGetLastError() == cudaSuccess ? BDH_OK : BDH_ERR_LAUNCH; }

// Blocks along the tokens: as many as run at once, so that the weights are read (and their gradients written) once per
// block and not once per token.
int token_blocks(const NormArgs& a, int per_sm) {
  const long long need = (static_cast<long long>(a.tokens) + a.TS - 1) / a.TS;
  const long long most = (148LL * per_sm + a.slices - 1) / a.slices;
  return static_cast<int>(need < most ? need : most);
}
int weight_rows(const NormArgs& a) { return a.d.per_head ? a.per_block * a.hr : 2; }

constexpr int FEW = 2, MANY = 5;     // groups of heads a block: registers for their rows on the way
// (The weights of MANY groups, the angles and the sums take at most 42 KB of shared memory, by all widths and numbers of heads.)

template <typename T, int V, bool VEC, int NV, int U>
int fwd_launch(const BdhNormRotateDesc& d, cudaStream_t s) {
  const NormArgs a = args_for(d, V, NV, U);
  const int w_rows = weight_rows(a);
  const size_t smem = sizeof(float) * 2 * w_rows * a.G * V * NV + sizeof(float2) * 2 * a.TS * d.P;
  auto kernel = subnormal(d) ? norm_rotate_fwd_kernel<T, V, VEC, NV, U, true> : norm_rotate_fwd_kernel<T, V, VEC, NV, U, false>;
  kernel<<<dim3(token_blocks(a, FWD_BLOCKS), a.slices), NT, smem, s>>>(a, w_rows);
  return launched();
}

template <typename T, int V, bool VEC, int NV>
int fwd_groups(const BdhNormRotateDesc& d, cudaStream_t s) {
  if constexpr (NV == 1)
    if (args_for(d, V, NV, MANY).groups > FEW) return fwd_launch<T, V, VEC, NV, MANY>(d, s);
  return fwd_launch<T, V, VEC, NV, FEW>(d, s);
}

struct BwdOut {
  float *dqw, *dkw, *dqb, *dkb, *dang, *scratch;
};

struct BwdPlan {
  int blocks, width;
  long long lines, partial, angles;     // floats of scratch
  size_t smem;
};

BwdPlan bwd_plan(const NormArgs& a, int v_nv, bool want_w, bool want_b, bool want_ang) {
  BwdPlan p;
  p.blocks = token_blocks(a, BWD_BLOCKS);
  p.width = a.d.per_head ? (a.d.Hq + a.d.Hk) * a.d.Dh : 2 * a.d.Dh;
  p.lines = static_cast<long long>(p.blocks) * (a.d.per_head ? 1 : a.slices);
  p.partial = (want_w || want_b) ? (want_b ? 2 : 1) * p.lines * p.width : 0;
  p.angles = (want_ang && a.slices > 1) ? static_cast<long long>(a.slices) * a.tokens * a.d.P : 0;
  const size_t work = sizeof(float) * 2 * weight_rows(a) * a.G * v_nv + sizeof(float2) * 2 * a.TS * a.d.P +
                      sizeof(float) * (want_ang ? a.TS * a.hr * a.d.P : 0);
  const size_t sums = sizeof(float) * a.TS * a.hr * a.d.Dh;
  p.smem = work > sums ? work : sums;
  return p;
}

template <typename T, int V, bool VEC, int NV, int U, bool PER_HEAD, bool BIAS>
int bwd_launch(const BdhNormRotateDesc& d, const BwdOut& o, cudaStream_t s) {
  const NormArgs a = args_for(d, V, NV, U);
  const bool want_w = o.dqw || o.dkw || o.dqb || o.dkb, want_b = BIAS && want_w;
  const BwdPlan p = bwd_plan(a, V * NV, want_w, want_b, o.dang != nullptr);
  float* partial = want_w ? o.scratch : nullptr;        // (with BIAS the bias' sums lie behind the weights')
  float* ang = o.dang ? (p.angles ? o.scratch + p.partial : o.dang) : nullptr;
  auto kernel = subnormal(d) ? norm_rotate_bwd_kernel<T, V, VEC, NV, U, PER_HEAD, BIAS, true>
                             : norm_rotate_bwd_kernel<T, V, VEC, NV, U, PER_HEAD, BIAS, false>;
  kernel<<<dim3(p.blocks, a.slices), NT, p.smem, s>>>(a, weight_rows(a), partial, ang);
  if (launched() != BDH_OK) return BDH_ERR_LAUNCH;
  if (want_w) {
    norm_rotate_params_kernel<<<dim3((p.width + 31) / 32, want_b ? 2 : 1), dim3(32, 16), 0, s>>>(
        partial, p.lines, p.width, d.per_head ? d.Hq * d.Dh : d.Dh, o.dqw, o.dkw, o.dqb, o.dkb);
    if (launched() != BDH_OK) return BDH_ERR_LAUNCH;
  }
  if (p.angles) {
    const long long n = static_cast<long long>(a.tokens) * d.P;
    norm_rotate_angles_kernel<<<static_cast<unsigned>((n + 255) / 256), 256, 0, s>>>(ang, o.dang, n, a.slices);
  }
  return launched();
}

template <typename T, int V, bool VEC, int NV, bool BIAS>
int bwd_bias(const BdhNormRotateDesc& d, const BwdOut& o, cudaStream_t s) {
  if (d.per_head) return bwd_launch<T, V, VEC, NV, FEW, true, true>(d, o, s);
  if constexpr (NV == 1)
    if (args_for(d, V, NV, MANY).groups > FEW) return bwd_launch<T, V, VEC, NV, MANY, false, BIAS>(d, o, s);
  return bwd_launch<T, V, VEC, NV, FEW, false, BIAS>(d, o, s);
}
template <typename T, int V, bool VEC, int NV>
int bwd_groups(const BdhNormRotateDesc& d, const BwdOut& o, cudaStream_t s) {
  return (o.dqb || o.dkb) ? bwd_bias<T, V, VEC, NV, true>(d, o, s) : bwd_bias<T, V, VEC, NV, false>(d, o, s);
}

// The row's width decides how many packs a lane holds (at most 32 lanes a row).
template <typename T, typename F>
int by_width(const BdhNormRotateDesc& d, const F& f) {
  constexpr int V = 16 / sizeof(T);
  if (packs_fit(d, V, sizeof(T))) {
    if (d.Dh <= 32 * V) return f(std::integral_constant<int, V>{}, std::true_type{}, std::integral_constant<int, 1>{});
    if (d.Dh <= 64 * V) return f(std::integral_constant<int, V>{}, std::true_type{}, std::integral_constant<int, 2>{});
    if constexpr (V == 4) return f(std::integral_constant<int, V>{}, std::true_type{}, std::integral_constant<int, 4>{});
  }
  if (d.Dh <= 128) return f(std::integral_constant<int, 4>{}, std::false_type{}, std::integral_constant<int, 1>{});
  return f(std::integral_constant<int, 4>{}, std::false_type{}, std::integral_constant<int, 4>{});
}

}  // namespace

// Of one row type each: compiled in a file of their own (norm_rotate_f32.cu, _f16.cu, _bf16.cu).
template <typename T>
int norm_rotate_fwd_of(const BdhNormRotateDesc& d, cudaStream_t s) {
  return by_width<T>(d, [&](auto v, auto vec, auto nv) { return fwd_groups<T, decltype(v)::value, decltype(vec)::value, decltype(nv)::value>(d, s); });
}
struct NormRotateGrads {
  float *dqw, *dkw, *dqb, *dkb, *dang, *scratch;
};
template <typename T>
int norm_rotate_bwd_of(const BdhNormRotateDesc& d, const NormRotateGrads& g, cudaStream_t s) {
  const BwdOut o{g.dqw, g.dkw, g.dqb, g.dkb, g.dang, g.scratch};
  return by_width<T>(d, [&](auto v, auto vec, auto nv) { return bwd_groups<T, decltype(v)::value, decltype(vec)::value, decltype(nv)::value>(d, o, s); });
}

#define BDH_NORM_ROTATE_OF(EXTERN, T)                                                             \
  EXTERN template int norm_rotate_fwd_of<T>(const BdhNormRotateDesc&, cudaStream_t);              \
  EXTERN template int norm_rotate_bwd_of<T>(const BdhNormRotateDesc&, const NormRotateGrads&, cudaStream_t);

}  // namespace bdh
