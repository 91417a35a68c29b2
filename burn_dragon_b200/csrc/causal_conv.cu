// Causal depthwise convolution along the sequence with a carried state, bias and SiLU:
//
//   s = [state (k - 1 rows) | x];   pre_t = bias + sum_j w_j s_{t+j};   y_t = pre_t sigmoid(pre_t)  (or pre_t)
//   state' = the last k - 1 rows of s before the sequence's length
//   d pre_t = dy_t silu'(pre_t);    d s_r = sum_j w_j d pre_{r-j};      d w_j = sum_t d pre_t s_{t+j};   d bias = sum_t d pre_t
//
// Bound by memory: 2 k + 5 operations on 2 (forward) or 3 (backward) tensors. A thread owns V adjacent channels and
// walks down a tile of the time axis with the k - 1 rows behind it in registers, so that each element of x is read
// once and k - 1 rows per tile twice (the second time from L2). fp32 throughout; the parameter gradients are summed
// in registers over every tile that a block walks, then over the block, then over the blocks in a fixed order (no
// atomics: two runs give the same bits). Channels go in pairs (one instruction for two), rows in sets that change
// places instead of moving, and the next set is on its way while one is worked on.
//
// Measured, 8 x 2048 x 4096 bf16: forward 57 us (0.73 of the copy rate), backward 110 us (0.57) and 7 us for the parameters' sums;
// one token of 64 streams 4.5 us. The backward pass issues about 30 instructions an element pair and row, but a scheduler is busy
// only 43 % of the time: its three warps wait for the results of their own arithmetic.
#include "bdh_kernels.h"
#include "pair_math.cuh"

#include <type_traits>

namespace bdh {
namespace {

constexpr int FWD_THREADS = 128;
constexpr int FWD_ROWS = 8;          // rows that a thread works on at once, forward and (width 2 to 4) backward
constexpr int BWD_ROWS = 4;
constexpr int BWD_LANES = 32;        // backward block: 32 channel packs x 4 tiles
constexpr int BWD_TILES = 4;
constexpr int BWD_THREADS = BWD_LANES * BWD_TILES;
enum { ANY_SET, FIRST_SET, MIDDLE_SET, LAST_SET };
constexpr int AHEAD = 2;             // sets of rows on their way, backward (AHEAD + 1 sets of shared memory)

struct ConvArgs {
  BdhConvDesc d;
  Lengths len;
  int packs;          // ceil(C / V)
  int tile, tiles;    // rows per tile, tiles per sequence
};

// Row r of [state | x] (r counts from the first row of x; negative: the state), V channels from c on, as it lies in
// memory. INSIDE: the row is one of x's for certain.
template <typename T, int V, bool INSIDE>
__device__ __forceinline__ typename Pack<T, V>::Raw load_seq(const BdhConvDesc& d, int b, int r, int len, int c) {
  Pack<T, V> p;
  if (INSIDE || (r >= 0 && r < len)) {
    return *reinterpret_cast<const typename Pack<T, V>::Raw*>(static_cast<const T*>(d.x) + b * d.x_sb + r * d.x_st + c);
  } else if (r < 0 && r + d.k - 1 >= 0 && d.state != nullptr) {
    p.load(static_cast<const T*>(d.state) + b * d.state_sb + (r + d.k - 1) * d.state_sr + c);
  } else {
    p.zero();
  }
  return *reinterpret_cast<const typename Pack<T, V>::Raw*>(&p);
}
// K: the kernel width, or 0 for a width of up to 8 known at run time (taps then sit at the end of the window; the leading
// ones are skipped, not multiplied by zero: a row there may hold anything). R: rows that a thread works on at once; with
// the R rows before them they hold every window, and the two sets change places instead of moving.
template <int V, int K, int R>
struct Taps {
  static constexpr int KM = K ? K : 8, N = (V + 1) / 2;
  static_assert(KM - 1 <= R, "a window lies within two sets of rows");
  f2 w[KM][N], bias[N];
  f2 first[K ? 1 : KM][N];             // K = 0: the taps again, from the window's start on
  __device__ __forceinline__ f2 tap(int j, int n) const { return K ? w[j][n] : first[K ? 0 : j][n]; }
  __device__ __forceinline__ void load(const BdhConvDesc& d, int k, int c, bool live) {
    const auto one = [&](int j, int v) { return (live && v < V && j >= KM - k && j < KM) ? d.w[static_cast<long long>(c + v) * k + j - (KM - k)] : 0.f; };
    const auto off = [&](int v) { return (live && v < V && d.bias) ? d.bias[c + v] : 0.f; };
#pragma unroll
    for (int n = 0; n < N; ++n) {
#pragma unroll
      for (int j = 0; j < KM; ++j) w[j][n] = pack2(one(j, 2 * n), one(j, 2 * n + 1));
      bias[n] = pack2(off(2 * n), off(2 * n + 1));
      if constexpr (K == 0) {
#pragma unroll
        for (int j = 0; j < KM; ++j) first[j][n] = pack2(one(j + KM - k, 2 * n), one(j + KM - k, 2 * n + 1));
      }
    }
  }
  __device__ __forceinline__ f2 pre(const f2 (&before)[R][N], const f2 (&s)[R][N], int r, int n, int k) const {
    f2 x = bias[n];
#pragma unroll
    for (int j = 0; j < KM; ++j)
      if (K || j >= KM - k) x = fma2(w[j][n], at(before, s, r - (KM - 1) + j, n), x);
    return x;
  }
  static __device__ __forceinline__ f2 at(const f2 (&before)[R][N], const f2 (&s)[R][N], int row, int n) {
    return row < 0 ? before[row < 0 ? row + R : 0][n] : s[row < 0 ? 0 : row][n];
  }
};

// Rows t0 .. t1 of one sequence. The next rows are on their way (as raw bits: taking the elements out behind the load
// would wait for it) while the present ones are worked on. INSIDE: every row that is read is one of x's, t1 - t0 is a
// multiple of R.
template <typename T, int V, int K, bool INSIDE>
__device__ __forceinline__ void conv_fwd_tile(const BdhConvDesc& d, const Taps<V, K, FWD_ROWS>& w, int b, int t0, int t1, int len, int c) {
  using W = Taps<V, K, FWD_ROWS>;
  constexpr int R = FWD_ROWS, N = W::N;
  using Raw = typename Pack<T, V>::Raw;
  const int k = K ? K : d.k;
  f2 one[R][N], two[R][N];
  Raw next[R];
  const T* px = static_cast<const T*>(d.x) + b * d.x_sb + t0 * d.x_st + c;
  const auto load = [&](int t) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      next[r] = INSIDE ? *reinterpret_cast<const Raw*>(px) : load_seq<T, V, false>(d, b, t + r, min(len, t1), c);
      px += d.x_st;
    }
  };
  load(t0);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (r <= R - W::KM) continue;                                            // (not in any window)
    Pairs<T, V>::get(load_seq<T, V, INSIDE>(d, b, t0 - R + r, len, c), one[r]);
  }
  T* y = static_cast<T*>(d.y) + (static_cast<long long>(b) * d.T + t0) * d.C + c;
  const auto rows = [&](int t, const f2 (&before)[R][N], f2 (&s)[R][N]) {
#pragma unroll
    for (int r = 0; r < R; ++r) Pairs<T, V>::get(next[r], s[r]);
    if (t + R < t1) load(t + R);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (!INSIDE && t + r >= t1) break;
      f2 o[N];
#pragma unroll
      for (int n = 0; n < N; ++n) {
        o[n] = w.pre(before, s, r, n, k);
        if (d.silu) o[n] = mul2(o[n], sigmoid_quick2(o[n]));
        if (!INSIDE && t + r >= len) o[n] = both(0.f);
      }
      *reinterpret_cast<Raw*>(y) = Pairs<T, V>::put(o);
      y += d.C;
    }
  };
#pragma unroll 1
  for (int t = t0; t < t1; t += 2 * R) {
    rows(t, one, two);
    if (t + R < t1) rows(t + R, two, one);
  }
}

template <typename T, int V, int K>
__global__ void __launch_bounds__(FWD_THREADS, 6) causal_conv_fwd_kernel(const ConvArgs a) {
  using W = Taps<V, K, FWD_ROWS>;
  const BdhConvDesc& d = a.d;
  const int k = K ? K : d.k;
  const long long i = static_cast<long long>(blockIdx.x) * FWD_THREADS + threadIdx.x;
  const int c = static_cast<int>(i % a.packs) * V;
  const long long bt = i / a.packs;
  const int per = a.tiles + 1;                      // one more "tile" per sequence writes its new state
  const int b = static_cast<int>(bt / per), tile = static_cast<int>(bt % per);
  if (b >= d.B) return;
  const int len = a.len.get(b, d.T);
  if (tile == a.tiles) {
    if (d.state_out != nullptr)
      for (int j = 0; j < k - 1; ++j)
        *reinterpret_cast<typename Pack<T, V>::Raw*>(static_cast<T*>(d.state_out) + b * d.state_out_sb + j * d.state_out_sr + c) =
            load_seq<T, V, false>(d, b, len - (k - 1) + j, len, c);
    return;
  }
  W w;
  w.load(d, k, c, true);
  const int t0 = tile * a.tile, t1 = min(t0 + a.tile, d.T);
  if (t0 >= FWD_ROWS && t1 <= len && (t1 - t0) % FWD_ROWS == 0)
    conv_fwd_tile<T, V, K, true>(d, w, b, t0, t1, len, c);
  else
    conv_fwd_tile<T, V, K, false>(d, w, b, t0, t1, len, c);
}

// Gradients of rows t0 .. t1: dx (and d state) need d pre of these rows and of the k - 1 behind them, which the thread
// computes too. INSIDE: every row of x and dy that is read exists, no row is one of the new state's, and t1 - t0 is an
// even number of sets. sw, sb: the thread's sums for w and bias.
template <typename T, int V, int K, bool INSIDE>
struct BwdTile {
  static constexpr int R = K ? BWD_ROWS : 8;
  using W = Taps<V, K, R>;
  static constexpr int KM = W::KM, N = W::N;
  using Raw = typename Pack<T, V>::Raw;
  // INSIDE: rows come by asynchronous copies AHEAD sets before their turn, each thread reading back its own; registers
  // for that many would leave too few threads to cover the way to memory. Else one set ahead, in registers.
  static constexpr bool RINGS = INSIDE && K != 0 && V * sizeof(T) >= 4;
  static constexpr int BYTES = V * static_cast<int>(sizeof(T));
  const BdhConvDesc& d;
  const W& w;
  f2 (&sw)[KM][N];
  f2 (&sb)[N];
  Raw* ring;
  int b, t0, t1, len, c, k;
  const T *px, *pd;                  // the next row to be fetched
  T* pg;                             // the next row of dx
  int set = 0;                       // of the next rows to be worked on
  Raw nx[R], nd[R];

  __device__ __forceinline__ void load(int t, int to) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if constexpr (RINGS) {
        if (t < t1 + k - 1) {
          copy_async<BYTES>(ring + (to * R + r) * 2 * BWD_THREADS, px, true);
          copy_async<BYTES>(ring + ((to * R + r) * 2 + 1) * BWD_THREADS, pd, true);
        }
      } else if (INSIDE || (t + r < len && t + r < t1 + k - 1)) {
        nx[r] = *reinterpret_cast<const Raw*>(px);
        nd[r] = *reinterpret_cast<const Raw*>(pd);
      } else {
        Pack<T, V> p;
        p.zero();
        nx[r] = nd[r] = *reinterpret_cast<const Raw*>(&p);
      }
      px += d.x_st;
      pd += d.dy_st;
    }
    if constexpr (RINGS) copy_close();
  }

  // One set of rows. Which of a tile's sets it is decides at compile time what INSIDE needs no test for: the first
  // completes no row before t0, the last (behind t1) gives d pre only.
  template <int SET>
  __device__ __forceinline__ void rows(int t, int first, const f2 (&sp)[R][N], f2 (&s)[R][N], const f2 (&gp)[R][N], f2 (&g)[R][N]) {
    if constexpr (RINGS) {
      copy_wait<AHEAD - 1>();
#pragma unroll
      for (int r = 0; r < R; ++r) {
        nx[r] = ring[(set * R + r) * 2 * BWD_THREADS];
        nd[r] = ring[((set * R + r) * 2 + 1) * BWD_THREADS];
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      Pairs<T, V>::get(nx[r], s[r]);
      Pairs<T, V>::get(nd[r], g[r]);                                         // dy for now
    }
    if constexpr (RINGS) {                                                   // into the set that was read before this one
      if constexpr (SET != LAST_SET) load(t + AHEAD * R, set == 0 ? AHEAD : set - 1);
      set = set == AHEAD ? 0 : set + 1;
    } else {
      if (t + R < t1 + k - 1) load(t + R, 0);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (SET == LAST_SET && r >= KM - 1) break;
      const bool in = SET != ANY_SET || t + r < len;
      const bool mine = SET == ANY_SET ? t + r < t1 && in : SET != LAST_SET;
#pragma unroll
      for (int n = 0; n < N; ++n) {
        if (d.silu) {                                                        // silu' = sg (1 + pre (1 - sg))
          const f2 pre = w.pre(sp, s, r, n, k), sg = sigmoid_quick2(pre);
          g[r][n] = mul2(g[r][n], mul2(sg, fma2(pre, fma2(sg, both(-1.f), both(1.f)), both(1.f))));
        }
        if (!in) g[r][n] = both(0.f);
        if (mine) {
          sb[n] = add2(sb[n], g[r][n]);
#pragma unroll
          for (int j = 0; j < KM; ++j)
            if (K || j >= KM - k) sw[j][n] = fma2(g[r][n], W::at(sp, s, r - (KM - 1) + j, n), sw[j][n]);
        }
      }
      const int row = t + r - (k - 1);                                       // complete now: every d pre it feeds is known
      if (SET == ANY_SET ? (row >= first && row < t1) : (SET != FIRST_SET || r >= KM - 1)) {
        f2 o[N];
#pragma unroll
        for (int n = 0; n < N; ++n) {
          o[n] = both(0.f);
#pragma unroll
          for (int j = 0; j < KM; ++j)                                       // tap j of output row + (k - 1) - j
            if (K || j < k) o[n] = fma2(w.tap(j, n), W::at(gp, g, r - j, n), o[n]);
        }
        const int j = row - (len - (k - 1));                                 // its place in the new state
        if (!INSIDE && d.dstate_out != nullptr && j >= 0 && j < k - 1) {
          f2 e[N];
          Pairs<T, V>::get(*reinterpret_cast<const Raw*>(static_cast<const T*>(d.dstate_out) +
                                                         (static_cast<long long>(b) * (k - 1) + j) * d.C + c), e);
#pragma unroll
          for (int n = 0; n < N; ++n) o[n] = add2(o[n], e[n]);
        }
        if (INSIDE || row >= 0) {
          *reinterpret_cast<Raw*>(pg) = Pairs<T, V>::put(o);
          pg += d.C;
        } else {
          *reinterpret_cast<Raw*>(static_cast<T*>(d.dstate) + (static_cast<long long>(b) * (k - 1) + row + k - 1) * d.C + c) =
              Pairs<T, V>::put(o);
        }
      }
    }
  }

  __device__ __forceinline__ void run() {
    f2 s1[R][N], s2[R][N], g1[R][N], g2[R][N];
    px = static_cast<const T*>(d.x) + b * d.x_sb + t0 * d.x_st + c;
    pd = static_cast<const T*>(d.dy) + b * d.dy_sb + t0 * d.dy_st + c;
    pg = static_cast<T*>(d.dx) + (static_cast<long long>(b) * d.T + t0) * d.C + c;
    load(t0, 0);
    if constexpr (RINGS) {
#pragma unroll
      for (int i = 1; i < AHEAD; ++i) load(t0 + i * R, i);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int n = 0; n < N; ++n) g1[r][n] = both(0.f);
      if (r <= R - KM) continue;                                             // (not in any window)
      Pairs<T, V>::get(load_seq<T, V, INSIDE>(d, b, t0 - R + r, len, c), s1[r]);
    }
    if constexpr (INSIDE && K != 0) {                                        // an even number of sets, and the one behind
      rows<FIRST_SET>(t0, t0, s1, s2, g1, g2);
      rows<MIDDLE_SET>(t0 + R, t0, s2, s1, g2, g1);
#pragma unroll 1
      for (int t = t0 + 2 * R; t < t1; t += 2 * R) {
        rows<MIDDLE_SET>(t, t0, s1, s2, g1, g2);
        rows<MIDDLE_SET>(t + R, t0, s2, s1, g2, g1);
      }
      rows<LAST_SET>(t1, t0, s1, s2, g1, g2);
    } else {
      const int first = (!INSIDE && t0 == 0 && d.dstate != nullptr) ? -(k - 1) : t0;  // first row whose gradient this tile writes
#pragma unroll 1
      for (int t = t0; t < t1 + k - 1; t += 2 * R) {
        rows<ANY_SET>(t, first, s1, s2, g1, g2);
        if (t + R < t1 + k - 1) rows<ANY_SET>(t + R, first, s2, s1, g2, g1);
      }
    }
  }
};

template <typename T, int V, int K>
__global__ void __launch_bounds__(BWD_THREADS, K ? 3 : 2) causal_conv_bwd_kernel(const ConvArgs a, float* partial, int groups) {
  using W = typename BwdTile<T, V, K, true>::W;
  constexpr int KM = W::KM, N = W::N, R = BwdTile<T, V, K, true>::R;
  const BdhConvDesc& d = a.d;
  const int k = K ? K : d.k;
  const int cblocks = (a.packs + BWD_LANES - 1) / BWD_LANES;
  const int pack = (blockIdx.x % cblocks) * BWD_LANES + threadIdx.x, group = blockIdx.x / cblocks;
  const bool live = pack < a.packs;
  const int c = pack * V;
  __shared__ typename Pack<T, V>::Raw ring[K ? (AHEAD + 1) * R * 2 * BWD_THREADS : 1];
  typename Pack<T, V>::Raw* own = ring + (K ? threadIdx.y * BWD_LANES + threadIdx.x : 0);
  W w;
  w.load(d, k, c, live);
  f2 sw[KM][N], sb[N];
#pragma unroll
  for (int n = 0; n < N; ++n) {
#pragma unroll
    for (int j = 0; j < KM; ++j) sw[j][n] = both(0.f);
    sb[n] = both(0.f);
  }
  const long long all = static_cast<long long>(d.B) * a.tiles;
  for (long long bt = static_cast<long long>(group) * BWD_TILES + threadIdx.y; live && bt < all;
       bt += static_cast<long long>(groups) * BWD_TILES) {
    const int b = static_cast<int>(bt / a.tiles), tile = static_cast<int>(bt % a.tiles);
    const int len = a.len.get(b, d.T);
    const int t0 = tile * a.tile, t1 = min(t0 + a.tile, d.T);
    // rows up to t1 + R + k are read inside; the new state's are behind them
    if (t0 >= R && t1 + k + R <= len && (t1 - t0) % (2 * R) == 0)
      BwdTile<T, V, K, true>{d, w, sw, sb, own, b, t0, t1, len, c, k}.run();
    else
      BwdTile<T, V, K, false>{d, w, sw, sb, own, b, t0, t1, len, c, k}.run();
  }
  if (partial == nullptr) return;
  // partial[group][tap or bias][channel]: the block's four tile rows added up
  __shared__ f2 sum[BWD_TILES][N][BWD_LANES];
#pragma unroll
  for (int j = 0; j <= KM; ++j) {
    if (j < KM - k) continue;
#pragma unroll
    for (int n = 0; n < N; ++n) sum[threadIdx.y][n][threadIdx.x] = j < KM ? sw[j < KM ? j : 0][n] : sb[n];
    __syncthreads();
    if (threadIdx.y == 0 && live) {
#pragma unroll
      for (int n = 0; n < N; ++n) {
        f2 x = sum[0][n][threadIdx.x];
#pragma unroll
        for (int y = 1; y < BWD_TILES; ++y) x = add2(x, sum[y][n][threadIdx.x]);
        float lo, hi;
        unpack2(x, lo, hi);
        float* to = partial + (static_cast<long long>(group) * (k + 1) + j - (KM - k)) * d.C + c + 2 * n;
        to[0] = lo;
        if (2 * n + 1 < V) to[1] = hi;
      }
    }
    __syncthreads();
  }
}

// dw[c][j], db[c] = sum over the groups, in order
__global__ void __launch_bounds__(128) causal_conv_params_kernel(const float* partial, float* dw, float* db, int groups, int C, int k) {
  const long long i = static_cast<long long>(blockIdx.x) * 128 + threadIdx.x;
  if (i >= static_cast<long long>(C) * (k + 1)) return;
  const int c = static_cast<int>(i % C), j = static_cast<int>(i / C);
  float x = 0.f;
#pragma unroll 8
  for (int g = 0; g < groups; ++g) x += partial[static_cast<long long>(g) * (k + 1) * C + i];
  if (j < k) {
    if (dw) dw[static_cast<long long>(c) * k + j] = x;
  } else if (db) {
    db[c] = x;
  }
}

// One token of every stream: y and the state moved on by one row (in place where the two states are the same).
template <typename T, int V>
__global__ void __launch_bounds__(FWD_THREADS) causal_conv_step_kernel(const ConvArgs a, const unsigned char* active) {
  const BdhConvDesc& d = a.d;
  const long long i = static_cast<long long>(blockIdx.x) * FWD_THREADS + threadIdx.x;
  const int c = static_cast<int>(i % a.packs) * V;
  const int b = static_cast<int>(i / a.packs);
  if (b >= d.B) return;
  const bool on = active == nullptr || active[b] != 0;
  const int k = d.k;
  const T* st = static_cast<const T*>(d.state) + b * d.state_sb + c;
  T* so = static_cast<T*>(d.state_out) + b * d.state_out_sb + c;
  using Raw = typename Pack<T, V>::Raw;
  constexpr int N = (V + 1) / 2;
  Raw row[7];
#pragma unroll
  for (int j = 0; j < 7; ++j)
    if (j < k - 1) row[j] = *reinterpret_cast<const Raw*>(st + j * d.state_sr);
  const Raw x = *reinterpret_cast<const Raw*>(static_cast<const T*>(d.x) + b * d.x_sb + c);
  const auto tap = [&](int v, int j) { return v < V ? d.w[static_cast<long long>(c + v) * k + j] : 0.f; };
  const auto add = [&](f2 (&o)[N], const Raw& r, int j) {
    f2 e[N];
    Pairs<T, V>::get(r, e);
#pragma unroll
    for (int n = 0; n < N; ++n) o[n] = fma2(pack2(tap(2 * n, j), tap(2 * n + 1, j)), e[n], o[n]);
  };
  f2 o[N];
#pragma unroll
  for (int n = 0; n < N; ++n) o[n] = d.bias ? pack2(d.bias[c + 2 * n], 2 * n + 1 < V ? d.bias[c + 2 * n + 1] : 0.f) : both(0.f);
#pragma unroll
  for (int j = 0; j < 7; ++j)
    if (j < k - 1) add(o, row[j], j);
  add(o, x, k - 1);
#pragma unroll
  for (int n = 0; n < N; ++n) {
    if (d.silu) o[n] = mul2(o[n], sigmoid_quick2(o[n]));
    if (!on) o[n] = both(0.f);
  }
  *reinterpret_cast<Raw*>(static_cast<T*>(d.y) + static_cast<long long>(b) * d.C + c) = Pairs<T, V>::put(o);
  if (!on && so == st) return;
#pragma unroll
  for (int j = 0; j < 7; ++j)
    if (j < k - 1) {
      Raw r = row[j];
      if (on) r = j + 1 < k - 1 ? row[j < 6 ? j + 1 : 6] : x;
      *reinterpret_cast<Raw*>(so + j * d.state_out_sr) = r;
    }
}

bool multiple(const void* p, long long bytes) { return reinterpret_cast<unsigned long long>(p) % bytes == 0; }

// Can every row of the call be moved in packs of `v` elements?
bool packs_fit(const BdhConvDesc& d, int v, int size) {
  const long long bytes = static_cast<long long>(v) * size;
  for (const void* p : {d.x, d.state, static_cast<const void*>(d.y), static_cast<const void*>(d.state_out), d.dy, d.dstate_out,
                        static_cast<const void*>(d.dx), static_cast<const void*>(d.dstate)})
    if (!multiple(p, bytes)) return false;
  for (long long s : {d.x_sb, d.x_st, d.state_sb, d.state_sr, d.state_out_sb, d.state_out_sr, d.dy_sb, d.dy_st})
    if (s % v) return false;
  return d.C % v == 0;
}

int checked(const BdhConvDesc& d) {
  if (d.k < 1 || d.k > 8 || d.B < 0 || d.T < 0 || d.C < 1 || d.dtype < 0 || d.dtype > 2) return BDH_ERR_ARGUMENT;
  return BDH_OK;
}

// Rows per tile: 64 keeps the rows that two tiles both read at (k - 1) / 64; shorter tiles, not below 16, while there are
// fewer threads than a quarter of what the GPU holds (4096 x 2048 bf16: 10.5 us, in tiles of 64 26 us).
int tile_rows(const BdhConvDesc& d, int packs) {
  int tile = 64;
  while (tile > 16 && static_cast<long long>(d.B) * ((d.T + tile - 1) / tile) * packs < 148LL * 512) tile /= 2;
  return tile;
}

ConvArgs args_for(const BdhConvDesc& d, int v) {
  ConvArgs a;
  a.d = d;
  a.len = Lengths{d.lengths, d.lengths64};
  a.packs = (d.C + v - 1) / v;
  a.tile = tile_rows(d, a.packs);
  a.tiles = (d.T + a.tile - 1) / a.tile;
  return a;
}

int launched() { return cudaGetLastError() == cudaSuccess ? BDH_OK : BDH_ERR_LAUNCH; }

template <typename T, int V, int K>
int fwd_launch(const BdhConvDesc& d, cudaStream_t s) {
  const ConvArgs a = args_for(d, V);
  const long long threads = static_cast<long long>(d.B) * (a.tiles + 1) * a.packs;
  const long long blocks = (threads + FWD_THREADS - 1) / FWD_THREADS;
  if (blocks > 0x7fffffffLL) return BDH_ERR_TOO_LARGE;
  causal_conv_fwd_kernel<T, V, K><<<static_cast<unsigned>(blocks), FWD_THREADS, 0, s>>>(a);
  return launched();
}

template <typename T, int V>
int fwd_width(const BdhConvDesc& d, cudaStream_t s) {
  switch (d.k) {
    case 2: return fwd_launch<T, V, 2>(d, s);
    case 3: return fwd_launch<T, V, 3>(d, s);
    case 4: return fwd_launch<T, V, 4>(d, s);
  }
  return fwd_launch<T, V, 0>(d, s);
}

int bwd_groups(const ConvArgs& a) {
  const long long all = (static_cast<long long>(a.d.B) * a.tiles + BWD_TILES - 1) / BWD_TILES;
  const int cblocks = (a.packs + BWD_LANES - 1) / BWD_LANES;
  const long long most = (148LL * 8 + cblocks - 1) / cblocks;          // about two waves of blocks
  return static_cast<int>(all < most ? all : most);
}

template <typename T, int V, int K>
int bwd_launch(const BdhConvDesc& d, float* dw, float* db, float* partial, cudaStream_t s) {
  const ConvArgs a = args_for(d, V);
  const int groups = bwd_groups(a), cblocks = (a.packs + BWD_LANES - 1) / BWD_LANES;
  float* part = (dw || db) ? partial : nullptr;
  if (groups > 0) {
    causal_conv_bwd_kernel<T, V, K><<<cblocks * groups, dim3(BWD_LANES, BWD_TILES), 0, s>>>(a, part, groups);
    if (launched() != BDH_OK) return BDH_ERR_LAUNCH;
  }
  if (part) {
    const long long n = static_cast<long long>(d.C) * (d.k + 1);
    causal_conv_params_kernel<<<static_cast<unsigned>((n + 127) / 128), 128, 0, s>>>(part, dw, db, groups, d.C, d.k);
  }
  return launched();
}

template <typename T, int V>
int bwd_width(const BdhConvDesc& d, float* dw, float* db, float* partial, cudaStream_t s) {
  switch (d.k) {
    case 2: return bwd_launch<T, V, 2>(d, dw, db, partial, s);
    case 3: return bwd_launch<T, V, 3>(d, dw, db, partial, s);
    case 4: return bwd_launch<T, V, 4>(d, dw, db, partial, s);
  }
  return bwd_launch<T, V, 0>(d, dw, db, partial, s);
}

template <typename T, int V>
int step_launch(const BdhConvDesc& d, const unsigned char* active, cudaStream_t s) {
  const ConvArgs a = args_for(d, V);
  const long long blocks = (static_cast<long long>(d.B) * a.packs + FWD_THREADS - 1) / FWD_THREADS;
  if (blocks > 0x7fffffffLL) return BDH_ERR_TOO_LARGE;
  causal_conv_step_kernel<T, V><<<static_cast<unsigned>(blocks), FWD_THREADS, 0, s>>>(a, active);
  return launched();
}

// Channels a thread. Forward two: the most threads that still store a pair (8 x 2048 x 4096 bf16, in one run: 55 us; four 57,
// eight 78 us; at 4096 x 2048 10.5, 18 and 26 us). Backward 8 bytes: rows come through shared memory there, and a
// thread's overhead is shared by more elements.
template <typename T>
int fwd_type(const BdhConvDesc& d, cudaStream_t s) {
  return packs_fit(d, 2, sizeof(T)) ? fwd_width<T, 2>(d, s) : fwd_width<T, 1>(d, s);
}
template <typename T>
int bwd_type(const BdhConvDesc& d, float* dw, float* db, float* partial, cudaStream_t s) {
  constexpr int V = 8 / sizeof(T);
  return packs_fit(d, V, sizeof(T)) ? bwd_width<T, V>(d, dw, db, partial, s) : bwd_width<T, 1>(d, dw, db, partial, s);
}
template <typename T>
int step_type(const BdhConvDesc& d, const unsigned char* active, cudaStream_t s) {
  constexpr int V = 8 / sizeof(T);
  return packs_fit(d, V, sizeof(T)) ? step_launch<T, V>(d, active, s) : step_launch<T, 1>(d, active, s);
}

}  // namespace
}  // namespace bdh

using namespace bdh;

extern "C" int bdh_causal_conv_fwd(const BdhConvDesc* d, cudaStream_t s) {
  if (const int rc = checked(*d)) return rc;
  if (d->B == 0) return BDH_OK;
  switch (d->dtype) {
    case BDH_F32: return fwd_type<float>(*d, s);
    case BDH_F16: return fwd_type<__half>(*d, s);
  }
  return fwd_type<__nv_bfloat16>(*d, s);
}

// The widest case (one element per pack) decides, so that the caller need not know which packs fit.
extern "C" long long bdh_causal_conv_partials(const BdhConvDesc* d) {
  if (checked(*d) != BDH_OK) return 0;
  long long most = 0;
  for (int v : {1, 2, 4}) {
    const long long n = static_cast<long long>(bwd_groups(args_for(*d, v))) * (d->k + 1) * d->C;
    most = n > most ? n : most;
  }
  return most;
}

extern "C" int bdh_causal_conv_bwd(const BdhConvDesc* d, float* dw, float* db, float* partial, cudaStream_t s) {
  if (const int rc = checked(*d)) return rc;
  if ((dw || db) && partial == nullptr) return BDH_ERR_ARGUMENT;
  switch (d->dtype) {
    case BDH_F32: return bwd_type<float>(*d, dw, db, partial, s);
    case BDH_F16: return bwd_type<__half>(*d, dw, db, partial, s);
  }
  return bwd_type<__nv_bfloat16>(*d, dw, db, partial, s);
}

extern "C" int bdh_causal_conv_step(const BdhConvDesc* d, const unsigned char* active, cudaStream_t s) {
  if (const int rc = checked(*d)) return rc;
  if (d->B == 0) return BDH_OK;
  switch (d->dtype) {
    case BDH_F32: return step_type<float>(*d, active, s);
    case BDH_F16: return step_type<__half>(*d, active, s);
  }
  return step_type<__nv_bfloat16>(*d, active, s);
}
