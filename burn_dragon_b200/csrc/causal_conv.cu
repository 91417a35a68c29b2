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
// atomics: two runs give the same bits).
#include "bdh_kernels.h"
#include "element_io.cuh"

namespace bdh {
namespace {

constexpr int ROWS = 4;              // rows of x in flight per thread
constexpr int FWD_THREADS = 128;
constexpr int BWD_LANES = 32;        // backward block: 32 channel packs x 4 tiles
constexpr int BWD_TILES = 4;

struct ConvArgs {
  BdhConvDesc d;
  Lengths len;
  int packs;          // ceil(C / V)
  int tile, tiles;    // rows per tile, tiles per sequence
};

// Row r of [state | x] (r counts from the first row of x; negative: the state), V channels from c on.
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_seq(const BdhConvDesc& d, int b, int r, int len, int c) {
  Pack<T, V> p;
  if (r >= 0 && r < len) {
    p.load(static_cast<const T*>(d.x) + b * d.x_sb + r * d.x_st + c);
  } else if (r < 0 && r + d.k - 1 >= 0 && d.state != nullptr) {
    p.load(static_cast<const T*>(d.state) + b * d.state_sb + (r + d.k - 1) * d.state_sr + c);
  } else {
    p.zero();
  }
  return p;
}

// K: the kernel width, or 0 for a width of up to 8 known at run time (taps then sit at the end of the window; the
// leading ones are skipped, not multiplied by zero: a row there may hold anything).
template <typename T, int V, int K>
__global__ void __launch_bounds__(FWD_THREADS) causal_conv_fwd_kernel(const ConvArgs a) {
  constexpr int KM = K ? K : 8;
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
        load_seq<T, V>(d, b, len - (k - 1) + j, len, c)
            .store(static_cast<T*>(d.state_out) + b * d.state_out_sb + j * d.state_out_sr + c);
    return;
  }
  float w[KM][V], bias[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
#pragma unroll
    for (int j = 0; j < KM; ++j) w[j][v] = (j >= KM - k) ? d.w[static_cast<long long>(c + v) * k + j - (KM - k)] : 0.f;
    bias[v] = d.bias ? d.bias[c + v] : 0.f;
  }
  const int t0 = tile * a.tile, t1 = min(t0 + a.tile, d.T);
  float s[KM - 1 + ROWS][V];
#pragma unroll
  for (int j = 0; j < KM - 1; ++j) {
    const Pack<T, V> p = load_seq<T, V>(d, b, t0 - (KM - 1) + j, len, c);
#pragma unroll
    for (int v = 0; v < V; ++v) s[j][v] = p[v];
  }
  T* y = static_cast<T*>(d.y) + (static_cast<long long>(b) * d.T) * d.C + c;
  for (int t = t0; t < t1; t += ROWS) {
    Pack<T, V> p[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) p[r] = load_seq<T, V>(d, b, t + r, min(len, t1), c);
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
      for (int v = 0; v < V; ++v) s[KM - 1 + r][v] = p[r][v];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      if (t + r >= t1) break;
      Pack<T, V> o;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float pre = bias[v];
#pragma unroll
        for (int j = 0; j < KM; ++j)
          if (K || j >= KM - k) pre = fmaf(w[j][v], s[r + j][v], pre);
        if (d.silu) pre *= sigmoid_f32(pre);
        o.set(v, t + r < len ? pre : 0.f);
      }
      o.store(y + static_cast<long long>(t + r) * d.C);
    }
#pragma unroll
    for (int j = 0; j < KM - 1; ++j)
#pragma unroll
      for (int v = 0; v < V; ++v) s[j][v] = s[j + ROWS][v];
  }
}

// dx (and d state) of a tile need d pre of the tile and of the k - 1 rows behind it, which the thread computes too.
template <typename T, int V, int K>
__global__ void __launch_bounds__(BWD_LANES * BWD_TILES) causal_conv_bwd_kernel(const ConvArgs a, float* partial, int groups) {
  constexpr int KM = K ? K : 8;
  const BdhConvDesc& d = a.d;
  const int k = K ? K : d.k;
  const int cblocks = (a.packs + BWD_LANES - 1) / BWD_LANES;
  const int pack = (blockIdx.x % cblocks) * BWD_LANES + threadIdx.x, group = blockIdx.x / cblocks;
  const bool live = pack < a.packs;
  const int c = pack * V;
  float w[KM][V], bias[V], gw[KM][V], gb[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
#pragma unroll
    for (int j = 0; j < KM; ++j) {
      w[j][v] = (live && j >= KM - k) ? d.w[static_cast<long long>(c + v) * k + j - (KM - k)] : 0.f;
      gw[j][v] = 0.f;
    }
    bias[v] = (live && d.bias) ? d.bias[c + v] : 0.f;
    gb[v] = 0.f;
  }
  const long long all = static_cast<long long>(d.B) * a.tiles;
  for (long long bt = static_cast<long long>(group) * BWD_TILES + threadIdx.y; live && bt < all;
       bt += static_cast<long long>(groups) * BWD_TILES) {
    const int b = static_cast<int>(bt / a.tiles), tile = static_cast<int>(bt % a.tiles);
    const int len = a.len.get(b, d.T);
    const int t0 = tile * a.tile, t1 = min(t0 + a.tile, d.T);
    float s[KM - 1 + ROWS][V], g[KM - 1 + ROWS][V];
#pragma unroll
    for (int j = 0; j < KM - 1; ++j) {
      const Pack<T, V> p = load_seq<T, V>(d, b, t0 - (KM - 1) + j, len, c);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        s[j][v] = p[v];
        g[j][v] = 0.f;
      }
    }
    const int first = (t0 == 0 && d.dstate != nullptr) ? -(k - 1) : t0;      // first row whose gradient this tile writes
    for (int t = t0; t < t1 + k - 1; t += ROWS) {
      Pack<T, V> px[ROWS], pd[ROWS];
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        px[r] = load_seq<T, V>(d, b, t + r, len, c);
        if (t + r < len && t + r < t1 + k - 1)
          pd[r].load(static_cast<const T*>(d.dy) + b * d.dy_sb + (t + r) * d.dy_st + c);
        else
          pd[r].zero();
      }
#pragma unroll
      for (int r = 0; r < ROWS; ++r)
#pragma unroll
        for (int v = 0; v < V; ++v) s[KM - 1 + r][v] = px[r][v];
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        const bool in = t + r < len;
        const bool mine = t + r < t1;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          float gr = pd[r][v];
          if (d.silu) {
            float pre = bias[v];
#pragma unroll
            for (int j = 0; j < KM; ++j)
              if (K || j >= KM - k) pre = fmaf(w[j][v], s[r + j][v], pre);
            const float sg = sigmoid_f32(pre);
            gr *= sg * fmaf(pre, 1.f - sg, 1.f);
          }
          gr = in ? gr : 0.f;
          g[KM - 1 + r][v] = gr;
          if (mine && in) {
            gb[v] += gr;
#pragma unroll
            for (int j = 0; j < KM; ++j)
              if (K || j >= KM - k) gw[j][v] = fmaf(gr, s[r + j][v], gw[j][v]);
          }
        }
        const int row = t + r - (k - 1);                                     // complete now: every d pre it feeds is known
        if (row >= first && row < t1) {
          float o[V];
#pragma unroll
          for (int v = 0; v < V; ++v) {
            o[v] = 0.f;
#pragma unroll
            for (int j = 0; j < KM; ++j)                                     // tap j of output row + (k - 1) - j
              if (K || j >= KM - k) o[v] = fmaf(w[j][v], g[KM - 1 + r - (j - (KM - k))][v], o[v]);
          }
          const int j = row - (len - (k - 1));                               // its place in the new state
          if (d.dstate_out != nullptr && j >= 0 && j < k - 1) {
            Pack<T, V> e;
            e.load(static_cast<const T*>(d.dstate_out) + (static_cast<long long>(b) * (k - 1) + j) * d.C + c);
#pragma unroll
            for (int v = 0; v < V; ++v) o[v] += e[v];
          }
          Pack<T, V> q;
#pragma unroll
          for (int v = 0; v < V; ++v) q.set(v, o[v]);
          if (row >= 0)
            q.store(static_cast<T*>(d.dx) + (static_cast<long long>(b) * d.T + row) * d.C + c);
          else
            q.store(static_cast<T*>(d.dstate) + (static_cast<long long>(b) * (k - 1) + row + k - 1) * d.C + c);
        }
      }
#pragma unroll
      for (int j = 0; j < KM - 1; ++j)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          s[j][v] = s[j + ROWS][v];
          g[j][v] = g[j + ROWS][v];
        }
    }
  }
  if (partial == nullptr) return;
  // partial[group][tap or bias][channel]: the block's four tile rows added up
  __shared__ float sum[BWD_TILES][V][BWD_LANES];
#pragma unroll
  for (int j = 0; j <= KM; ++j) {
    if (j < KM - k) continue;
#pragma unroll
    for (int v = 0; v < V; ++v) sum[threadIdx.y][v][threadIdx.x] = j < KM ? gw[j < KM ? j : 0][v] : gb[v];
    __syncthreads();
    if (threadIdx.y == 0 && live) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float x = 0.f;
#pragma unroll
        for (int y = 0; y < BWD_TILES; ++y) x += sum[y][v][threadIdx.x];
        partial[(static_cast<long long>(group) * (k + 1) + j - (KM - k)) * d.C + c + v] = x;
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
  Pack<T, V> row[8];
#pragma unroll
  for (int j = 0; j < 7; ++j)
    if (j < k - 1) row[j].load(st + j * d.state_sr);
  row[7].load(static_cast<const T*>(d.x) + b * d.x_sb + c);
  float pre[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    pre[v] = d.bias ? d.bias[c + v] : 0.f;
    const float* w = d.w + static_cast<long long>(c + v) * k;
#pragma unroll
    for (int j = 0; j < 7; ++j)
      if (j < k - 1) pre[v] = fmaf(w[j], row[j][v], pre[v]);
    pre[v] = fmaf(w[k - 1], row[7][v], pre[v]);
    if (d.silu) pre[v] *= sigmoid_f32(pre[v]);
  }
  Pack<T, V> o;
#pragma unroll
  for (int v = 0; v < V; ++v) o.set(v, on ? pre[v] : 0.f);
  o.store(static_cast<T*>(d.y) + static_cast<long long>(b) * d.C + c);
  if (on) {
#pragma unroll
    for (int j = 0; j < 7; ++j)
      if (j < k - 1) (j + 1 < k - 1 ? row[j < 6 ? j + 1 : 7] : row[7]).store(so + j * d.state_out_sr);
  } else if (so != st) {
#pragma unroll
    for (int j = 0; j < 7; ++j)
      if (j < k - 1) row[j].store(so + j * d.state_out_sr);
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

// Rows per tile: 64 keeps the rows that two tiles both read at (k - 1) / 64; shorter tiles (not below 8) while there
// are fewer than two waves of threads.
int tile_rows(const BdhConvDesc& d, int packs) {
  int tile = 64;
  while (tile > 8 && static_cast<long long>(d.B) * ((d.T + tile - 1) / tile) * packs < 148LL * 1024) tile /= 2;
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
  // the window of 8 rows in registers: packs of half the bytes
  return fwd_launch<T, (V > 4 ? 4 : V), 0>(d, s);
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

template <typename T>
int fwd_type(const BdhConvDesc& d, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  return packs_fit(d, V, sizeof(T)) ? fwd_width<T, V>(d, s) : fwd_width<T, 1>(d, s);
}
template <typename T>
int bwd_type(const BdhConvDesc& d, float* dw, float* db, float* partial, cudaStream_t s) {
  return packs_fit(d, 4, sizeof(T)) ? bwd_width<T, 4>(d, dw, db, partial, s) : bwd_width<T, 1>(d, dw, db, partial, s);
}
template <typename T>
int step_type(const BdhConvDesc& d, const unsigned char* active, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
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
  for (int v : {1, 4}) {
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
