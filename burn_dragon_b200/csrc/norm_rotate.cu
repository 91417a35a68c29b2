// RMS norm of every query and key head and its rotation, in one pass and in both directions:
//
//   r = 1 / sqrt(mean x^2 + eps);  v = x r w + b;  (o_2i, o_2i+1) = R(angle_i) (v_2i, v_2i+1) for the first P pairs
//   dv = R^T do;  db = sum dv;  dw = sum dv x r;  dx = r (w dv - x r mean(w dv x r));
//   d angle_i = sum over heads of v_2i dv_2i+1 - v_2i+1 dv_2i                     (a rotation keeps this cross product)
//
// The angle of a token's pair is given, or 2 pi frac(position * freq) with the product in 64 bits (a position of 10^6
// leaves 4 of 24 bits of the fraction in 32). Bound by memory: ~10 (forward) or ~30 operations an element against one
// tensor in and one out (two in, one out). A group of G lanes holds one head's row in registers, so x is read once;
// the sines and cosines of a token are made once per block and shared by its heads through shared memory, because a
// sine and cosine a pair and head would cost more than the rest of the row. Heads of q and k form one list; a block
// takes a slice of it (whole, up to 2048 elements) and steps through the tokens, so that each thread stays with one
// head and the gradients of its weights stay in registers. Sums are fp32, in a fixed order.
#include "bdh_kernels.h"
#include "element_io.cuh"

#include <type_traits>

namespace bdh {
namespace {

constexpr int NT = 256;
constexpr int WARPS = NT / 32;

struct NormArgs {
  BdhNormRotateDesc d;
  Lengths len;
  int tokens;                // B * T
  int H, G, rows;            // heads of q and k; lanes per row; rows per block
  int HS, slices, TS;        // heads per slice; slices; tokens at once
  int shared_w;              // one weight for all heads
};

struct Row {                 // one head of one token
  bool live;                 // it exists
  bool in;                   // and its token is not behind its sequence's length
  int head, h;               // in the joint list; in its tensor
  bool key;
  int b, t;
};

__device__ __forceinline__ Row row_of(const NormArgs& a, int token, int head, bool slot_ok) {
  Row r;
  r.live = slot_ok && head < a.H && token < a.tokens;
  r.head = head;
  r.key = head >= a.d.Hq;
  r.h = r.key ? head - a.d.Hq : head;
  const int tk = r.live ? token : 0;
  r.b = tk / a.d.T;
  r.t = tk - r.b * a.d.T;
  r.in = r.live && r.t < a.len.get(r.b, a.d.T);
  return r;
}

__device__ __forceinline__ long long in_offset(const BdhNormRotateDesc& d, const Row& r) {
  return r.key ? r.b * d.k_sb + r.t * d.k_st + r.h * d.k_sh : r.b * d.q_sb + r.t * d.q_st + r.h * d.q_sh;
}
__device__ __forceinline__ long long out_offset(const BdhNormRotateDesc& d, const Row& r) {
  return ((static_cast<long long>(r.b) * d.T + r.t) * (r.key ? d.Hk : d.Hq) + r.h) * d.Dh;
}

// V elements from column c on, as fp32; columns behind Dh read as 0.
template <typename T, int V, bool VEC>
__device__ __forceinline__ void load_cols(const T* p, int c, int Dh, float (&f)[V]) {
  if constexpr (VEC) {
    Pack<T, V> k;
    if (c < Dh) k.load(p + c); else k.zero();
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = k[i];
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = c + i < Dh ? elem_to_float<T>(p[c + i]) : 0.f;
  }
}

template <typename T, int V, bool VEC>
__device__ __forceinline__ void store_cols(T* p, int c, int Dh, const float (&f)[V]) {
  if constexpr (VEC) {
    if (c >= Dh) return;
    Pack<T, V> k;
#pragma unroll
    for (int i = 0; i < V; ++i) k.set(i, f[i]);
    k.store(p + c);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (c + i < Dh) p[c + i] = elem_from_float<T>(f[i]);
  }
}

__device__ __forceinline__ float group_sum(float v, int G) {
  for (int o = G >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// cs[s][i] = (cos, sin) of pair i of token first + s
__device__ __forceinline__ void fill_angles(const NormArgs& a, float2* cs, int first, int count) {
  const BdhNormRotateDesc& d = a.d;
  for (int s = threadIdx.x >> 5; s < count; s += WARPS) {
    const int token = first + s;
    if (token >= a.tokens) break;
    const int b = token / d.T, t = token - b * d.T;
    if (t >= a.len.get(b, d.T)) continue;                       // (an angle there may be anything; no row uses it)
    double pos = 0;
    if (d.angles == nullptr) {
      const long long at = b * d.pos_sb + t * d.pos_st;
      pos = static_cast<double>(d.positions == nullptr ? d.pos0 + t
                                : d.positions64 ? static_cast<const long long*>(d.positions)[at]
                                                : static_cast<long long>(static_cast<const int*>(d.positions)[at]));
    }
    for (int i = threadIdx.x & 31; i < d.P; i += 32) {
      float sn, c;
      if (d.angles != nullptr) {
        sincosf(d.angles[b * d.ang_sb + t * d.ang_st + i], &sn, &c);
      } else {
        const double turns = pos * static_cast<double>(d.freqs[2 * i]);
        sincospif(2.f * static_cast<float>(turns - floor(turns)), &sn, &c);
      }
      cs[s * d.P + i] = make_float2(c, sn);
    }
  }
}

template <typename T, int V, bool VEC, int NV, int U>
__global__ void __launch_bounds__(NT) norm_rotate_fwd_kernel(const NormArgs a) {
  extern __shared__ float2 cs[];
  const BdhNormRotateDesc& d = a.d;
  const int lane = threadIdx.x % a.G, slot = threadIdx.x / a.G;
  const int ts = slot / a.HS, head = blockIdx.y * a.HS + slot - ts * a.HS;
  const bool slot_ok = slot < a.TS * a.HS;
  const bool key = head >= d.Hq;
  const float* wp = key ? d.k_weight : d.q_weight;
  const float* bp = key ? d.k_bias : d.q_bias;
  const long long w_at = a.shared_w ? 0 : static_cast<long long>(key ? head - d.Hq : head) * d.Dh;
  const bool par = slot_ok && head < a.H;
  float w[NV][V], bias[NV][V];
#pragma unroll
  for (int n = 0; n < NV; ++n)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = (n * a.G + lane) * V + i;
      w[n][i] = (par && wp && c < d.Dh) ? wp[w_at + c] : 1.f;
      bias[n][i] = (par && bp && c < d.Dh) ? bp[w_at + c] : 0.f;
    }
  for (int first = blockIdx.x * a.TS * U; first < a.tokens; first += gridDim.x * a.TS * U) {
    Row r[U];
    float x[U][NV][V];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      r[u] = row_of(a, first + u * a.TS + ts, head, slot_ok);
      const T* p = static_cast<const T*>(r[u].key ? d.k : d.q) + (r[u].in ? in_offset(d, r[u]) : 0);
#pragma unroll
      for (int n = 0; n < NV; ++n) load_cols<T, V, VEC>(p, r[u].in ? (n * a.G + lane) * V : d.Dh, d.Dh, x[u][n]);
    }
    fill_angles(a, cs, first, U * a.TS);
    __syncthreads();
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float ss = 0.f;
#pragma unroll
      for (int n = 0; n < NV; ++n)
#pragma unroll
        for (int i = 0; i < V; ++i) ss = fmaf(x[u][n][i], x[u][n][i], ss);
      const float rs = rsqrtf(group_sum(ss, a.G) / d.Dh + d.eps);
      if (!r[u].live) continue;
      T* o = static_cast<T*>(r[u].key ? d.k_out : d.q_out) + out_offset(d, r[u]);
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        const int c = (n * a.G + lane) * V;
        float f[V];
#pragma unroll
        for (int i = 0; i < V; i += 2) {
          const float v0 = fmaf(x[u][n][i] * rs, w[n][i], bias[n][i]), v1 = fmaf(x[u][n][i + 1] * rs, w[n][i + 1], bias[n][i + 1]);
          const int pair = (c + i) >> 1;
          const float2 e = (r[u].in && pair < d.P) ? cs[(u * a.TS + ts) * d.P + pair] : make_float2(1.f, 0.f);
          f[i] = r[u].in ? v0 * e.x - v1 * e.y : 0.f;
          f[i + 1] = r[u].in ? v1 * e.x + v0 * e.y : 0.f;
        }
        store_cols<T, V, VEC>(o, c, d.Dh, f);
      }
    }
    __syncthreads();
  }
}

// Shared memory: the angles of U * TS tokens; then (DANG) the pairs' cross products of every row, or (at the end) the
// rows' sums for the weights. partial: [2 (weight, bias)][gridDim.x (* slices)][width], see norm_rotate_params_kernel.
template <typename T, int V, bool VEC, int NV, int U>
__global__ void __launch_bounds__(NT) norm_rotate_bwd_kernel(const NormArgs a, float* partial, float* dang, int has_bias) {
  extern __shared__ float2 cs[];
  const BdhNormRotateDesc& d = a.d;
  float* rowbuf = reinterpret_cast<float*>(cs + U * a.TS * d.P);
  const int lane = threadIdx.x % a.G, slot = threadIdx.x / a.G;
  const int ts = slot / a.HS, head = blockIdx.y * a.HS + slot - ts * a.HS;
  const bool slot_ok = slot < a.TS * a.HS;
  const bool key = head >= d.Hq;
  const float* wp = key ? d.k_weight : d.q_weight;
  const float* bp = key ? d.k_bias : d.q_bias;
  const long long w_at = a.shared_w ? 0 : static_cast<long long>(key ? head - d.Hq : head) * d.Dh;
  const bool par = slot_ok && head < a.H;
  float w[NV][V], gw[NV][V], gb[NV][V];
#pragma unroll
  for (int n = 0; n < NV; ++n)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = (n * a.G + lane) * V + i;
      w[n][i] = (par && wp && c < d.Dh) ? wp[w_at + c] : 1.f;
      gw[n][i] = gb[n][i] = 0.f;
    }
  for (int first = blockIdx.x * a.TS * U; first < a.tokens; first += gridDim.x * a.TS * U) {
    Row r[U];
    float x[U][NV][V], g[U][NV][V];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      r[u] = row_of(a, first + u * a.TS + ts, head, slot_ok);
      const T* p = static_cast<const T*>(r[u].key ? d.k : d.q) + (r[u].in ? in_offset(d, r[u]) : 0);
      const T* pd = static_cast<const T*>(r[u].key ? d.dk_out : d.dq_out) + (r[u].in ? out_offset(d, r[u]) : 0);
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        const int c = r[u].in ? (n * a.G + lane) * V : d.Dh;
        load_cols<T, V, VEC>(p, c, d.Dh, x[u][n]);
        load_cols<T, V, VEC>(pd, c, d.Dh, g[u][n]);
      }
    }
    fill_angles(a, cs, first, U * a.TS);
    __syncthreads();
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float ss = 0.f, dot = 0.f;
#pragma unroll
      for (int n = 0; n < NV; ++n)
#pragma unroll
        for (int i = 0; i < V; i += 2) {
          const int pair = ((n * a.G + lane) * V + i) >> 1;
          const float2 e = (r[u].in && pair < d.P) ? cs[(u * a.TS + ts) * d.P + pair] : make_float2(1.f, 0.f);
          const float g0 = g[u][n][i], g1 = g[u][n][i + 1];
          g[u][n][i] = g0 * e.x + g1 * e.y;                     // dv = R^T do
          g[u][n][i + 1] = g1 * e.x - g0 * e.y;
#pragma unroll
          for (int j = i; j < i + 2; ++j) {
            ss = fmaf(x[u][n][j], x[u][n][j], ss);
            dot = fmaf(g[u][n][j] * w[n][j], x[u][n][j], dot);
          }
        }
      const float rs = rsqrtf(group_sum(ss, a.G) / d.Dh + d.eps);
      const float m = group_sum(dot, a.G) / d.Dh * rs * rs;     // mean(w dv x r) r, per element of x
      if (!r[u].live) continue;
      T* o = static_cast<T*>(r[u].key ? d.dk : d.dq) + out_offset(d, r[u]);
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        const int c = (n * a.G + lane) * V;
        float f[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float dv = g[u][n][i], hat = x[u][n][i] * rs;
          f[i] = rs * (dv * w[n][i] - x[u][n][i] * m);
          gw[n][i] = fmaf(dv, hat, gw[n][i]);
          gb[n][i] += dv;
        }
        store_cols<T, V, VEC>(o, c, d.Dh, f);
        if (dang != nullptr) {
#pragma unroll
          for (int i = 0; i < V; i += 2) {
            if (((c + i) >> 1) >= d.P) continue;
            const bool hb = bp != nullptr;
            const float v0 = fmaf(x[u][n][i] * rs, w[n][i], hb ? bp[w_at + c + i] : 0.f);
            const float v1 = fmaf(x[u][n][i + 1] * rs, w[n][i + 1], hb ? bp[w_at + c + i + 1] : 0.f);
            rowbuf[(u * a.rows + slot) * d.P + ((c + i) >> 1)] = r[u].in ? v0 * g[u][n][i + 1] - v1 * g[u][n][i] : 0.f;
          }
        }
      }
    }
    __syncthreads();
    if (dang != nullptr) {
      const int heads = min(a.HS, a.H - static_cast<int>(blockIdx.y) * a.HS);
      for (int s = threadIdx.x >> 5; s < U * a.TS; s += WARPS) {
        const int token = first + s, u = s / a.TS;
        if (token >= a.tokens) break;
        for (int i = threadIdx.x & 31; i < d.P; i += 32) {
          float sum = 0.f;
          for (int h = 0; h < heads; ++h) sum += rowbuf[(u * a.rows + (s - u * a.TS) * a.HS + h) * d.P + i];
          dang[(static_cast<long long>(blockIdx.y) * a.tokens + token) * d.P + i] = sum;
        }
      }
      __syncthreads();
    }
  }
  if (partial == nullptr) return;
  // the block's sums: per head over its token slots, or (one weight for all heads) over the slice's query and key rows
  const int width = a.shared_w ? 2 * d.Dh : a.H * d.Dh;
  const long long lines = static_cast<long long>(gridDim.x) * (a.shared_w ? gridDim.y : 1);
  const long long line = a.shared_w ? static_cast<long long>(blockIdx.x) * gridDim.y + blockIdx.y : blockIdx.x;
  float* buf = reinterpret_cast<float*>(cs);
  for (int what = 0; what < (has_bias ? 2 : 1); ++what) {
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NV; ++n)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int c = (n * a.G + lane) * V + i;
        if (c < d.Dh) buf[slot * d.Dh + c] = what ? gb[n][i] : gw[n][i];
      }
    __syncthreads();
    float* out = partial + (what * lines + line) * width;
    const int heads = min(a.HS, a.H - static_cast<int>(blockIdx.y) * a.HS);
    if (a.shared_w) {
      for (int c = threadIdx.x; c < d.Dh; c += NT) {
        float sq = 0.f, sk = 0.f;
        for (int s = 0; s < a.TS; ++s)
          for (int h = 0; h < heads; ++h) {
            const float v = buf[(s * a.HS + h) * d.Dh + c];
            if (static_cast<int>(blockIdx.y) * a.HS + h >= d.Hq) sk += v; else sq += v;
          }
        out[c] = sq;
        out[d.Dh + c] = sk;
      }
    } else {
      for (int i = threadIdx.x; i < heads * d.Dh; i += NT) {
        float sum = 0.f;
        for (int s = 0; s < a.TS; ++s) sum += buf[s * a.HS * d.Dh + i];
        out[static_cast<long long>(blockIdx.y) * a.HS * d.Dh + i] = sum;
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

NormArgs args_for(const BdhNormRotateDesc& d, int v, int nv) {
  NormArgs a;
  a.d = d;
  a.len = Lengths{d.lengths, d.lengths64};
  a.tokens = d.B * d.T;
  a.H = d.Hq + d.Hk;
  a.G = 1;
  while (a.G * v * nv < d.Dh) a.G *= 2;
  a.rows = NT / a.G;
  a.slices = (a.H + a.rows - 1) / a.rows;
  a.HS = (a.H + a.slices - 1) / a.slices;
  a.TS = a.rows / a.HS;
  a.shared_w = !d.per_head;
  return a;
}

int launched() { return cudaGetLastError() == cudaSuccess ? BDH_OK : BDH_ERR_LAUNCH; }

// Blocks along the tokens: as many as fill the GPU about `waves` times over, so that the weights are loaded (and their
// gradients written) a few times per SM and not once per token.
int token_blocks(const NormArgs& a, int U, int per_sm) {
  const long long need = (static_cast<long long>(a.tokens) + a.TS * U - 1) / (a.TS * U);
  const long long most = (148LL * per_sm + a.slices - 1) / a.slices;
  return static_cast<int>(need < most ? need : most);
}

template <typename T, int V, bool VEC, int NV, int U>
int fwd_launch(const BdhNormRotateDesc& d, cudaStream_t s) {
  const NormArgs a = args_for(d, V, NV);
  const size_t smem = sizeof(float2) * U * a.TS * d.P;
  norm_rotate_fwd_kernel<T, V, VEC, NV, U><<<dim3(token_blocks(a, U, 16), a.slices), NT, smem, s>>>(a);
  return launched();
}

// Four tokens in flight per thread once there are enough of them to fill the GPU that way.
template <typename T, int V, bool VEC, int NV>
int fwd_unroll(const BdhNormRotateDesc& d, cudaStream_t s) {
  if constexpr (NV == 1) {
    const NormArgs a = args_for(d, V, NV);
    if (a.tokens >= 4LL * 148 * a.TS) return fwd_launch<T, V, VEC, NV, 4>(d, s);
  }
  return fwd_launch<T, V, VEC, NV, 1>(d, s);
}

struct BwdOut {
  float *dqw, *dkw, *dqb, *dkb, *dang, *scratch;
};

struct BwdPlan {
  int blocks, width;
  long long lines, partial, angles;     // floats of scratch
  size_t smem;
};

BwdPlan bwd_plan(const NormArgs& a, int U, bool want_w, bool want_b, bool want_ang) {
  BwdPlan p;
  p.blocks = token_blocks(a, U, 6);
  p.width = a.shared_w ? 2 * a.d.Dh : a.H * a.d.Dh;
  p.lines = static_cast<long long>(p.blocks) * (a.shared_w ? a.slices : 1);
  p.partial = (want_w || want_b) ? (want_b ? 2 : 1) * p.lines * p.width : 0;
  p.angles = (want_ang && a.slices > 1) ? static_cast<long long>(a.slices) * a.tokens * a.d.P : 0;
  const size_t cs = sizeof(float2) * U * a.TS * a.d.P;
  const size_t rows = sizeof(float) * a.rows * (want_ang ? U * a.d.P : 0);
  const size_t sums = sizeof(float) * a.rows * a.d.Dh;
  p.smem = cs + rows > sums ? cs + rows : sums;
  return p;
}

template <typename T, int V, bool VEC, int NV, int U>
int bwd_launch(const BdhNormRotateDesc& d, const BwdOut& o, cudaStream_t s) {
  const NormArgs a = args_for(d, V, NV);
  const bool want_b = o.dqb || o.dkb, want_w = o.dqw || o.dkw || want_b;
  const BwdPlan p = bwd_plan(a, U, want_w, want_b, o.dang != nullptr);
  float* partial = want_w ? o.scratch : nullptr;
  float* ang = o.dang ? (p.angles ? o.scratch + p.partial : o.dang) : nullptr;
  auto kernel = norm_rotate_bwd_kernel<T, V, VEC, NV, U>;
  if (p.smem > 48 * 1024 && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(p.smem)) != cudaSuccess)
    return BDH_ERR_LAUNCH;
  kernel<<<dim3(p.blocks, a.slices), NT, p.smem, s>>>(a, partial, ang, want_b);
  if (launched() != BDH_OK) return BDH_ERR_LAUNCH;
  if (want_w) {
    norm_rotate_params_kernel<<<dim3((p.width + 31) / 32, want_b ? 2 : 1), dim3(32, 16), 0, s>>>(
        partial, p.lines, p.width, a.shared_w ? d.Dh : d.Hq * d.Dh, o.dqw, o.dkw, o.dqb, o.dkb);
    if (launched() != BDH_OK) return BDH_ERR_LAUNCH;
  }
  if (p.angles) {
    const long long n = static_cast<long long>(a.tokens) * d.P;
    norm_rotate_angles_kernel<<<static_cast<unsigned>((n + 255) / 256), 256, 0, s>>>(ang, o.dang, n, a.slices);
  }
  return launched();
}

template <typename T, int V, bool VEC, int NV>
int bwd_unroll(const BdhNormRotateDesc& d, const BwdOut& o, cudaStream_t s) {
  if constexpr (NV == 1) {
    const NormArgs a = args_for(d, V, NV);
    if (a.tokens >= 2LL * 148 * a.TS) return bwd_launch<T, V, VEC, NV, 2>(d, o, s);
  }
  return bwd_launch<T, V, VEC, NV, 1>(d, o, s);
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
  if (d.Dh <= 256) return f(std::integral_constant<int, 4>{}, std::false_type{}, std::integral_constant<int, 2>{});
  return f(std::integral_constant<int, 4>{}, std::false_type{}, std::integral_constant<int, 4>{});
}

template <typename T>
int fwd_type(const BdhNormRotateDesc& d, cudaStream_t s) {
  return by_width<T>(d, [&](auto v, auto vec, auto nv) { return fwd_unroll<T, decltype(v)::value, decltype(vec)::value, decltype(nv)::value>(d, s); });
}
template <typename T>
int bwd_type(const BdhNormRotateDesc& d, const BwdOut& o, cudaStream_t s) {
  return by_width<T>(d, [&](auto v, auto vec, auto nv) { return bwd_unroll<T, decltype(v)::value, decltype(vec)::value, decltype(nv)::value>(d, o, s); });
}

}  // namespace
}  // namespace bdh

using namespace bdh;

extern "C" int bdh_norm_rotate_fwd(const BdhNormRotateDesc* d, cudaStream_t s) {
  if (const int rc = checked(*d)) return rc;
  if (static_cast<long long>(d->B) * d->T == 0) return BDH_OK;
  switch (d->dtype) {
    case BDH_F32: return fwd_type<float>(*d, s);
    case BDH_F16: return fwd_type<__half>(*d, s);
  }
  return fwd_type<__nv_bfloat16>(*d, s);
}

// Room for whichever kernel the pointers of the later call select.
extern "C" long long bdh_norm_rotate_scratch(const BdhNormRotateDesc* d, int want_weight, int want_bias, int want_angles) {
  if (d->B < 1 || d->T < 1 || d->Hq < 1 || d->Dh < 2) return 0;
  long long most = 0;
  for (int v : {4, 8})
    for (int nv : {1, 2, 4}) {
      if (32 * v * nv < d->Dh) continue;
      const NormArgs a = args_for(*d, v, nv);
      for (int U : {1, 2}) {
        const BwdPlan p = bwd_plan(a, U, want_weight, want_bias, want_angles);
        most = p.partial + p.angles > most ? p.partial + p.angles : most;
      }
    }
  return most;
}

extern "C" int bdh_norm_rotate_bwd(const BdhNormRotateDesc* d, float* dq_weight, float* dk_weight, float* dq_bias, float* dk_bias,
                                   float* dangles, float* scratch, cudaStream_t s) {
  if (const int rc = checked(*d)) return rc;
  if (static_cast<long long>(d->B) * d->T == 0) return BDH_ERR_ARGUMENT;
  if (dangles != nullptr && d->angles == nullptr) return BDH_ERR_ARGUMENT;
  const BwdOut o{dq_weight, dk_weight, dq_bias, dk_bias, dangles, scratch};
  switch (d->dtype) {
    case BDH_F32: return bwd_type<float>(*d, o, s);
    case BDH_F16: return bwd_type<__half>(*d, o, s);
  }
  return bwd_type<__nv_bfloat16>(*d, o, s);
}
