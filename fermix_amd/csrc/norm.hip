// The norms around a residual block fused with its gate and residual scale, and their gradient:
//   a = norm(h) w1 + b1,  y = x + alpha s g a,  z = norm(y) w2 + b2.
//
// One pass over the rows each way, bound by memory: the forward reads x, h (and g) and writes y
// and z, the gradient reads x, h, dy, dz (and g) and writes dx and dh (and dg); y, a and both
// normed rows are formed again from x and h, which costs nothing next to reading them. A row
// belongs to TPR lanes (a part of a wave, a wave, or several) that hold EPT elements each in
// registers. The column sums (weights, biases, scale, a broadcast gate) stay in registers over all
// the rows that a lane sees, are added over the workgroup's row groups in LDS, and over the
// workgroups by a second launch, each in a fixed order.
//
// MI355X: 4096 x 128 rows of 512, bfloat16, a gate of the sample: 450 us forward (4.8 TB/s; a large copy reaches 5.1),
// 803 us gradient (4.0 TB/s, half of its time in vector instructions); 2000 x 90 rows of 333, float32, layer norm, a
// gate per element: 238 us (5.0 TB/s) and 409 us (4.7 TB/s).
//
// With c = y - mean (or y), r the reciprocal deviation, n = c r and dn = dz w2, the norm's
// gradient is r (dn - n mean(n dn) [- mean(dn)]).
#include "net.h"

namespace fx {
namespace net {
namespace {

struct NormArgs {
  fx_residual_norm p;
  int64_t items;      // samples * chunks
  int64_t chunk_rows;  // rows of an item
  int64_t chunks;     // items of a sample
  float* part;        // workgroups' column sums [quantity][workgroup][columns]
  float* gate_part;   // items' gate sums [item][columns]
};

constexpr int EPT = 8;  // elements of a lane

enum { Q_W1, Q_B1, Q_S, Q_W2, Q_B2, Q_COLUMNS };

// Column of element e of lane t: vectors of V elements, a row's lanes side by side.
template <int V, int TPR>
__device__ __forceinline__ int column(int t, int e) {
  return ((e / V) * TPR + t) * V + e % V;
}

// V: a vector of 16 bytes, aligned to its elements only (rows of odd widths); one access all the same. For float32 rows
// that are not 16-byte aligned single elements (V = 1) are faster, 2000 x 90 rows of 333: 418 us for 481; for
// 16-bit ones they would be two bytes each.
template <class T, int V>
using loose_t = T __attribute__((ext_vector_type(V), aligned(alignof(T))));

// A lane's part of a row as it is in memory, so that the next row's can be on its way while one is worked on.
template <class T, int V, int TPR>
struct Raw {
  vec_t<T, V> v[EPT / V];

  __device__ __forceinline__ void load(const void* base, int64_t at, int t, int C, bool live) {
    const T* p = static_cast<const T*>(base) + at;
#pragma unroll
    for (int i = 0; i < EPT / V; ++i) {
      const int c = column<V, TPR>(t, i * V);
      v[i] = {};
      if (live && c + V <= C) {
        v[i] = *reinterpret_cast<const loose_t<T, V>*>(p + c);
      } else if (live && c < C) {
#pragma unroll
        for (int e = 0; e < V - 1; ++e)
          if (c + e < C) v[i][e] = p[c + e];
      }
    }
  }
  __device__ __forceinline__ void get(float (&x)[EPT]) const {
#pragma unroll
    for (int e = 0; e < EPT; ++e) x[e] = (float)v[e / V][e % V];
  }
};

template <class T, int V, int TPR>
__device__ __forceinline__ void store_row(void* base, int64_t at, int t, int C, const float (&x)[EPT]) {
  T* p = static_cast<T*>(base) + at;
#pragma unroll
  for (int e = 0; e < EPT; e += V) {
    const int c = column<V, TPR>(t, e);
    vec_t<T, V> v;
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = (T)x[e + i];
    if (c + V <= C) {
      *reinterpret_cast<loose_t<T, V>*>(p + c) = v;
    } else if (c < C) {
#pragma unroll
      for (int i = 0; i < V - 1; ++i)
        if (c + i < C) p[c + i] = v[i];
    }
  }
}

// A column vector of wdtype (float32, or T), `none` where it is not given.
template <class T, int V, int TPR>
__device__ __forceinline__ void load_columns(const void* base, bool wide, float none, int t, int C, float (&x)[EPT]) {
#pragma unroll
  for (int e = 0; e < EPT; ++e) {
    const int c = column<V, TPR>(t, e);
    x[e] = none;
    if (base && c < C) x[e] = wide ? static_cast<const float*>(base)[c] : (float)static_cast<const T*>(base)[c];
  }
}

// The gate of a row: per element, or one value.
template <class T, int V, int TPR>
struct RawGate : Raw<T, V, TPR> {
  T one;
  __device__ __forceinline__ void load(const fx_residual_norm& p, int64_t at, int t, bool live) {
    if (!p.gate) return;
    if (p.gc)
      Raw<T, V, TPR>::load(p.gate, at, t, p.columns, live);
    else
      one = live ? static_cast<const T*>(p.gate)[at] : T(0);
  }
  __device__ __forceinline__ void get(const fx_residual_norm& p, float (&g)[EPT]) const {
    if (p.gate && p.gc) {
      Raw<T, V, TPR>::get(g);
    } else {
#pragma unroll
      for (int e = 0; e < EPT; ++e) g[e] = p.gate ? (float)one : 1.0f;
    }
  }
};

// Sum of two values over the TPR lanes of a row; with TPR > 64 through LDS (one row a workgroup,
// every lane calls it).
template <int TPR>
__device__ __forceinline__ float2 row_sum(float2 v, float2* lds) {
  constexpr int W = TPR < 64 ? TPR : 64;
  v.x = group_sum<W>(v.x);
  v.y = group_sum<W>(v.y);
  if constexpr (TPR > 64) {
    __syncthreads();  // the last sum has been read
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < TPR / 64; ++w) {
      v.x += lds[w].x;
      v.y += lds[w].y;
    }
  }
  return v;
}

// x becomes the normed row; mean and reciprocal deviation are returned. The deviation is summed from
// the centred row, so a large mean costs no digits. Columns past C are left 0.
template <class T, int V, int TPR>
__device__ __forceinline__ float2 norm_row(float (&x)[EPT], int t, int C, float inv_c, bool layer, float eps,
                                           float2* lds) {
  float mean = 0.0f;
  if (layer) {
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < EPT; ++e) s += x[e];
    mean = row_sum<TPR>(make_float2(s, 0.0f), lds).x * inv_c;
#pragma unroll
    for (int e = 0; e < EPT; ++e) x[e] = column<V, TPR>(t, e) < C ? x[e] - mean : 0.0f;
  }
  float s = 0.0f;
#pragma unroll
  for (int e = 0; e < EPT; ++e) s += x[e] * x[e];
  const float r = 1.0f / sqrtf(row_sum<TPR>(make_float2(s, 0.0f), lds).x * inv_c + eps);
#pragma unroll
  for (int e = 0; e < EPT; ++e) x[e] *= r;
  return make_float2(mean, r);
}

// One row a workgroup where it takes several waves, else 256 lanes of row groups.
constexpr int norm_threads(int tpr) { return tpr <= 64 ? 256 : tpr; }

template <class T, int V, int TPR>
__global__ __launch_bounds__(norm_threads(TPR)) void norm_kernel(const NormArgs a) {
  constexpr int GROUPS = norm_threads(TPR) / TPR;
  __shared__ float2 lds[TPR > 64 ? TPR / 64 : 1];
  const fx_residual_norm& p = a.p;
  const int t = threadIdx.x % TPR, group = threadIdx.x / TPR, C = p.columns;
  const bool wide = p.wdtype == FX_F32, layer = p.flags & FX_NORM_LAYER;
  const float inv_c = 1.0f / (float)C;
  float w1[EPT], b1[EPT], s[EPT], w2[EPT], b2[EPT];
  load_columns<T, V, TPR>(p.post_weight, wide, 1.0f, t, C, w1);
  load_columns<T, V, TPR>(p.post_bias, wide, 0.0f, t, C, b1);
  load_columns<T, V, TPR>(p.scale, wide, 1.0f, t, C, s);
  load_columns<T, V, TPR>(p.pre_weight, wide, 1.0f, t, C, w2);
  load_columns<T, V, TPR>(p.pre_bias, wide, 0.0f, t, C, b2);
#pragma unroll
  for (int e = 0; e < EPT; ++e) s[e] *= p.alpha;
  const int64_t total = p.samples * p.rows, step = (int64_t)gridDim.x * GROUPS;
  const int64_t ds = step / p.rows, dr = step - ds * p.rows;
  int64_t first = (int64_t)blockIdx.x * GROUPS;
  int64_t sample = (first + group) / p.rows, row = first + group - sample * p.rows;
  Raw<T, V, TPR> rx, rh;
  RawGate<T, V, TPR> rg;
  auto fetch = [&](int64_t s, int64_t r, bool live) {
    rx.load(p.x, s * p.xs + r * p.xr, t, C, live);
    rh.load(p.h, s * p.hs + r * p.hr, t, C, live);
    rg.load(p, s * p.gs + r * p.gr, t, live);
  };
  // Every group of a workgroup makes the same number of turns (the sums over several waves meet at
  // barriers); a turn past the last row works on zeros and stores nothing.
  bool live = first + group < total;
  fetch(sample, row, live);
  while (first < total) {
    float x[EPT], h[EPT], g[EPT];
    rx.get(x);
    rh.get(h);
    rg.get(p, g);
    const int64_t out = sample * p.os + row * p.or_, stat = sample * p.rows + row;
    const bool stores = live;
    first += step;
    sample += ds;
    row += dr;
    if (row >= p.rows) row -= p.rows, ++sample;
    live = first + group < total;
    if (first < total) fetch(sample, row, live);

    float2 s1 = make_float2(0.0f, 1.0f), s2 = make_float2(0.0f, 1.0f);
    if (p.flags & FX_NORM_POST) s1 = norm_row<T, V, TPR>(h, t, C, inv_c, layer, p.eps, lds);
#pragma unroll
    for (int e = 0; e < EPT; ++e) x[e] += s[e] * g[e] * (h[e] * w1[e] + b1[e]);
    if (stores) store_row<T, V, TPR>(p.y, out, t, C, x);
    if (p.flags & FX_NORM_PRE) {
      s2 = norm_row<T, V, TPR>(x, t, C, inv_c, layer, p.eps, lds);
#pragma unroll
      for (int e = 0; e < EPT; ++e) x[e] = x[e] * w2[e] + b2[e];
      if (stores) store_row<T, V, TPR>(p.z, out, t, C, x);
    }
    if (p.stats && stores && t == 0) reinterpret_cast<float4*>(p.stats)[stat] = make_float4(s1.x, s1.y, s2.x, s2.y);
  }
}

// Sums of v over the workgroup's row groups, per column, into out[column].
template <class T, int V, int TPR>
__device__ __forceinline__ void columns_out(const float (&v)[EPT], float* lds, int t, int group, int C, float* out) {
  constexpr int GROUPS = norm_threads(TPR) / TPR;
  if constexpr (GROUPS == 1) {
#pragma unroll
    for (int e = 0; e < EPT; ++e) {
      const int c = column<V, TPR>(t, e);
      if (c < C) out[c] = v[e];
    }
  } else {
    __syncthreads();  // the last quantity has been read
#pragma unroll
    for (int e = 0; e < EPT; ++e) lds[(group * EPT + e) * TPR + t] = v[e];
    __syncthreads();
    // lane (group, t) adds element e of lane t for e = group, group + GROUPS, ..
#pragma unroll
    for (int e0 = 0; e0 < EPT; e0 += GROUPS) {
      const int e = e0 + group;
      if (e < EPT) {
        float sum = 0.0f;
        for (int k = 0; k < GROUPS; ++k) sum += lds[(k * EPT + e) * TPR + t];
        const int c = column<V, TPR>(t, e);
        if (c < C) out[c] = sum;
      }
    }
  }
}

// BIAS: layer norm or a bias; without, the means and the biases' sums do not take registers.
template <class T, int V, int TPR, bool BIAS>
__global__ __launch_bounds__(norm_threads(TPR)) void norm_grad_kernel(const NormArgs a) {
  constexpr int GROUPS = norm_threads(TPR) / TPR;
  __shared__ float2 lds[TPR > 64 ? TPR / 64 : 1];
  __shared__ float sums[GROUPS > 1 ? GROUPS * EPT * TPR : 1];
  const fx_residual_norm& p = a.p;
  const int t = threadIdx.x % TPR, group = threadIdx.x / TPR, C = p.columns;
  const bool wide = p.wdtype == FX_F32, layer = BIAS && (p.flags & FX_NORM_LAYER);
  const bool post = p.flags & FX_NORM_POST, pre = (p.flags & FX_NORM_PRE) && p.grad_z;
  const float inv_c = 1.0f / (float)C;
  float w1[EPT], b1[EPT], s[EPT], w2[EPT];
  load_columns<T, V, TPR>(p.post_weight, wide, 1.0f, t, C, w1);
  load_columns<T, V, TPR>(BIAS ? p.post_bias : nullptr, wide, 0.0f, t, C, b1);
  load_columns<T, V, TPR>(p.scale, wide, 1.0f, t, C, s);
  load_columns<T, V, TPR>(p.pre_weight, wide, 1.0f, t, C, w2);
#pragma unroll
  for (int e = 0; e < EPT; ++e) s[e] *= p.alpha;
  float dw1[EPT], db1[EPT], dsc[EPT], dw2[EPT], db2[EPT];
#pragma unroll
  for (int e = 0; e < EPT; ++e) dw1[e] = db1[e] = dsc[e] = dw2[e] = db2[e] = 0.0f;
  const bool gate_rows = p.gate && p.gr && p.gc;   // a gradient per element
  const bool gate_row = p.gate && p.gr && !p.gc;   // one per row
  const bool gate_sum = p.gate && !p.gr;           // summed over the rows of a sample
  Raw<T, V, TPR> rx, rh, ry = {}, rz = {};  // zero without a cotangent
  RawGate<T, V, TPR> rg;
  float4 rs;
  // a row that is not live is zeros, and adds nothing to any sum
  auto fetch = [&](int64_t sample, int64_t row, bool live) {
    rx.load(p.x, sample * p.xs + row * p.xr, t, C, live);
    rh.load(p.h, sample * p.hs + row * p.hr, t, C, live);
    if (p.grad_y) ry.load(p.grad_y, sample * p.os + row * p.or_, t, C, live);
    if (pre) rz.load(p.grad_z, sample * p.os + row * p.or_, t, C, live);
    rg.load(p, sample * p.gs + row * p.gr, t, live);
    rs = live ? reinterpret_cast<const float4*>(p.stats)[sample * p.rows + row] : make_float4(0.0f, 1.0f, 0.0f, 1.0f);
  };
  for (int64_t item = blockIdx.x; item < a.items; item += gridDim.x) {
    const int64_t sample = item / a.chunks, row0 = (item - sample * a.chunks) * a.chunk_rows;
    const int64_t left = p.rows - row0;
    const int64_t rows = left < a.chunk_rows ? left : a.chunk_rows;
    float dgs[EPT];
#pragma unroll
    for (int e = 0; e < EPT; ++e) dgs[e] = 0.0f;
    bool live = group < rows;
    fetch(sample, row0 + group, live);
    for (int64_t r0 = 0; r0 < rows; r0 += GROUPS) {
      const int64_t row = row0 + r0 + group;
      const int64_t io = sample * p.os + row * p.or_;
      const bool stores = live;
      float x[EPT], h[EPT], dy[EPT], dz[EPT], g[EPT];
      rx.get(x);
      rh.get(h);
      ry.get(dy);
      rz.get(dz);
      rg.get(p, g);
      const float4 st = rs;
      live = r0 + GROUPS + group < rows;
      if (r0 + GROUPS < rows) fetch(sample, row + GROUPS, live);
      // n1 in h, a in x's place of y = x + u a, n2 in x
      float av[EPT];
#pragma unroll
      for (int e = 0; e < EPT; ++e) {
        // past C all is zero, but for what a mean makes of it
        if (post) h[e] = !layer ? h[e] * st.y : column<V, TPR>(t, e) < C ? (h[e] - st.x) * st.y : 0.0f;
        av[e] = h[e] * w1[e] + b1[e];
        x[e] += s[e] * g[e] * av[e];
      }
      float2 m = make_float2(0.0f, 0.0f);
      if (pre) {
#pragma unroll
        for (int e = 0; e < EPT; ++e) {
          x[e] = !layer ? x[e] * st.w : column<V, TPR>(t, e) < C ? (x[e] - st.z) * st.w : 0.0f;
          const float dn = dz[e] * w2[e];
          m.x += dn * x[e];
          m.y += dn;
        }
        m = row_sum<TPR>(m, lds);
        m.x *= inv_c;
        m.y = layer ? m.y * inv_c : 0.0f;
#pragma unroll
        for (int e = 0; e < EPT; ++e) {
          dw2[e] += dz[e] * x[e];
          if (BIAS) db2[e] += dz[e];
          dy[e] += st.w * (dz[e] * w2[e] - x[e] * m.x - m.y);
        }
      }
      if (stores && p.grad_x) store_row<T, V, TPR>(p.grad_x, io, t, C, dy);
      float dg = 0.0f;
      m = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int e = 0; e < EPT; ++e) {
        const float d = layer && column<V, TPR>(t, e) >= C ? 0.0f : dy[e];
        const float du = d * av[e];
        const float dge = du * s[e];
        dg += dge;
        const float da = d * s[e] * g[e];
        dsc[e] += du * g[e];
        dgs[e] += dge;
        if (BIAS) db1[e] += da;
        dw1[e] += da * h[e];
        x[e] = da * w1[e];  // dn1
        m.x += x[e] * h[e];
        m.y += x[e];
        dz[e] = dge;
      }
      if (gate_rows && stores) store_row<T, V, TPR>(p.grad_gate, (sample * p.rows + row) * C, t, C, dz);
      if (post) {
        m = row_sum<TPR>(m, lds);
        m.x *= inv_c;
        m.y = layer ? m.y * inv_c : 0.0f;
#pragma unroll
        for (int e = 0; e < EPT; ++e) x[e] = st.y * (x[e] - h[e] * m.x - m.y);
      }
      if (stores && p.grad_h) store_row<T, V, TPR>(p.grad_h, io, t, C, x);
      if (gate_row) {
        dg = row_sum<TPR>(make_float2(dg, 0.0f), lds).x;
        if (stores && t == 0) static_cast<T*>(p.grad_gate)[sample * p.rows + row] = (T)dg;
      }
    }
    if (gate_sum) columns_out<T, V, TPR>(dgs, sums, t, group, C, a.gate_part + item * C);
  }
#pragma unroll
  for (int e = 0; e < EPT; ++e) dsc[e] *= p.alpha;
  const int64_t plane = (int64_t)gridDim.x * C;
  float* out = a.part + blockIdx.x * (int64_t)C;
  if (p.grad_post_weight) columns_out<T, V, TPR>(dw1, sums, t, group, C, out + Q_W1 * plane);
  if (p.grad_post_bias) columns_out<T, V, TPR>(db1, sums, t, group, C, out + Q_B1 * plane);
  if (p.grad_scale) columns_out<T, V, TPR>(dsc, sums, t, group, C, out + Q_S * plane);
  if (p.grad_pre_weight) columns_out<T, V, TPR>(dw2, sums, t, group, C, out + Q_W2 * plane);
  if (p.grad_pre_bias) columns_out<T, V, TPR>(db2, sums, t, group, C, out + Q_B2 * plane);
}

// The workgroups' column sums added: 16 columns a workgroup, its 64 rows of lanes every 64th part.
constexpr int JOIN_COLUMNS = 16, JOIN_ROWS = 64, JOIN_NT = JOIN_COLUMNS * JOIN_ROWS;
struct JoinArgs {
  const float* part;
  int64_t parts;
  int columns;
  int wide;
  void* out[Q_COLUMNS];
};
template <class T>
__global__ __launch_bounds__(JOIN_NT) void columns_join_kernel(const JoinArgs a) {
  __shared__ double s[JOIN_NT];
  void* const out = a.out[blockIdx.y];
  if (!out) return;
  const int l = threadIdx.x % JOIN_COLUMNS, r = threadIdx.x / JOIN_COLUMNS, c = blockIdx.x * JOIN_COLUMNS + l;
  const float* p = a.part + (int64_t)blockIdx.y * a.parts * a.columns;
  double x = 0.0;
  if (c < a.columns) {
#pragma unroll 8
    for (int64_t i = r; i < a.parts; i += JOIN_ROWS) x += (double)p[i * a.columns + c];
  }
  s[threadIdx.x] = x;
  __syncthreads();
  for (int m = JOIN_ROWS / 2; m; m >>= 1) {
    if (r < m) s[threadIdx.x] += s[threadIdx.x + m * JOIN_COLUMNS];
    __syncthreads();
  }
  if (r == 0 && c < a.columns) {
    x = s[l];
    if (a.wide)
      static_cast<float*>(out)[c] = (float)x;
    else
      static_cast<T*>(out)[c] = (T)x;
  }
}

// The gate's gradient of each sample (or of all: one) from its items' column sums: per column, or (gc == 0) over
// them. Zero without items (no rows).
constexpr int64_t GATE_GROUPS = 1 << 20;  // most workgroups for the samples (a launch's lanes are counted in 32 bits)
template <class T>
__global__ __launch_bounds__(256) void gate_join_kernel(const float* part, int64_t samples, int64_t chunks, int C,
                                                        int gc, T* out) {
  __shared__ double s[256];
  for (int64_t sample = blockIdx.x; sample < samples; sample += gridDim.x) {
    const float* p = part + sample * chunks * C;
    if (gc) {
      for (int c = blockIdx.y * 256 + threadIdx.x; c < C; c += 256 * gridDim.y) {
        double x = 0.0;
        for (int64_t i = 0; i < chunks; ++i) x += (double)p[i * C + c];
        out[sample * C + c] = (T)x;
      }
    } else {
      double x = 0.0;
      for (int64_t i = threadIdx.x; i < chunks * C; i += 256) x += (double)p[i];
      s[threadIdx.x] = x;
      __syncthreads();
      for (int m = 128; m; m >>= 1) {
        if ((int)threadIdx.x < m) s[threadIdx.x] += s[threadIdx.x + m];
        __syncthreads();
      }
      if (threadIdx.x == 0) out[sample] = (T)s[0];
    }
  }
}

// Lanes of a row, eight elements each.
int norm_tpr(int columns) {
  int t = 8;
  while (t < 1024 && t * 8 < columns) t *= 2;
  return t;
}

// Work of the gradient in items of a sample's rows: about two workgroups a CU share
// them. Items never span samples, so that a gate of the sample is summed within them.
struct NormPlan {
  int64_t chunks, chunk_rows, items, groups;
};
NormPlan norm_plan(const fx_residual_norm& p) {
  const int tpr = norm_tpr(p.columns);
  const int64_t per = norm_threads(tpr) / tpr;  // rows at a time
  const int64_t want = tpr >= 1024 ? 512 : 1024;
  int64_t chunks = p.samples >= want ? 1 : cdiv(want, p.samples);
  const int64_t most = cdiv(p.rows, per);
  chunks = chunks < most ? chunks : most;
  NormPlan n;
  n.chunk_rows = cdiv(cdiv(p.rows, chunks), per) * per;
  n.chunks = cdiv(p.rows, n.chunk_rows);
  n.items = p.samples * n.chunks;
  n.groups = n.items < want ? n.items : want;
  return n;
}

bool norm_sizes_ok(const fx_residual_norm* p) {
  return p && p->samples >= 0 && p->rows >= 0 && p->columns >= 1 && p->columns <= FX_MAX_COLUMNS &&
         (p->dtype == FX_F32 || p->dtype == FX_BF16 || p->dtype == FX_F16) &&
         (p->wdtype == FX_F32 || p->wdtype == p->dtype) && (p->gc == 0 || p->gc == 1) && !(p->flags & ~7);
}

bool norm_pointers_ok(const fx_residual_norm& p) {
  const size_t e = dtype_size(p.dtype), w = dtype_size(p.wdtype);
  for (const void* q : {p.x, p.h, p.gate, (const void*)p.y, (const void*)p.z, p.grad_y, p.grad_z,
                        (const void*)p.grad_x, (const void*)p.grad_h, (const void*)p.grad_gate})
    if (!aligned(q, e)) return false;
  for (const void* q : {p.post_weight, p.post_bias, p.scale, p.pre_weight, p.pre_bias,
                        (const void*)p.grad_post_weight, (const void*)p.grad_post_bias, (const void*)p.grad_scale,
                        (const void*)p.grad_pre_weight, (const void*)p.grad_pre_bias})
    if (!aligned(q, w)) return false;
  return p.x && p.h && aligned(p.stats, 16);
}

// Whether some row is not 16-byte aligned.
bool norm_loose(const fx_residual_norm& p) {
  const int64_t v = 16 / (int64_t)dtype_size(p.dtype);
  uintptr_t ptrs = 0;
  for (const void* q : {p.x, p.h, p.gc ? p.gate : nullptr, (const void*)p.y, (const void*)p.z, p.grad_y, p.grad_z,
                        (const void*)p.grad_x, (const void*)p.grad_h, p.gc ? (const void*)p.grad_gate : nullptr})
    ptrs |= (uintptr_t)q;
  int64_t strides = p.columns | p.xs | p.xr | p.hs | p.hr | p.os | p.or_;
  if (p.gate && p.gc) strides |= p.gs | p.gr;
  return (ptrs & 15) || strides % v;
}

// f(elements of a vector, lanes of a row)
template <class T, class F>
void norm_shape(const fx_residual_norm& p, F&& f) {
  auto by_lanes = [&](auto v) {
    switch (norm_tpr(p.columns)) {
      case 8: return f(v, ic<8>{});
      case 16: return f(v, ic<16>{});
      case 32: return f(v, ic<32>{});
      case 64: return f(v, ic<64>{});
      case 128: return f(v, ic<128>{});
      case 256: return f(v, ic<256>{});
      case 512: return f(v, ic<512>{});
      default: return f(v, ic<1024>{});
    }
  };
  if constexpr (sizeof(T) == 4)
    if (norm_loose(p)) return by_lanes(ic<1>{});
  by_lanes(ic<VEC16<T>>{});
}

}  // namespace
}  // namespace net
}  // namespace fx

using namespace fx;
using namespace fx::net;

extern "C" {

int fx_residual_norm_forward(const fx_residual_norm* p, fx_stream_t stream) {
  if (!norm_sizes_ok(p)) return FX_ERR_INVALID_ARGUMENT;
  if (p->samples == 0 || p->rows == 0) return FX_OK;
  if (!norm_pointers_ok(*p) || !p->y || ((p->flags & FX_NORM_PRE) && !p->z)) return FX_ERR_INVALID_ARGUMENT;
  NormArgs a{};
  a.p = *p;
  return with_type<false>(p->dtype, [&](auto t) {
    using T = decltype(t);
    norm_shape<T>(*p, [&](auto v, auto tpr) {
      constexpr int V = decltype(v)::value, TPR = decltype(tpr)::value, NT = norm_threads(TPR);
      const int64_t most = cdiv(p->samples * p->rows, NT / TPR), fit = 256 * 2048 / NT;
      hipLaunchKernelGGL((norm_kernel<T, V, TPR>), dim3((unsigned)(most < fit ? most : fit)), dim3(NT), 0, (hipStream_t)stream, a);
    });
    return launched();
  });
}

size_t fx_residual_norm_grad_workspace(const fx_residual_norm* p) {
  if (!norm_sizes_ok(p) || p->samples == 0 || p->rows == 0) return 0;
  const NormPlan n = norm_plan(*p);
  return sizeof(float) * (size_t)p->columns * (Q_COLUMNS * n.groups + (p->gate && !p->gr ? n.items : 0));
}

int fx_residual_norm_grad(const fx_residual_norm* p, void* workspace, size_t workspace_bytes, fx_stream_t stream) {
  if (!norm_sizes_ok(p)) return FX_ERR_INVALID_ARGUMENT;
  if (p->gate && p->gr && !p->gs && p->samples > 1) return FX_ERR_UNSUPPORTED;  // sums over samples, not rows
  const hipStream_t s = (hipStream_t)stream;
  const bool none = p->samples == 0 || p->rows == 0;
  // values (or rows of columns) of a gate that is summed over the rows: there are some even where there are no rows
  const int64_t gates = !p->gate || p->gr ? 0 : p->gs ? p->samples : 1;
  if (gates && (!p->grad_gate || !aligned(p->grad_gate, dtype_size(p->dtype)))) return FX_ERR_INVALID_ARGUMENT;
  if (!none) {
    if (!norm_pointers_ok(*p) || !p->stats || (p->gate && !p->grad_gate)) return FX_ERR_INVALID_ARGUMENT;
    if (!workspace || !aligned(workspace, 16) || workspace_bytes < fx_residual_norm_grad_workspace(p))
      return FX_ERR_WORKSPACE;
  }
  NormArgs a{};
  a.p = *p;
  NormPlan n{};
  if (!none) n = norm_plan(*p);
  a.items = n.items;
  a.chunks = n.chunks;
  a.chunk_rows = n.chunk_rows;
  a.part = static_cast<float*>(workspace);
  a.gate_part = a.part + Q_COLUMNS * n.groups * p->columns;
  return with_type<false>(p->dtype, [&](auto t) {
    using T = decltype(t);
    if (!none) {
      norm_shape<T>(*p, [&](auto v, auto tpr) {
        constexpr int V = decltype(v)::value, TPR = decltype(tpr)::value;
        const dim3 grid((unsigned)n.groups), block(norm_threads(TPR));
        if ((p->flags & FX_NORM_LAYER) || p->post_bias || p->pre_bias)
          hipLaunchKernelGGL((norm_grad_kernel<T, V, TPR, true>), grid, block, 0, s, a);
        else
          hipLaunchKernelGGL((norm_grad_kernel<T, V, TPR, false>), grid, block, 0, s, a);
      });
      if (launched() != FX_OK) return FX_ERR_LAUNCH;
    }
    JoinArgs j{a.part, n.groups, p->columns, p->wdtype == FX_F32,
               {p->grad_post_weight, p->grad_post_bias, p->grad_scale, p->grad_pre_weight, p->grad_pre_bias}};
    hipLaunchKernelGGL((columns_join_kernel<T>), dim3((p->columns + JOIN_COLUMNS - 1) / JOIN_COLUMNS, Q_COLUMNS),
                       dim3(JOIN_NT), 0, s, j);
    if (gates) {
      const dim3 grid((unsigned)(gates < GATE_GROUPS ? gates : GATE_GROUPS), p->gc ? (p->columns + 255) / 256 : 1);
      hipLaunchKernelGGL((gate_join_kernel<T>), grid, dim3(256), 0, s, a.gate_part, gates, n.items / gates, p->columns,
                         (int)p->gc, static_cast<T*>(p->grad_gate));
    }
    return launched();
  });
}

}  // extern "C"
