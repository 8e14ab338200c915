// Relative position bias by distance buckets, and its gradient.
//
// Values: out[b,h,i,j] = table[bucket(k_j - q_i), h]. Bound by the writes. A workgroup takes
// rows (b, i); a lane takes one 16-byte vector of keys, finds its buckets once and writes that
// vector for every head, the table being in LDS by heads so that lanes with different buckets
// read different banks.
//
// Gradient: d table[t, h] = sum of g over the pairs in bucket t. Bound by the reads. Each lane adds
// to sums of its own in LDS, [bucket][lane], so that no two lanes meet in a bank and no order of
// atomics enters the result. The lanes' and then the workgroups' sums are added in a fixed order, in
// double: 256 float32 sums of one sign one after the other would lose two bits, at no less time.
//
// MI355X: 4096 samples of 128 x 128 pairs, float32, values 49 us (5.5 TB/s), gradient 89 us (3.0 TB/s); 8 heads of
// 2048 x 2048, float64, 44 us (6.1 TB/s) and 90 us (3.0 TB/s).
#include "net.h"

namespace fx {
namespace net {
namespace {

constexpr int BIAS_NT = 256;

struct BiasArgs {
  const void* table;  // gradient: the cotangent
  const unsigned char* map;
  int radius, buckets;
  const int *q_pos, *k_pos;
  int64_t batch;
  int heads, nq, nk;
  void* out;  // gradient: the workgroups' sums
  int first, some;  // values: heads of this launch
};

// Bytes of the table that a workgroup of the values' launch holds; further heads take launches of their own.
constexpr int64_t BIAS_TABLE = 64 * 1024;

// How a workgroup of nt lanes goes over the pairs: 2^shift lanes take a row's vectors (of V keys) in turn, the rest
// of it further rows; an item is BIAS_UNROLL x BIAS_TURNS such sets of rows of one sample. A lane's keys
// then stay in registers for all rows of an item, and its rows' loads are in flight together.
constexpr int BIAS_UNROLL = 4, BIAS_TURNS = 4;
struct Tiling {
  int shift, rows, item_rows;
  int64_t items;  // of all samples
  __host__ __device__ Tiling(int nt, int64_t batch, int nq, int chunks) {
    shift = 0;
    while ((1 << shift) < chunks && (2 << shift) <= nt) ++shift;
    rows = nt >> shift;
    item_rows = rows * BIAS_UNROLL * BIAS_TURNS;
    items = batch * ((nq + item_rows - 1) / item_rows);
  }
};

// The map, its entries within the table, into LDS.
__device__ __forceinline__ void stage_map(const BiasArgs& a, unsigned char* map, int nt) {
  for (int i = threadIdx.x; i <= 2 * a.radius; i += nt) map[i] = (unsigned char)min((int)a.map[i], a.buckets - 1);
}

// f(first row, end, first key) for each vector column of each of the workgroup's items; sample b.
template <int V, class F>
__device__ __forceinline__ void for_items(const BiasArgs& a, int nt, F&& f) {
  const int chunks = a.nk / V;
  const Tiling t(nt, a.batch, a.nq, chunks);
  const int per = (a.nq + t.item_rows - 1) / t.item_rows, lane = threadIdx.x & ((1 << t.shift) - 1);
  for (int64_t item = blockIdx.x; item < t.items; item += gridDim.x) {
    const int64_t b = item / per;
    const int r0 = (int)(item - b * per) * t.item_rows, r1 = min(a.nq, r0 + t.item_rows);
    for (int c = lane; c < chunks; c += 1 << t.shift) f(b, r0 + (int)(threadIdx.x >> t.shift), r1, t.rows, c * V);
  }
}

template <int V>
__device__ __forceinline__ void load_keys(const int* p, int (&k)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) k[v] = p[v];
}

// V: elements of a store; 1 where rows of nk elements are not 16-byte aligned.
template <class T, int V>
__global__ __launch_bounds__(BIAS_NT) void bias_kernel(const BiasArgs a) {
  extern __shared__ __align__(16) unsigned char smem[];
  T* tab = reinterpret_cast<T*>(smem);  // [head][bucket]
  unsigned char* map = smem + (size_t)a.some * a.buckets * sizeof(T);
  const T* table = static_cast<const T*>(a.table) + a.first;
  for (int i = threadIdx.x; i < a.some * a.buckets; i += BIAS_NT)
    tab[i] = table[(int64_t)(i % a.buckets) * a.heads + i / a.buckets];
  stage_map(a, map, BIAS_NT);
  __syncthreads();
  for_items<V>(a, BIAS_NT, [&](int64_t b, int first, int end, int step, int key) {
    int k[V];
    load_keys<V>(a.k_pos + b * a.nk + key, k);
    const int* qp = a.q_pos + b * a.nq;
    T* const out = static_cast<T*>(a.out) + (b * a.heads + a.first) * a.nq * (int64_t)a.nk + key;
#pragma unroll 2
    for (int i = first; i < end; i += step) {
      const int q = qp[i];
      int bucket[V];
#pragma unroll
      for (int v = 0; v < V; ++v) bucket[v] = distance_bucket(map, a.radius, k[v], q);
      T* o = out + (int64_t)i * a.nk;
      for (int h = 0; h < a.some; ++h, o += (int64_t)a.nq * a.nk) {
        vec_t<T, V> x;
#pragma unroll
        for (int v = 0; v < V; ++v) x[v] = tab[h * a.buckets + bucket[v]];
        *reinterpret_cast<vec_t<T, V>*>(o) = x;
      }
    }
  });
}

template <class T>
struct acc_of {
  using type = float;
};
template <>
struct acc_of<double> {
  using type = double;
};

// One head a workgroup row (blockIdx.y); W waves.
template <class T, int V, int W>
__global__ __launch_bounds__(64 * W) void bias_grad_kernel(const BiasArgs a) {
  using A = typename acc_of<T>::type;
  extern __shared__ __align__(16) unsigned char smem[];
  A* sums = reinterpret_cast<A*>(smem);  // [wave][bucket][lane]
  unsigned char* map = smem + (size_t)W * a.buckets * 64 * sizeof(A);
  for (int i = threadIdx.x; i < W * a.buckets * 64; i += 64 * W) sums[i] = A(0);
  stage_map(a, map, 64 * W);
  __syncthreads();
  A* mine = sums + (threadIdx.x >> 6) * a.buckets * 64 + (threadIdx.x & 63);
  const int h = blockIdx.y;
  for_items<V>(a, 64 * W, [&](int64_t b, int first, int end, int step, int key) {
    int k[V];
    load_keys<V>(a.k_pos + b * a.nk + key, k);
    const int* qp = a.q_pos + b * a.nq;
    const T* g = static_cast<const T*>(a.table) + (b * a.heads + h) * a.nq * (int64_t)a.nk + key;
    vec_t<T, V> x[BIAS_UNROLL], y[BIAS_UNROLL];
    int q[BIAS_UNROLL], r[BIAS_UNROLL];
    // rows from i on; a row past the end adds zeros
    auto fetch = [&](int i, vec_t<T, V>(&to)[BIAS_UNROLL], int(&pos)[BIAS_UNROLL]) {
#pragma unroll
      for (int u = 0; u < BIAS_UNROLL; ++u) {
        const int at = i + u * step;
        to[u] = {};
        pos[u] = qp[min(at, end - 1)];
        if (at < end) to[u] = *reinterpret_cast<const vec_t<T, V>*>(g + (int64_t)at * a.nk);
      }
    };
    if (first < end) fetch(first, y, r);
    for (int i = first; i < end; i += BIAS_UNROLL * step) {
#pragma unroll
      for (int u = 0; u < BIAS_UNROLL; ++u) x[u] = y[u], q[u] = r[u];
      if (i + BIAS_UNROLL * step < end) fetch(i + BIAS_UNROLL * step, y, r);  // on their way while these are added
      int t[BIAS_UNROLL * V];
#pragma unroll
      for (int j = 0; j < BIAS_UNROLL * V; ++j) t[j] = distance_bucket(map, a.radius, k[j % V], q[j / V]);
#pragma unroll
      for (int j = 0; j < BIAS_UNROLL * V; j += 2)
        add_pair(mine, t[j], (A)x[j / V][j % V], t[j + 1], (A)x[(j + 1) / V][(j + 1) % V]);
    }
  });
  __syncthreads();
  A* out = static_cast<A*>(a.out) + ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * a.buckets;
  for (int t = threadIdx.x; t < a.buckets; t += 64 * W) {
    double s[4] = {};  // four chains, so that an add does not wait for the one before it
    for (int w = 0; w < W; ++w)
#pragma unroll 4
      for (int l = 0; l < 64; ++l) s[l & 3] += (double)sums[(w * a.buckets + t) * 64 + ((l + t) & 63)];  // rotated: no shared bank
    out[t] = (A)((s[0] + s[1]) + (s[2] + s[3]));
  }
}

// table gradient [bucket][head] = the sum over n parts of part[head][part][bucket], in double.
template <class T, class A>
__global__ __launch_bounds__(BIAS_NT) void bucket_join_kernel(const A* part, int64_t n, int buckets, int heads,
                                                              T* out) {
  const int t = blockIdx.y, h = blockIdx.x;
  __shared__ double s[BIAS_NT];
  double x = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += BIAS_NT) x += (double)part[((int64_t)h * n + i) * buckets + t];
  s[threadIdx.x] = x;
  __syncthreads();
  for (int m = BIAS_NT / 2; m; m >>= 1) {
    if ((int)threadIdx.x < m) s[threadIdx.x] += s[threadIdx.x + m];
    __syncthreads();
  }
  if (threadIdx.x == 0) out[(int64_t)t * heads + h] = (T)s[0];
}

int bias_waves(int buckets) { return buckets <= 32 ? 4 : buckets <= 64 ? 2 : 1; }

// Workgroups of a head in the gradient: about what the card holds at once, with as many items each.
int64_t bias_grad_groups(int buckets, int64_t batch, int heads, int nq, int nk, int v) {
  const int64_t items = Tiling(64 * bias_waves(buckets), batch, nq, nk / v).items;
  return cdiv(items, cdiv(items, cdiv(1280, heads)));
}

int bias_vec(int nk, size_t size, const void* p) {
  const int v = (int)(16 / size);
  return nk % v == 0 && aligned(p, 16) ? v : 1;
}

bool bias_sizes_ok(int32_t radius, int32_t buckets, int64_t batch, int32_t heads, int32_t nq, int32_t nk,
                   int32_t dtype) {
  return radius >= 0 && radius <= FX_MAX_RADIUS && buckets >= 1 && buckets <= 256 && batch >= 0 && heads >= 1 &&
         heads <= FX_MAX_BIAS_HEADS && nq >= 0 && nq <= FX_MAX_POSITIONS && nk >= 0 && nk <= FX_MAX_POSITIONS &&
         dtype_size(dtype);
}

}  // namespace

int launch_bucket_join(const float* part, int64_t n, int buckets, int heads, float* out, hipStream_t s) {
  hipLaunchKernelGGL((bucket_join_kernel<float, float>), dim3(heads, buckets), dim3(BIAS_NT), 0, s, part, n, buckets,
                     heads, out);
  return launched();
}

}  // namespace net
}  // namespace fx

using namespace fx;
using namespace fx::net;

extern "C" {

int fx_relative_bias(const void* table, const uint8_t* map, int32_t radius, int32_t buckets, const int32_t* q_pos,
                     const int32_t* k_pos, int64_t batch, int32_t heads, int32_t nq, int32_t nk, int32_t dtype,
                     void* out, fx_stream_t stream) {
  if (!bias_sizes_ok(radius, buckets, batch, heads, nq, nk, dtype)) return FX_ERR_INVALID_ARGUMENT;
  const size_t size = dtype_size(dtype);
  if (batch == 0 || nq == 0 || nk == 0) return FX_OK;
  if (!table || !map || !q_pos || !k_pos || !out || !aligned(table, size) || !aligned(out, size) ||
      !aligned(q_pos, 4) || !aligned(k_pos, 4))
    return FX_ERR_INVALID_ARGUMENT;
  BiasArgs a{table, map, radius, buckets, q_pos, k_pos, batch, heads, nq, nk, out};
  const int at_once = (int)(BIAS_TABLE / (buckets * size));
  return with_type<true>(dtype, [&](auto t) {
    using T = decltype(t);
    constexpr int V = VEC16<T>;
    const int v = bias_vec(nk, sizeof(T), out);
    const int64_t most = Tiling(BIAS_NT, batch, nq, nk / v).items;
    const unsigned grid = (unsigned)(most < 4096 ? most : 4096);
    for (a.first = 0; a.first < heads; a.first += at_once) {
      a.some = heads - a.first < at_once ? heads - a.first : at_once;
      const size_t lds = (size_t)a.some * buckets * sizeof(T) + 2 * radius + 1;
      if (v == V)
        hipLaunchKernelGGL((bias_kernel<T, V>), dim3(grid), dim3(BIAS_NT), lds, (hipStream_t)stream, a);
      else
        hipLaunchKernelGGL((bias_kernel<T, 1>), dim3(grid), dim3(BIAS_NT), lds, (hipStream_t)stream, a);
    }
    return launched();
  });
}

size_t fx_relative_bias_grad_workspace(int32_t buckets, int64_t batch, int32_t heads, int32_t nq, int32_t nk,
                                       int32_t dtype) {
  if (!bias_sizes_ok(0, buckets, batch, heads, nq, nk, dtype) || batch == 0 || nq == 0 || nk == 0) return 0;
  // of whichever way to load has the more workgroups: the pointer decides
  const int v = (int)(16 / dtype_size(dtype));
  const int64_t single = bias_grad_groups(buckets, batch, heads, nq, nk, 1);
  const int64_t whole = nk % v ? 0 : bias_grad_groups(buckets, batch, heads, nq, nk, v);
  return (size_t)(single > whole ? single : whole) * heads * buckets * (dtype == FX_F64 ? 8 : 4);
}

int fx_relative_bias_grad(const void* grad_out, const uint8_t* map, int32_t radius, int32_t buckets,
                          const int32_t* q_pos, const int32_t* k_pos, int64_t batch, int32_t heads, int32_t nq,
                          int32_t nk, int32_t dtype, void* grad_table, void* workspace, size_t workspace_bytes,
                          fx_stream_t stream) {
  if (!bias_sizes_ok(radius, buckets, batch, heads, nq, nk, dtype)) return FX_ERR_INVALID_ARGUMENT;
  const size_t size = dtype_size(dtype);
  if (!grad_table || !aligned(grad_table, size)) return FX_ERR_INVALID_ARGUMENT;
  const bool none = batch == 0 || nq == 0 || nk == 0;
  if (!none) {
    if (!grad_out || !map || !q_pos || !k_pos || !aligned(grad_out, size) || !aligned(q_pos, 4) || !aligned(k_pos, 4))
      return FX_ERR_INVALID_ARGUMENT;
    if (!workspace || !aligned(workspace, 16) ||
        workspace_bytes < fx_relative_bias_grad_workspace(buckets, batch, heads, nq, nk, dtype))
      return FX_ERR_WORKSPACE;
  }
  const hipStream_t s = (hipStream_t)stream;
  return with_type<true>(dtype, [&](auto t) {
    using T = decltype(t);
    using A = typename acc_of<T>::type;
    int64_t groups = 0;
    if (!none) {
      const int v = bias_vec(nk, sizeof(T), grad_out);
      const BiasArgs a{grad_out, map, radius, buckets, q_pos, k_pos, batch, heads, nq, nk, workspace, 0, heads};
      const int w = bias_waves(buckets);
      groups = bias_grad_groups(buckets, batch, heads, nq, nk, v);
      const size_t lds = (size_t)w * buckets * 64 * sizeof(A) + 2 * radius + 1;
      const dim3 grid((unsigned)groups, heads);
      auto go = [&](auto vv, auto ww) {
        constexpr int V = decltype(vv)::value, W = decltype(ww)::value;
        hipLaunchKernelGGL((bias_grad_kernel<T, V, W>), grid, dim3(64 * W), lds, s, a);
      };
      auto by_waves = [&](auto vv) {
        if (w == 4)
          go(vv, ic<4>{});
        else if (w == 2)
          go(vv, ic<2>{});
        else
          go(vv, ic<1>{});
      };
      if (v == 1)
        by_waves(ic<1>{});
      else
        by_waves(ic<VEC16<T>>{});
      const int st = launched();
      if (st != FX_OK) return st;
    }
    hipLaunchKernelGGL((bucket_join_kernel<T, A>), dim3(heads, buckets), dim3(BIAS_NT), 0, s,
                       static_cast<const A*>(workspace), groups, buckets, heads, static_cast<T*>(grad_table));
    return launched();
  });
}

}  // extern "C"
