// Relative position bias by distance buckets, and its gradient.
//
// Values: out[b,h,i,j] = table[bucket(k_j - q_i), h]. Bound by the writes. A workgroup takes
// rows (b, i); a lane takes one 16-byte vector of keys, finds its buckets once and writes that
// vector for every head, the table being in LDS by heads so that lanes with different buckets
// read different banks.
//
// Gradient: d table[t, h] = sum of g over the pairs in bucket t. Bound by the reads. Each lane adds
// to sums of its own in LDS, [bucket][lane], so that no two lanes meet in a bank and no order of
// atomics enters the result: a wave's LDS operations complete in the order of issue. The lanes' and
// then the workgroups' sums are added in a fixed order, the last in double.
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
};

// The vectors (sample b, row i, first key V chunk) that a thread takes, in steps of the whole
// grid: the divisions are made once, a step only adds with carries.
struct Walk {
  int64_t b;
  int i, chunk;  // chunk = first key / V
  int64_t db;
  int di, dchunk;
  int nq, chunks;

  __device__ __forceinline__ Walk(int64_t first, int64_t step, int nq_, int chunks_) : nq(nq_), chunks(chunks_) {
    const int64_t row = first / chunks, drow = step / chunks;
    chunk = (int)(first - row * chunks);
    dchunk = (int)(step - drow * chunks);
    b = row / nq;
    i = (int)(row - b * nq);
    db = drow / nq;
    di = (int)(drow - db * nq);
  }
  __device__ __forceinline__ void next() {
    chunk += dchunk;
    const int c = chunk >= chunks;
    chunk -= c ? chunks : 0;
    i += di + c;
    const int d = i >= nq;
    i -= d ? nq : 0;
    b += db + d;
  }
};

__device__ __forceinline__ void stage_map(const BiasArgs& a, unsigned char* map) {
  for (int i = threadIdx.x; i <= 2 * a.radius; i += BIAS_NT) map[i] = a.map[i];
}

// V: elements of a store; 1 where rows of nk elements are not 16-byte aligned.
template <class T, int V>
__global__ __launch_bounds__(BIAS_NT) void bias_kernel(const BiasArgs a) {
  extern __shared__ __align__(16) unsigned char smem[];
  T* tab = reinterpret_cast<T*>(smem);  // [head][bucket]
  unsigned char* map = smem + (size_t)a.heads * a.buckets * sizeof(T);
  const T* table = static_cast<const T*>(a.table);
  for (int i = threadIdx.x; i < a.heads * a.buckets; i += BIAS_NT)
    tab[i] = table[(i % a.buckets) * a.heads + i / a.buckets];
  stage_map(a, map);
  __syncthreads();
  T* out = static_cast<T*>(a.out);
  for (Walk w((int64_t)blockIdx.x * BIAS_NT + threadIdx.x, (int64_t)gridDim.x * BIAS_NT, a.nq, a.nk / V); w.b < a.batch;
       w.next()) {
    const int q = a.q_pos[w.b * a.nq + w.i];
    const int* kp = a.k_pos + w.b * a.nk + w.chunk * V;
    int bucket[V];
#pragma unroll
    for (int v = 0; v < V; ++v) bucket[v] = distance_bucket(map, a.radius, a.buckets, kp[v], q);
    T* o = out + ((w.b * a.heads) * a.nq + w.i) * (int64_t)a.nk + w.chunk * V;
    for (int h = 0; h < a.heads; ++h, o += (int64_t)a.nq * a.nk) {
      vec_t<T, V> x;
#pragma unroll
      for (int v = 0; v < V; ++v) x[v] = tab[h * a.buckets + bucket[v]];
      *reinterpret_cast<vec_t<T, V>*>(o) = x;
    }
  }
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
  for (int i = threadIdx.x; i <= 2 * a.radius; i += 64 * W) map[i] = a.map[i];
  __syncthreads();
  A* mine = sums + (threadIdx.x >> 6) * a.buckets * 64 + (threadIdx.x & 63);
  const int h = blockIdx.y;
  const T* g = static_cast<const T*>(a.table);
  for (Walk w((int64_t)blockIdx.x * 64 * W + threadIdx.x, (int64_t)gridDim.x * 64 * W, a.nq, a.nk / V); w.b < a.batch;
       w.next()) {
    const int q = a.q_pos[w.b * a.nq + w.i];
    const int* kp = a.k_pos + w.b * a.nk + w.chunk * V;
    const vec_t<T, V> x =
        *reinterpret_cast<const vec_t<T, V>*>(g + ((w.b * a.heads + h) * a.nq + w.i) * (int64_t)a.nk + w.chunk * V);
#pragma unroll
    for (int v = 0; v < V; ++v)
      unsafeAtomicAdd(mine + distance_bucket(map, a.radius, a.buckets, kp[v], q) * 64, (A)x[v]);
  }
  __syncthreads();
  A* out = static_cast<A*>(a.out) + ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * a.buckets;
  for (int t = threadIdx.x; t < a.buckets; t += 64 * W) {
    A s = A(0);
    for (int w = 0; w < W; ++w)
      for (int l = 0; l < 64; ++l) s += sums[(w * a.buckets + t) * 64 + ((l + t) & 63)];  // rotated: no shared bank
    out[t] = s;
  }
}

// table gradient [bucket][head] = the sum over n parts of part[head][part][bucket], in double.
template <class T, class A>
__global__ __launch_bounds__(BIAS_NT) void bucket_join_kernel(const A* part, int64_t n, int buckets, int heads,
                                                              T* out) {
  const int t = blockIdx.x, h = blockIdx.y;
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

// Workgroups of a head in the gradient: as many as fit the card twice over, none with less than
// one vector a lane.
int64_t bias_grad_groups(int buckets, int64_t rows, int heads, int nk, int v) {
  const int64_t nt = 64 * bias_waves(buckets);
  const int64_t most = cdiv(rows * cdiv(nk, v), nt);
  const int64_t fit = cdiv(2048, heads);
  return most < fit ? most : fit;
}

int bias_vec(int nk, size_t size, const void* p) {
  const int v = (int)(16 / size);
  return nk % v == 0 && aligned(p, 16) ? v : 1;
}

bool bias_sizes_ok(int32_t radius, int32_t buckets, int64_t batch, int32_t heads, int32_t nq, int32_t nk,
                   int32_t dtype) {
  return radius >= 0 && radius <= FX_MAX_RADIUS && buckets >= 1 && buckets <= 256 && batch >= 0 && heads >= 1 &&
         heads <= 4096 && nq >= 0 && nk >= 0 && dtype_size(dtype);
}

}  // namespace

int launch_bucket_join(const float* part, int64_t n, int buckets, int heads, float* out, hipStream_t s) {
  hipLaunchKernelGGL((bucket_join_kernel<float, float>), dim3(buckets, heads), dim3(BIAS_NT), 0, s, part, n, buckets,
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
  if ((size_t)heads * buckets * size > 64 * 1024) return FX_ERR_UNSUPPORTED;
  if (batch == 0 || nq == 0 || nk == 0) return FX_OK;
  if (!table || !map || !q_pos || !k_pos || !out || !aligned(table, size) || !aligned(out, size) ||
      !aligned(q_pos, 4) || !aligned(k_pos, 4))
    return FX_ERR_INVALID_ARGUMENT;
  const BiasArgs a{table, map, radius, buckets, q_pos, k_pos, batch, heads, nq, nk, out};
  return with_type<true>(dtype, [&](auto t) {
    using T = decltype(t);
    constexpr int V = VEC16<T>;
    const int v = bias_vec(nk, sizeof(T), out);
    const int64_t most = cdiv(batch * nq * cdiv(nk, v), BIAS_NT);
    const unsigned grid = (unsigned)(most < 4096 ? most : 4096);
    const size_t lds = (size_t)heads * buckets * sizeof(T) + 2 * radius + 1;
    if (v == V)
      hipLaunchKernelGGL((bias_kernel<T, V>), dim3(grid), dim3(BIAS_NT), lds, (hipStream_t)stream, a);
    else
      hipLaunchKernelGGL((bias_kernel<T, 1>), dim3(grid), dim3(BIAS_NT), lds, (hipStream_t)stream, a);
    return launched();
  });
}

size_t fx_relative_bias_grad_workspace(int32_t buckets, int64_t batch, int32_t heads, int32_t nq, int32_t nk,
                                       int32_t dtype) {
  if (!bias_sizes_ok(0, buckets, batch, heads, nq, nk, dtype) || batch == 0 || nq == 0 || nk == 0) return 0;
  // of the scalar kernel, which has the most workgroups
  return (size_t)bias_grad_groups(buckets, batch * nq, heads, nk, 1) * heads * buckets * (dtype == FX_F64 ? 8 : 4);
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
      const BiasArgs a{grad_out, map, radius, buckets, q_pos, k_pos, batch, heads, nq, nk, workspace};
      const int w = bias_waves(buckets);
      groups = bias_grad_groups(buckets, batch * nq, heads, nk, v);
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
    hipLaunchKernelGGL((bucket_join_kernel<T, A>), dim3(buckets, heads), dim3(BIAS_NT), 0, s,
                       static_cast<const A*>(workspace), groups, buckets, heads, static_cast<T*>(grad_table));
    return launched();
  });
}

}  // extern "C"
