// Attention of one new token a sample over a paged key-value cache, with the relative position bias.
//
// Bound by reading the cache once. A workgroup takes one kv head of a sample and a part of its
// tokens; the LPT lanes that hold a 16-byte vector each make up a token's row, a wave reads 64 / LPT
// tokens at a time, four times over, straight into registers (K and V are used once, LDS would
// only delay them). The lanes of a row add up its scores for all the heads that share it; each row
// position of the wave keeps a running maximum and sum of its own, joined at the end. Where there are
// few samples the tokens are split over workgroups (as evenly as the sample's own length allows), whose
// sums a second launch joins.
#include "net.h"

namespace fx {
namespace net {
namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float F32_MAX = 3.402823466e38f;
constexpr int STEP_WAVES = 4, STEP_NT = 64 * STEP_WAVES;

struct StepArgs {
  fx_attention_step p;
  int splits, vec;
  int unit;         // a part's tokens are a multiple of this
  uint32_t magic;   // token / page_size = (token magic) >> shift for tokens below 2^31
  int shift;
  float* part;      // [batch][heads][splits][dim]
  float2* stat;     // [batch][heads][splits]: maximum and sum
};

// A bias in units of log2 e; finite entries stay finite.
__device__ __forceinline__ float log2_bias(float b) {
  const float x = b * LOG2E;
  return isinf(b) || !(fabsf(x) > F32_MAX) ? x : copysignf(F32_MAX, b);
}

template <class T, int DP, int G>
__global__ __launch_bounds__(STEP_NT) void step_kernel(const StepArgs a) {
  constexpr int V = VEC16<T>, LPT = DP / V, ROWS = 64 / LPT, U = 4;
  extern __shared__ __align__(16) unsigned char smem[];
  const fx_attention_step& p = a.p;
  float* const acc_lds = reinterpret_cast<float*>(smem);           // [wave][G][DP]
  float2* const stat_lds = reinterpret_cast<float2*>(acc_lds + STEP_WAVES * G * DP);  // [wave][G]
  float* const tab = reinterpret_cast<float*>(stat_lds + STEP_WAVES * G);             // [G][buckets]
  unsigned char* const map = reinterpret_cast<unsigned char*>(tab + G * p.buckets);

  const int group = p.heads / p.kv_heads, blocks = (group + G - 1) / G;
  const int split = blockIdx.x;
  const int kh = blockIdx.y / blocks, h0 = kh * group + (blockIdx.y % blocks) * G;
  const int heads = min(G, group - (int)(blockIdx.y % blocks) * G);
  const int64_t b = blockIdx.z;
  const int len = p.lengths[b];
  const int n = p.k ? (len < 0 ? 0 : len == 0x7fffffff ? len : len + 1) : max(len, 0);  // tokens attended to
  const bool over = (int64_t)n > (int64_t)p.max_pages * p.page_size;
  int per = (int)(((int64_t)n + a.splits - 1) / a.splits);
  per = (int)min((int64_t)n, ((int64_t)per + a.unit - 1) / a.unit * a.unit);
  const int64_t t0 = (int64_t)split * per, t1 = over ? 0 : min((int64_t)n, t0 + per);
  const int64_t row0 = (b * p.heads + h0) * a.splits + split;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, part = lane % LPT, d0 = part * V;
  if (t0 >= t1 && a.splits > 1 && !over) {
    if ((int)threadIdx.x < heads) a.stat[row0 + (int64_t)threadIdx.x * a.splits] = make_float2(-INFINITY, 0.0f);
    return;
  }
  if (p.table) {
    for (int i = threadIdx.x; i < heads * p.buckets; i += STEP_NT)
      tab[i] = log2_bias(p.table[(int64_t)(i % p.buckets) * p.heads + h0 + i / p.buckets]);
    for (int i = threadIdx.x; i <= p.radius; i += STEP_NT) map[i] = (unsigned char)min((int)p.map[i], p.buckets - 1);
  }
  float q[G][V], acc[G][V], m[G], l[G];
  const float c = p.scale * LOG2E;
#pragma unroll
  for (int g = 0; g < G; ++g) {
    m[g] = -INFINITY;
    l[g] = 0.0f;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      acc[g][e] = 0.0f;
      q[g][e] = g < heads && d0 + e < p.dim ? c * (float)static_cast<const T*>(p.q)[(b * p.heads + h0 + g) * p.dim + d0 + e] : 0.0f;
    }
  }
  bool bad = over;
  __syncthreads();

  const int64_t row_size = (int64_t)p.kv_heads * p.dim;
  const T* const kc = static_cast<const T*>(p.k_cache) + (int64_t)kh * p.dim;
  const T* const vc = static_cast<const T*>(p.v_cache) + (int64_t)kh * p.dim;
  const int* const table = p.page_table + b * p.max_pages;
  auto load = [&](const T* src, float (&x)[V]) {
    if (a.vec) {
      vec_t<T, V> v = {};
      if (d0 < p.dim) v = *reinterpret_cast<const vec_t<T, V>*>(src + d0);
#pragma unroll
      for (int e = 0; e < V; ++e) x[e] = (float)v[e];
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) x[e] = d0 + e < p.dim ? (float)src[d0 + e] : 0.0f;
    }
  };
  for (int64_t base = t0 + wave * ROWS; base < t1; base += STEP_WAVES * ROWS * U) {
    float k[U][V], v[U][V];
    bool on[U];
    int dist[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t t = base + u * STEP_WAVES * ROWS + lane / LPT;
      on[u] = t < t1;
      dist[u] = (int)(t - (n - 1));
#pragma unroll
      for (int e = 0; e < V; ++e) k[u][e] = v[u][e] = 0.0f;
      if (!on[u]) continue;
      const T *ks, *vs;
      const uint32_t pg = (uint32_t)(((uint64_t)(uint32_t)t * a.magic) >> a.shift);
      const int page = table[pg];
      const bool ok = (uint32_t)page < (uint64_t)p.pages;
      if (!ok) {
        bad = true;
        continue;
      }
      const int64_t slot = ((int64_t)page * p.page_size + ((uint32_t)t - pg * (uint32_t)p.page_size)) * row_size;
      if (p.k && t == n - 1) {
        // the new token: from the call, and into the cache once (by the group's first heads)
        ks = static_cast<const T*>(p.k) + (b * p.kv_heads + kh) * p.dim;
        vs = static_cast<const T*>(p.v) + (b * p.kv_heads + kh) * p.dim;
        if (blockIdx.y % blocks == 0) {
#pragma unroll
          for (int e = 0; e < V; ++e)
            if (d0 + e < p.dim) {
              static_cast<T*>(p.k_cache)[slot + (int64_t)kh * p.dim + d0 + e] = ks[d0 + e];
              static_cast<T*>(p.v_cache)[slot + (int64_t)kh * p.dim + d0 + e] = vs[d0 + e];
            }
        }
      } else {
        ks = kc + slot;
        vs = vc + slot;
      }
      load(ks, k[u]);
      load(vs, v[u]);
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
      if (g >= heads) break;
      float s[U], top = m[g];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float x = 0.0f;
#pragma unroll
        for (int e = 0; e < V; ++e) x += q[g][e] * k[u][e];
        x = group_sum<LPT>(x);
        if (p.table && on[u]) x += tab[g * p.buckets + map[max(dist[u], -p.radius) + p.radius]];
        s[u] = on[u] ? x : -INFINITY;
        top = fmaxf(top, s[u]);
      }
      const float at = top == -INFINITY ? 0.0f : top;
      const float keep = __builtin_amdgcn_exp2f(m[g] - at);
      m[g] = top;
      l[g] *= keep;
#pragma unroll
      for (int e = 0; e < V; ++e) acc[g][e] *= keep;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float w = __builtin_amdgcn_exp2f(s[u] - at);
        l[g] += w;
#pragma unroll
        for (int e = 0; e < V; ++e) acc[g][e] += w * v[u][e];
      }
    }
  }

  // the wave's row positions, then the waves
#pragma unroll
  for (int g = 0; g < G; ++g) {
    float top = m[g];
#pragma unroll
    for (int x = LPT; x < 64; x <<= 1) top = fmaxf(top, shfl_xor(top, x));
    const float at = top == -INFINITY ? 0.0f : top;
    const float keep = __builtin_amdgcn_exp2f(m[g] - at);
    l[g] *= keep;
#pragma unroll
    for (int x = LPT; x < 64; x <<= 1) l[g] += shfl_xor(l[g], x);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      acc[g][e] *= keep;
#pragma unroll
      for (int x = LPT; x < 64; x <<= 1) acc[g][e] += shfl_xor(acc[g][e], x);
      if (lane < LPT) acc_lds[(wave * G + g) * DP + d0 + e] = acc[g][e];
    }
    if (lane == 0) stat_lds[wave * G + g] = make_float2(top, l[g]);
  }
  const bool any_bad = __syncthreads_or(bad);
  for (int i = threadIdx.x; i < heads * DP; i += STEP_NT) {
    const int g = i / DP, d = i % DP;
    float top = -INFINITY, sum = 0.0f, x = 0.0f;
    for (int w = 0; w < STEP_WAVES; ++w) top = fmaxf(top, stat_lds[w * G + g].x);
    for (int w = 0; w < STEP_WAVES; ++w) {
      const float f = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(stat_lds[w * G + g].x - top);
      sum += f * stat_lds[w * G + g].y;
      x += f * acc_lds[(w * G + g) * DP + d];
    }
    if (any_bad) x = sum = NAN;
    if (d >= p.dim) continue;
    if (a.splits == 1) {
      static_cast<T*>(p.out)[(b * p.heads + h0 + g) * p.dim + d] = (T)(sum == 0.0f ? 0.0f : x / sum);
    } else {
      const int64_t r = row0 + (int64_t)g * a.splits;
      a.part[r * p.dim + d] = x;
      if (d == 0) a.stat[r] = make_float2(any_bad ? NAN : top, sum);
    }
  }
}

// One row of heads x dim a wave: the parts in order.
template <class T>
__global__ __launch_bounds__(STEP_NT) void step_join_kernel(const StepArgs a) {
  const int64_t row = (int64_t)blockIdx.x * STEP_WAVES + (threadIdx.x >> 6);
  if (row >= a.p.batch * a.p.heads) return;
  const float2* st = a.stat + row * a.splits;
  float top = -INFINITY;
  bool bad = false;
  for (int i = 0; i < a.splits; ++i) {
    bad |= st[i].x != st[i].x;
    top = fmaxf(top, st[i].x);
  }
  for (int d = threadIdx.x & 63; d < a.p.dim; d += 64) {
    float x = 0.0f, sum = 0.0f;
    for (int i = 0; i < a.splits; ++i) {
      if (st[i].y == 0.0f) continue;
      const float f = __builtin_amdgcn_exp2f(st[i].x - top);
      sum += f * st[i].y;
      x += f * a.part[(row * a.splits + i) * a.p.dim + d];
    }
    if (bad) x = sum = NAN;
    static_cast<T*>(a.p.out)[row * a.p.dim + d] = (T)(sum == 0.0f ? 0.0f : x / sum);
  }
}

bool step_sizes_ok(const fx_attention_step* p) {
  if (!p || p->batch < 0 || p->heads < 1 || p->kv_heads < 1 || p->heads % p->kv_heads || p->dim < 1 || p->dim > 128 ||
      p->pages < 0 || p->page_size < 1 || p->max_pages < 0)
    return false;
  if (p->dtype != FX_F32 && p->dtype != FX_BF16 && p->dtype != FX_F16) return false;
  if (!(p->scale > 0.0f) || !(p->scale <= F32_MAX)) return false;
  return p->table ? p->buckets >= 1 && p->buckets <= FX_MAX_ATTENTION_BUCKETS && p->radius >= 0 && p->radius <= FX_MAX_RADIUS
                  : p->buckets == 0 && p->radius == 0;
}

int step_heads(int group) { return group >= 3 ? 4 : group; }  // heads that a workgroup takes at once

// Parts of a sample's tokens: enough workgroups for the card, none under 256 tokens of the longest sample
// that the table can hold.
int step_splits(const fx_attention_step& p) {
  const int group = p.heads / p.kv_heads;
  const int64_t rows = p.batch * p.kv_heads * cdiv(group, step_heads(group));
  const int64_t want = cdiv(1024, rows), most = cdiv((int64_t)p.max_pages * p.page_size, 256);
  const int64_t s = want < most ? want : most;
  return (int)(s < 1 ? 1 : s);
}

int64_t step_part_floats(const fx_attention_step& p, int splits) {
  return cdiv(p.batch * p.heads * splits * p.dim, 4) * 4;
}

}  // namespace
}  // namespace net
}  // namespace fx

using namespace fx;
using namespace fx::net;

extern "C" {

size_t fx_attention_step_workspace(const fx_attention_step* p) {
  if (!step_sizes_ok(p) || p->batch == 0) return 0;
  const int splits = step_splits(*p);
  if (splits == 1) return 0;
  return sizeof(float) * (size_t)(step_part_floats(*p, splits) + 2 * p->batch * p->heads * splits);
}

int fx_attention_step_run(const fx_attention_step* p, void* workspace, size_t workspace_bytes, fx_stream_t stream) {
  if (!step_sizes_ok(p) || !p->k != !p->v) return FX_ERR_INVALID_ARGUMENT;
  if (p->batch == 0) return FX_OK;
  const bool cache = p->pages > 0 && p->max_pages > 0;
  if (!p->q || !p->out || !p->lengths || (p->table && !p->map) ||
      (cache && (!p->k_cache || !p->v_cache || !p->page_table)))
    return FX_ERR_INVALID_ARGUMENT;
  const size_t e = dtype_size(p->dtype);
  for (const void* x : {p->q, p->k, p->v, (const void*)p->k_cache, (const void*)p->v_cache, (const void*)p->out})
    if (!aligned(x, e)) return FX_ERR_INVALID_ARGUMENT;
  for (const void* x : {(const void*)p->lengths, (const void*)p->page_table, (const void*)p->table})
    if (!aligned(x, 4)) return FX_ERR_INVALID_ARGUMENT;
  const int splits = step_splits(*p);
  if (splits > 1 && (!workspace || !aligned(workspace, 16) || workspace_bytes < fx_attention_step_workspace(p)))
    return FX_ERR_WORKSPACE;
  const int group = p->heads / p->kv_heads, per = step_heads(group);
  const int64_t rows = p->kv_heads * cdiv(group, per);
  if (rows > 65535 || (int64_t)p->max_pages * p->page_size > 0x7fffffff) return FX_ERR_UNSUPPORTED;

  StepArgs a{};
  a.p = *p;
  a.splits = splits;
  a.unit = 64;
  a.vec = p->dim % (16 / (int)e) == 0 && aligned(p->k_cache, 16) && aligned(p->v_cache, 16) && aligned(p->k, 16) &&
          aligned(p->v, 16);
  int bits = 0;  // ceil(log2 page_size)
  while ((1ll << bits) < p->page_size) ++bits;
  a.shift = 31 + bits;
  a.magic = (uint32_t)(((1ull << a.shift) + p->page_size - 1) / p->page_size);
  a.part = static_cast<float*>(workspace);
  a.stat = reinterpret_cast<float2*>(a.part + step_part_floats(*p, splits));
  const hipStream_t s = (hipStream_t)stream;
  return with_type<false>(p->dtype, [&](auto t) {
    using T = decltype(t);
    // the batch goes on a grid dimension of at most 65535
    for (int64_t b0 = 0; b0 < p->batch; b0 += 65535) {
      StepArgs c = a;
      const int64_t nb = p->batch - b0 < 65535 ? p->batch - b0 : 65535;
      const int64_t e = (int64_t)sizeof(T);
      auto add = [](const void* x, int64_t bytes) { return x ? (const void*)((const char*)x + bytes) : nullptr; };
      c.p.batch = nb;
      c.p.q = add(p->q, b0 * p->heads * p->dim * e);
      c.p.k = add(p->k, b0 * p->kv_heads * p->dim * e);
      c.p.v = add(p->v, b0 * p->kv_heads * p->dim * e);
      c.p.out = (void*)add(p->out, b0 * p->heads * p->dim * e);
      c.p.lengths = p->lengths + b0;
      if (p->page_table) c.p.page_table = p->page_table + b0 * p->max_pages;
      auto go = [&](auto dp, auto g) {
        constexpr int DP = decltype(dp)::value, G = decltype(g)::value;
        const size_t lds = 4 * STEP_WAVES * G * DP + 8 * STEP_WAVES * G + 4 * (size_t)G * p->buckets + p->radius + 1;
        hipLaunchKernelGGL((step_kernel<T, DP, G>), dim3(splits, (unsigned)rows, (unsigned)nb), dim3(STEP_NT), lds, s, c);
      };
      auto by_heads = [&](auto dp) {
        if (per == 1)
          go(dp, ic<1>{});
        else if (per == 2)
          go(dp, ic<2>{});
        else
          go(dp, ic<4>{});
      };
      if (p->dim <= 16)
        by_heads(ic<16>{});
      else if (p->dim <= 32)
        by_heads(ic<32>{});
      else if (p->dim <= 64)
        by_heads(ic<64>{});
      else
        by_heads(ic<128>{});
      if (launched() != FX_OK) return FX_ERR_LAUNCH;
      if (splits > 1)
        hipLaunchKernelGGL((step_join_kernel<T>), dim3((unsigned)cdiv(nb * p->heads, STEP_WAVES)), dim3(STEP_NT), 0, s, c);
    }
    return launched();
  });
}

}  // extern "C"
