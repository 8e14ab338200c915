// Attention of one new token a sample over a paged key-value cache, with the relative position bias.
//
// Bound by reading the cache once. The LPT lanes that hold a 16-byte vector each make up a token's row, a wave
// reads 64 / LPT tokens at a time, four times over, straight into registers (K and V are used once, LDS
// would only delay them), with the next tokens' rows and the page numbers after those already on their way.
// The lanes of a row add up its scores for all the heads that share it; each row position of the wave keeps a
// running maximum and sum of its own, joined at the end by lane moves.
//
// Heads that share K and V, 16-bit types (step_mma_kernel): up to sixteen heads are the columns of 16 x 16 products,
// S^T = K q^T with K straight from memory, then O^T = V^T P^T with V through LDS of the wave's own for its column
// reads; a lane has one head's scores of eight tokens in registers. Whatever the heads, the work is that of one pass.
//
// With many samples a wave takes a kv head of a sample by itself. With few, four waves take it together, and
// where that is not enough either its tokens are split over workgroups (as evenly as the sample's own length
// allows), whose sums a second launch joins.
//
// MI355X: 4096 samples x 8 heads, 64 .. 128 tokens, head dimension 32, bfloat16, 118 us (3.3 TB/s, vector instructions
// half of it); 4 samples of 32 heads on 8, 32768 .. 65536 tokens, head dimension 128, 160 + 10 us (5.0 TB/s; a large
// copy reaches 5.1); float32, 48 samples of 6 heads on 2, up to 2000 tokens, 26 + 4 us.
//
// The order of all sums depends on sizes and lengths alone.
#include "attention.h"

namespace fx {
namespace net {
namespace {

constexpr int STEP_WAVES = 4, STEP_NT = 64 * STEP_WAVES;

struct StepArgs {
  fx_attention_step p;
  int splits, vec;
  int unit;         // a part's tokens are a multiple of this
  uint32_t magic;   // token / page_size = the high word of token magic, >> shift, for tokens below 2^31 (page_size > 1)
  int shift;
  uint32_t row_size, page_elements;
  float* part;      // [batch][heads][splits][dim]
  float2* stat;     // [batch][heads][splits]: maximum and sum
  int sums_bytes, stat_at;  // step_mma_kernel's LDS: the V tiles (then the waves' sums, statistics at stat_at)
};

// A bias in units of log2 e; finite entries stay finite.
__device__ __forceinline__ float log2_bias(float b) {
  const float x = b * LOG2E;
  return isinf(b) || !(fabsf(x) > F32_MAX) ? x : copysignf(F32_MAX, b);
}

// First element of a token's row in the cache, -1 for a page outside it: three 32-bit products (a 64-bit address
// calculation for each token costs as much as the token's scores).
__device__ __forceinline__ int64_t token_slot(const StepArgs& a, const int* pages, uint32_t t) {
  const uint32_t pg = a.p.page_size == 1 ? t : __umulhi(t, a.magic) >> a.shift;
  const uint32_t page = (uint32_t)pages[pg];
  if ((uint64_t)page >= (uint64_t)a.p.pages) return -1;
  return (int64_t)((uint64_t)page * a.page_elements + (t - pg * (uint32_t)a.p.page_size) * a.row_size);
}

template <int V, class T>
__device__ __forceinline__ void widen(const vec_t<T, V>& x, float (&y)[V]) {
#pragma unroll
  for (int e = 0; e < V; ++e) y[e] = (float)x[e];
}

// A token's vector of this lane; elements past dim are zero.
template <class T>
__device__ __forceinline__ vec_t<T, VEC16<T>> load_part(const T* row, int d0, int dim, bool vec) {
  constexpr int V = VEC16<T>;
  vec_t<T, V> x = {};
  if (vec) {
    if (d0 < dim) x = *reinterpret_cast<const vec_t<T, V>*>(row + d0);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (d0 + e < dim) x[e] = row[d0 + e];
  }
  return x;
}

// G: heads at a time. W: waves that share a unit (a block of G heads of a kv head of a sample), 1 or 4.
template <class T, int DP, int G, int W>
__global__ __launch_bounds__(STEP_NT, 3) void step_kernel(const StepArgs a) {
  constexpr int V = VEC16<T>, LPT = DP / V, ROWS = 64 / LPT, U = W == 1 ? 2 : 4, STRIDE = W * ROWS * U;
  extern __shared__ __align__(16) unsigned char smem[];
  const fx_attention_step& p = a.p;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, mine = W == 1 ? wave : 0;
  float* const acc_lds = reinterpret_cast<float*>(smem);                                 // [wave][G][DP] (W > 1)
  float2* const stat_lds = reinterpret_cast<float2*>(acc_lds + (W > 1 ? W * G * DP : 0));  // [wave][G] (W > 1)
  float* const tabs = reinterpret_cast<float*>(stat_lds + (W > 1 ? W * G : 0));            // [unit][G][buckets]
  unsigned char* const map = reinterpret_cast<unsigned char*>(tabs + (W == 1 ? STEP_WAVES : 1) * G * p.buckets);
  float* const tab = tabs + mine * G * p.buckets;

  const int group = p.heads / p.kv_heads, blocks = (group + G - 1) / G, units = p.kv_heads * blocks;
  const int split = blockIdx.x, unit = min(units - 1, W == 1 ? (int)blockIdx.y * STEP_WAVES + wave : (int)blockIdx.y);
  const bool spare = W == 1 && (int)blockIdx.y * STEP_WAVES + wave >= units;  // a wave without a unit
  const int kh = unit / blocks, h0 = kh * group + (unit % blocks) * G, heads = min(G, group - (unit % blocks) * G);
  const int64_t b = blockIdx.z;
  const int len = p.lengths[b];
  const int n = p.k ? (len < 0 ? 0 : len == 0x7fffffff ? len : len + 1) : max(len, 0);  // tokens attended to
  const bool over = (int64_t)n > (int64_t)p.max_pages * p.page_size;
  int per = (int)(((int64_t)n + a.splits - 1) / a.splits);
  per = (int)min((int64_t)n, ((int64_t)per + a.unit - 1) / a.unit * a.unit);
  // tokens from here on in 32 bits: all are below 2^31, and what is added to them is small
  const uint32_t t0 = (uint32_t)min((int64_t)n, (int64_t)split * per), t1 = over ? 0u : (uint32_t)min((int64_t)n, (int64_t)t0 + per);
  const int64_t row0 = (b * p.heads + h0) * a.splits + split;
  const int part = lane % LPT, d0 = part * V, row = lane / LPT;
  if (t0 >= t1 && a.splits > 1 && !over) {
    if ((int)threadIdx.x < heads) a.stat[row0 + (int64_t)threadIdx.x * a.splits] = make_float2(-INFINITY, 0.0f);
    return;
  }

  const bool own = p.k && t1 == (uint32_t)n && n > 0;  // this part has the new token, which is in the call, not the cache
  const uint32_t end = own ? t1 - 1 : t1;              // of the cached tokens
  const T* const kc = static_cast<const T*>(p.k_cache) + (int64_t)kh * p.dim;
  const T* const vc = static_cast<const T*>(p.v_cache) + (int64_t)kh * p.dim;
  const int* const table = p.page_table + b * p.max_pages;
  bool bad = over;
  const uint32_t first = t0 + (W == 1 ? 0 : wave * ROWS * U);
  int64_t slot[U];
  vec_t<T, V> k[U], v[U], nk[U], nv[U];
  auto find = [&](uint32_t base) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t t = base + u * ROWS + row;
      slot[u] = -1;
      if (t < end) {
        slot[u] = token_slot(a, table, t);
        if (slot[u] < 0) bad = true;
      }
    }
  };
  auto fetch = [&](vec_t<T, V>(&x)[U], vec_t<T, V>(&y)[U]) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      x[u] = y[u] = {};
      if (slot[u] >= 0) {
        x[u] = load_part<T>(kc + slot[u], d0, p.dim, a.vec);
        y[u] = load_part<T>(vc + slot[u], d0, p.dim, a.vec);
      }
    }
  };
  find(first);
  if (W > 1) {
    fetch(k, v);
    find(first + STRIDE);
  }

  if (p.table) {
    const int at = W == 1 ? lane : threadIdx.x, nt = W == 1 ? 64 : STEP_NT;
    for (int i = at; i < heads * p.buckets; i += nt)
      tab[i] = log2_bias(p.table[(int64_t)(i % p.buckets) * p.heads + h0 + i / p.buckets]);
    for (int i = threadIdx.x; i <= p.radius; i += STEP_NT) map[i] = (unsigned char)min((int)p.map[i], p.buckets - 1);
  }
  float q[G][V], acc[G][V], m[G], l[G];
  const float c = p.scale * LOG2E;
#pragma unroll
  for (int g = 0; g < G; ++g) {
    m[g] = -INFINITY;
    l[g] = 0.0f;
    vec_t<T, V> x = {};
    if (g < heads) x = load_part<T>(static_cast<const T*>(p.q) + (b * p.heads + h0 + g) * p.dim, d0, p.dim, false);
    widen<V>(x, q[g]);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      acc[g][e] = 0.0f;
      q[g][e] *= c;
    }
  }
  __syncthreads();

  if (own && !spare) {
    // the new token: into the cache (by the first wave of the kv head's first heads), and the start of the sums
    // of the wave's first row position
    const int64_t at = (b * p.kv_heads + kh) * p.dim;
    const vec_t<T, V> xk = load_part<T>(static_cast<const T*>(p.k) + at, d0, p.dim, false);
    const vec_t<T, V> xv = load_part<T>(static_cast<const T*>(p.v) + at, d0, p.dim, false);
    const int64_t to = token_slot(a, table, n - 1);
    if (to < 0) bad = true;
    if (W == 1 || wave == 0) {
      if (to >= 0 && unit % blocks == 0 && row == 0) {
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (d0 + e < p.dim) {
            static_cast<T*>(p.k_cache)[to + (int64_t)kh * p.dim + d0 + e] = xk[e];
            static_cast<T*>(p.v_cache)[to + (int64_t)kh * p.dim + d0 + e] = xv[e];
          }
      }
      float kf[V], vf[V];
      widen<V>(xk, kf);
      widen<V>(xv, vf);
#pragma unroll
      for (int g = 0; g < G; ++g) {
        if (g >= heads) break;
        float x = 0.0f;
#pragma unroll
        for (int e = 0; e < V; ++e) x += q[g][e] * kf[e];
        x = group_sum<LPT>(x);
        if (p.table) x += tab[g * p.buckets + map[p.radius]];
        if (row == 0 && x != -INFINITY) {
          m[g] = x;
          l[g] = 1.0f;
#pragma unroll
          for (int e = 0; e < V; ++e) acc[g][e] = vf[e];
        }
      }
    }
  }

  for (uint32_t base = first; base < end; base += STRIDE) {
    if (W > 1) {
      fetch(nk, nv);
      find(base + 2 * STRIDE);
    } else {
      fetch(k, v);
      find(base + STRIDE);
    }
    float s[U][G];
    int dist[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float kf[V];
      widen<V>(k[u], kf);
      dist[u] = max((int)(base + u * ROWS + row - (n - 1)), -p.radius) + p.radius;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        float x = 0.0f;
#pragma unroll
        for (int e = 0; e < V; ++e) x += q[g][e] * kf[e];
        s[u][g] = group_sum<LPT>(x);
      }
    }
    if (p.table) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int t = map[min(dist[u], p.radius)];
#pragma unroll
        for (int g = 0; g < G; ++g)
          if (g < heads) s[u][g] += tab[g * p.buckets + t];
      }
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float top = m[g];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (base + u * ROWS + row >= end) s[u][g] = -INFINITY;
        top = fmaxf(top, s[u][g]);
      }
      const float at = top == -INFINITY ? 0.0f : top;
      const float keep = __builtin_amdgcn_exp2f(m[g] - at);
      m[g] = top;
      l[g] *= keep;
#pragma unroll
      for (int e = 0; e < V; ++e) acc[g][e] *= keep;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        s[u][g] = __builtin_amdgcn_exp2f(s[u][g] - at);
        l[g] += s[u][g];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float vf[V];
      widen<V>(v[u], vf);
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int e = 0; e < V; ++e) acc[g][e] += s[u][g] * vf[e];
      if (W > 1) {
        k[u] = nk[u];
        v[u] = nv[u];
      }
    }
  }

  // the wave's row positions
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const float top = stride_join<LPT, MaxOp>(m[g]);
    const float keep = __builtin_amdgcn_exp2f(m[g] - (top == -INFINITY ? 0.0f : top));
    m[g] = top;
    l[g] = stride_join<LPT, AddOp>(l[g] * keep);
#pragma unroll
    for (int e = 0; e < V; ++e) acc[g][e] = stride_join<LPT, AddOp>(acc[g][e] * keep);
  }
  if constexpr (W == 1) {
    bad = __any(bad);
    if (spare || row != 0) return;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      if (g >= heads) break;
      const float inv = bad ? NAN : l[g] == 0.0f ? 0.0f : 1.0f / l[g];
      T* o = static_cast<T*>(p.out) + (b * p.heads + h0 + g) * p.dim + d0;
      vec_t<T, V> x;
#pragma unroll
      for (int e = 0; e < V; ++e) x[e] = (T)(acc[g][e] * inv);
      if (a.vec) {
        if (d0 < p.dim) *reinterpret_cast<vec_t<T, V>*>(o) = x;
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (d0 + e < p.dim) o[e] = x[e];
      }
    }
    return;
  } else {
#pragma unroll
    for (int g = 0; g < G; ++g) {
      if (row == 0) {
#pragma unroll
        for (int e = 0; e < V; ++e) acc_lds[(wave * G + g) * DP + d0 + e] = acc[g][e];
      }
      if (lane == 0) stat_lds[wave * G + g] = make_float2(m[g], l[g]);
    }
    const bool any_bad = __syncthreads_or(bad);
    for (int i = threadIdx.x; i < heads * DP; i += STEP_NT) {
      const int g = i / DP, d = i % DP;
      float top = -INFINITY, sum = 0.0f, x = 0.0f;
      for (int w = 0; w < W; ++w) top = fmaxf(top, stat_lds[w * G + g].x);
      for (int w = 0; w < W; ++w) {
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
}

typedef float v4f_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ v4f_t mma16(vec_t<__bf16, 8> a, vec_t<__bf16, 8> b, v4f_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ v4f_t mma16(vec_t<_Float16, 8> a, vec_t<_Float16, 8> b, v4f_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

constexpr int STEP_TOKENS = 32, STEP_HEADS = 16;

// Lane l = 16 g + c. K operand: token c (and 16 + c), elements 32 s + 8 g ..; scores: head c, tokens 4 g + r and
// 16 + 4 g + r; these, rounded, are the second product's operand; V is stored as Tile has it and read by columns.
template <class T, int DP, int W>
__global__ __launch_bounds__(STEP_NT, 2) void step_mma_kernel(const StepArgs a) {
  constexpr int KS = DP / 32, DB = DP / 16, S = Tile<T, DP>::STRIDE;
  using V8 = vec_t<T, 8>;
  extern __shared__ __align__(16) unsigned char smem[];
  const fx_attention_step& p = a.p;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
  T* const vt = reinterpret_cast<T*>(smem) + wave * STEP_TOKENS * S;  // [token][dim]
  float* const tabs = reinterpret_cast<float*>(smem + a.sums_bytes);  // [unit][bucket][STEP_HEADS]
  unsigned char* const map = reinterpret_cast<unsigned char*>(tabs + (W == 1 ? STEP_WAVES : 1) * STEP_HEADS * p.buckets);
  float* const tab = tabs + (W == 1 ? wave : 0) * STEP_HEADS * p.buckets;

  const int group = p.heads / p.kv_heads, blocks = (group + STEP_HEADS - 1) / STEP_HEADS, units = p.kv_heads * blocks;
  const int at_unit = W == 1 ? (int)blockIdx.y * STEP_WAVES + wave : (int)blockIdx.y, unit = min(units - 1, at_unit);
  const bool spare = at_unit >= units;  // a wave without a unit
  const int kh = unit / blocks, h0 = kh * group + (unit % blocks) * STEP_HEADS;
  const int heads = min(STEP_HEADS, group - (unit % blocks) * STEP_HEADS);
  const int split = blockIdx.x;
  const int64_t b = blockIdx.z;
  const int len = p.lengths[b];
  const int n = p.k ? (len < 0 ? 0 : len == 0x7fffffff ? len : len + 1) : max(len, 0);  // tokens attended to
  const bool over = (int64_t)n > (int64_t)p.max_pages * p.page_size;
  int per = (int)(((int64_t)n + a.splits - 1) / a.splits);
  per = (int)min((int64_t)n, ((int64_t)per + a.unit - 1) / a.unit * a.unit);
  // tokens from here on in 32 bits: all are below 2^31, and what is added to them is small
  const uint32_t t0 = (uint32_t)min((int64_t)n, (int64_t)split * per), t1 = over ? 0u : (uint32_t)min((int64_t)n, (int64_t)t0 + per);
  const int64_t row0 = (b * p.heads + h0) * a.splits + split;
  if (t0 >= t1 && a.splits > 1 && !over) {
    if ((int)threadIdx.x < heads) a.stat[row0 + (int64_t)threadIdx.x * a.splits] = make_float2(-INFINITY, 0.0f);
    return;
  }

  const T* const kc = static_cast<const T*>(p.k_cache) + (int64_t)kh * p.dim;
  const T* const vc = static_cast<const T*>(p.v_cache) + (int64_t)kh * p.dim;
  const int64_t new_row = (b * p.kv_heads + kh) * p.dim;
  const int* const table = p.page_table + b * p.max_pages;
  bool bad = over;
  V8 k[2][KS], v[2][KS];
  int64_t slot[2];
  // the next tokens' places in the cache; -1 without one
  auto find = [&](uint32_t base) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint32_t at = base + 16 * t + c;
      slot[t] = -1;
      if (at < t1) {
        slot[t] = token_slot(a, table, at);
        if (slot[t] < 0) bad = true;
      }
    }
  };
  // their rows; the new token's are in the call, and go into the cache (by the kv head's first heads)
  auto fetch = [&](uint32_t base) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const bool fresh = p.k && base + 16 * t + c == (uint32_t)n - 1;
      const T* ks = fresh ? static_cast<const T*>(p.k) + new_row : kc + slot[t];
      const T* vs = fresh ? static_cast<const T*>(p.v) + new_row : vc + slot[t];
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        k[t][s] = v[t][s] = {};
        if (slot[t] >= 0) {
          k[t][s] = load_part<T>(ks, 32 * s + 8 * g, p.dim, a.vec);
          v[t][s] = load_part<T>(vs, 32 * s + 8 * g, p.dim, a.vec);
        }
      }
      if (fresh && slot[t] >= 0 && unit % blocks == 0 && !spare) {
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int d = 32 * s + 8 * g + e;
            if (d < p.dim) {
              static_cast<T*>(p.k_cache)[slot[t] + (int64_t)kh * p.dim + d] = k[t][s][e];
              static_cast<T*>(p.v_cache)[slot[t] + (int64_t)kh * p.dim + d] = v[t][s][e];
            }
          }
      }
    }
  };
  constexpr int STRIDE = W * STEP_TOKENS;
  const uint32_t first = t0 + (W == 1 ? 0 : wave * STEP_TOKENS);
  find(first);
  fetch(first);
  V8 q[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    q[s] = {};
    if (c < heads)
      q[s] = load_part<T>(static_cast<const T*>(p.q) + (b * p.heads + h0 + c) * p.dim, 32 * s + 8 * g, p.dim, false);
  }
  if (p.table) {
    const int at = W == 1 ? lane : threadIdx.x, nt = W == 1 ? 64 : STEP_NT;
    for (int i = at; i < STEP_HEADS * p.buckets; i += nt) {
      const int h = i % STEP_HEADS;
      tab[i] = h < heads ? log2_bias(p.table[(int64_t)(i / STEP_HEADS) * p.heads + h0 + h]) : 0.0f;
    }
    for (int i = threadIdx.x; i <= p.radius; i += STEP_NT) map[i] = (unsigned char)min((int)p.map[i], p.buckets - 1);
  }
  __syncthreads();

  const float scale = p.scale * LOG2E;
  float m = -INFINITY, l = 0.0f;
  v4f_t o[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) o[d] = v4f_t{};
  const float far = p.table ? tab[STEP_HEADS * map[0] + c] : 0.0f;
  for (uint32_t base = first; base < t1; base += STRIDE) {
    // V into the wave's own tile, as in Tile::at; K's products
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int s = 0; s < KS; ++s)
        *reinterpret_cast<V8*>(vt + Tile<T, DP>::at(16 * t + c, 32 * s + 8 * g)) = v[t][s];
    v4f_t s[2] = {};
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < KS; ++i) s[t] = mma16(k[t][i], q[i], s[t]);
    find(base + STRIDE);
    if (base + STRIDE < t1) fetch(base + STRIDE);

    float top = -INFINITY;
    const bool near = p.table && (int)(base + STEP_TOKENS) - n > -p.radius;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const uint32_t at = base + 16 * t + 4 * g + r;
        float bias = far;
        if (near) bias = tab[STEP_HEADS * map[max(min((int)at - (n - 1), 0), -p.radius) + p.radius] + c];
        s[t][r] = at < t1 ? __builtin_fmaf(s[t][r], scale, bias) : -INFINITY;
        top = fmaxf(top, s[t][r]);
      }
    const float next = fmaxf(m, join32<MaxOp>(join16<MaxOp>(top)));
    const float ref = next == -INFINITY ? 0.0f : next;
    const float keep = __builtin_amdgcn_exp2f(m - ref);
    m = next;
    V8 w;
    float sum = 0.0f;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float x = __builtin_amdgcn_exp2f(s[t][r] - ref);
        sum += x;
        w[4 * t + r] = (T)(x * (1.0f / WEIGHT_UNIT<T>));
      }
    l = l * keep + sum;
    if (__any(keep != 1.0f)) {
#pragma unroll
      for (int d = 0; d < DB; ++d) o[d] *= keep;
    }
    // tokens 4 g + 0..3 and 16 on, one column a lane
    const T* const col = vt + (g + 4 * (c >> 2)) * S + 4 * (c & 3);
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      const s16x4 x = read_columns4(col + 16 * d), y = read_columns4(col + 16 * S + 16 * d);
      o[d] = mma16(__builtin_bit_cast(V8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7)), w, o[d]);
    }
  }
  l = join32<AddOp>(join16<AddOp>(l));

  if constexpr (W == 1) {
    bad = __any(bad);
    if (spare || c >= heads) return;
    const float inv = bad ? NAN : l == 0.0f ? 0.0f : WEIGHT_UNIT<T> / l;
    T* const out = static_cast<T*>(p.out) + (b * p.heads + h0 + c) * p.dim;
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      vec_t<T, 4> x;
#pragma unroll
      for (int r = 0; r < 4; ++r) x[r] = (T)(o[d][r] * inv);
      if (a.vec) {
        if (16 * d + 4 * g < p.dim) *reinterpret_cast<vec_t<T, 4>*>(out + 16 * d + 4 * g) = x;
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (16 * d + 4 * g + r < p.dim) out[16 * d + 4 * g + r] = x[r];
      }
    }
  } else {
    // the waves' sums, in the V tiles' place
    const bool any_bad = __syncthreads_or(bad);
    float* const acc_lds = reinterpret_cast<float*>(smem);                      // [wave][head][DP + 1]
    float2* const stat_lds = reinterpret_cast<float2*>(smem + a.stat_at);       // [wave][head]
    constexpr int R = DP + 1;
    if (c < heads) {
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc_lds[(wave * heads + c) * R + 16 * d + 4 * g + r] = o[d][r] * WEIGHT_UNIT<T>;
      if (g == 0) stat_lds[wave * heads + c] = make_float2(m, l);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < heads * DP; i += STEP_NT) {
      const int h = i / DP, d = i % DP;
      float top = -INFINITY, sum = 0.0f, x = 0.0f;
      for (int w = 0; w < W; ++w) top = fmaxf(top, stat_lds[w * heads + h].x);
      for (int w = 0; w < W; ++w) {
        const float2 st = stat_lds[w * heads + h];
        const float f = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(st.x - top);
        sum += f * st.y;
        x += f * acc_lds[(w * heads + h) * R + d];
      }
      if (any_bad) x = sum = NAN;
      if (d >= p.dim) continue;
      if (a.splits == 1) {
        static_cast<T*>(p.out)[(b * p.heads + h0 + h) * p.dim + d] = (T)(sum == 0.0f ? 0.0f : x / sum);
      } else {
        const int64_t r = row0 + (int64_t)h * a.splits;
        a.part[r * p.dim + d] = x;
        if (d == 0) a.stat[r] = make_float2(any_bad ? NAN : top, sum);
      }
    }
  }
}

// One (sample, head) a workgroup: the parts' weights by the first wave, then each lane a column of a share of the
// parts, the shares joined in order.
template <class T>
__global__ __launch_bounds__(STEP_NT) void step_join_kernel(const StepArgs a) {
  extern __shared__ __align__(16) unsigned char smem[];
  float* const weight = reinterpret_cast<float*>(smem);  // [splits]
  float* const sums = weight + a.splits;                 // [share][dim]
  __shared__ float inv;
  const int64_t row = blockIdx.x;
  const float2* st = a.stat + row * a.splits;
  if (threadIdx.x < 64) {
    float top = -INFINITY, sum = 0.0f;
    bool bad = false;
    for (int i = threadIdx.x; i < a.splits; i += 64) {
      bad |= st[i].x != st[i].x;
      top = fmaxf(top, st[i].x);
    }
    top = join32<MaxOp>(join16<MaxOp>(stride_join<1, MaxOp>(top)));
    for (int i = threadIdx.x; i < a.splits; i += 64) {
      const float f = st[i].y == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(st[i].x - top);
      weight[i] = f;
      sum += f * st[i].y;
    }
    sum = group_sum<64>(sum);
    bad = __any(bad);
    if (threadIdx.x == 0) inv = bad ? NAN : sum == 0.0f ? 0.0f : 1.0f / sum;
  }
  __syncthreads();
  const int dim = a.p.dim, shares = STEP_NT / dim, share = threadIdx.x / dim, d = threadIdx.x % dim;
  if (share < shares) {
    float x = 0.0f;
#pragma unroll 4
    for (int i = share; i < a.splits; i += shares) {
      const float f = weight[i];
      if (f != 0.0f) x += f * a.part[(row * a.splits + i) * dim + d];  // a part of weight 0 may hold nothing
    }
    sums[share * dim + d] = x;
  }
  __syncthreads();
  if ((int)threadIdx.x < dim) {
    float x = 0.0f;
    for (int i = 0; i < shares; ++i) x += sums[i * dim + d];
    static_cast<T*>(a.p.out)[row * dim + d] = (T)(x * inv);
  }
}

bool step_sizes_ok(const fx_attention_step* p) {
  if (!p || p->batch < 0 || p->heads < 1 || p->kv_heads < 1 || p->heads % p->kv_heads || p->dim < 1 || p->dim > 128 ||
      p->pages < 0 || p->page_size < 1 || p->max_pages < 0)
    return false;
  if (p->dtype != FX_F32 && p->dtype != FX_BF16 && p->dtype != FX_F16) return false;
  if (!scale_ok(p->scale)) return false;
  return p->table ? p->buckets >= 1 && p->buckets <= FX_MAX_ATTENTION_BUCKETS && p->radius >= 0 && p->radius <= FX_MAX_RADIUS
                  : p->buckets == 0 && p->radius == 0;
}

// Whether the heads that share K and V are the columns of a product. (With one head fifteen columns are idle: 167 us for
// 128 at 4096 samples of 8 heads, up to 128 tokens, head dimension 32.)
bool step_mma(const fx_attention_step& p) { return p.dtype != FX_F32 && p.heads > p.kv_heads; }

// Heads that a unit takes at once.
int step_heads(const fx_attention_step& p) {
  const int group = p.heads / p.kv_heads;
  return step_mma(p) ? STEP_HEADS : group >= 3 ? 4 : group;
}

// Units (samples x kv heads x blocks of their heads) from which each gets one wave: four waves a SIMD of the card.
constexpr int64_t STEP_ALONE = 4096;

// Parts of a sample's tokens: enough workgroups for the card, none under 256 tokens of the longest sample
// that the table can hold.
int step_splits(const fx_attention_step& p) {
  const int64_t rows = p.batch * p.kv_heads * cdiv(p.heads / p.kv_heads, step_heads(p));
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
  const int group = p->heads / p->kv_heads, per = step_heads(*p);
  const int64_t rows = p->kv_heads * cdiv(group, per);
  const bool alone = p->batch * rows >= STEP_ALONE;
  if (rows > 65535 || (int64_t)p->max_pages * p->page_size > FX_MAX_STEP_TOKENS ||
      (int64_t)p->kv_heads * p->dim * p->page_size > 0xffffffffll)
    return FX_ERR_UNSUPPORTED;

  StepArgs a{};
  a.p = *p;
  a.splits = splits;
  a.unit = 64;
  a.vec = p->dim % (16 / (int)e) == 0 && aligned(p->k_cache, 16) && aligned(p->v_cache, 16) && aligned(p->k, 16) &&
          aligned(p->v, 16) && aligned(p->out, 16);
  // token / page_size for tokens below 2^31: ceil(2^(31 + bits) / page_size) has 32 bits, bits = ceil(log2 page_size)
  int bits = 0;
  while ((1ll << bits) < p->page_size) ++bits;
  a.shift = bits - 1;
  a.magic = (uint32_t)(((1ull << (31 + bits)) + p->page_size - 1) / p->page_size);
  a.row_size = (uint32_t)p->kv_heads * p->dim;
  a.page_elements = (uint32_t)((int64_t)a.row_size * p->page_size);
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
        const size_t tab = 4 * (size_t)G * p->buckets, map = p->radius + 1;
        if (alone)
          hipLaunchKernelGGL((step_kernel<T, DP, G, 1>), dim3(1, (unsigned)cdiv(rows, STEP_WAVES), (unsigned)nb),
                             dim3(STEP_NT), STEP_WAVES * tab + map, s, c);
        else
          hipLaunchKernelGGL((step_kernel<T, DP, G, STEP_WAVES>), dim3(splits, (unsigned)rows, (unsigned)nb),
                             dim3(STEP_NT), STEP_WAVES * G * (4 * DP + 8) + tab + map, s, c);
      };
      auto by_heads = [&](auto dp) {
        if constexpr (sizeof(T) == 2) {  // heads that share K and V are above
          go(dp, ic<1>{});
        } else {
          if (per == 1)
            go(dp, ic<1>{});
          else if (per == 2)
            go(dp, ic<2>{});
          else
            go(dp, ic<4>{});
        }
      };
      if constexpr (sizeof(T) == 2) {
        if (step_mma(*p)) {
          auto mma = [&](auto dp) {
            constexpr int DP = decltype(dp)::value;
            const int tiles = STEP_WAVES * STEP_TOKENS * Tile<T, DP>::STRIDE * (int)sizeof(T);
            c.stat_at = STEP_WAVES * STEP_HEADS * (DP + 1) * 4;
            const int sums = alone ? 0 : c.stat_at + STEP_WAVES * STEP_HEADS * 8;
            c.sums_bytes = (int)cdiv(tiles > sums ? tiles : sums, 16) * 16;
            const size_t lds = c.sums_bytes + 4 * (size_t)(alone ? STEP_WAVES : 1) * STEP_HEADS * p->buckets + p->radius + 1;
            if (alone)
              hipLaunchKernelGGL((step_mma_kernel<T, DP, 1>), dim3(1, (unsigned)cdiv(rows, STEP_WAVES), (unsigned)nb),
                                 dim3(STEP_NT), lds, s, c);
            else
              hipLaunchKernelGGL((step_mma_kernel<T, DP, STEP_WAVES>), dim3(splits, (unsigned)rows, (unsigned)nb),
                                 dim3(STEP_NT), lds, s, c);
          };
          if (p->dim <= 32)
            mma(ic<32>{});
          else if (p->dim <= 64)
            mma(ic<64>{});
          else
            mma(ic<128>{});
          if (launched() != FX_OK) return FX_ERR_LAUNCH;
          if (splits > 1)
            hipLaunchKernelGGL((step_join_kernel<T>), dim3((unsigned)(nb * p->heads)), dim3(STEP_NT),
                               sizeof(float) * (splits + STEP_NT), s, c);
          continue;
        }
      }
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
        hipLaunchKernelGGL((step_join_kernel<T>), dim3((unsigned)(nb * p->heads)), dim3(STEP_NT),
                           sizeof(float) * (splits + STEP_NT), s, c);
    }
    return launched();
  });
}

}  // extern "C"
