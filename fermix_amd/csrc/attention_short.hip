// Attention's gradient in one launch, for sequences of up to 128 queries and keys of the 16-bit types.
//
// A workgroup has one head of a sample, a wave 32 of its queries, one to a lane as in the forward, with the
// scores' and dP's transposed products of all keys in registers. So delta = sum P dP is exact where it is
// needed: `out` is not read, dS add up to zero, the bucket sums need no correction. dq comes from the
// wave's own dS; dk and dv contract over all queries: P, then dS, go through LDS, rounded, as [query][key],
// beside the waves' query and cotangent rows, and a wave takes 32 of the keys. Five products, each tensor read
// or written once: 316 us at 1024 x 8 heads x 128, head dimension 64, bfloat16 (2.9 TB/s), where the two launches
// for long sequences took 680; bound by the latency of its phases, with two workgroups a CU. Where heads share K
// and V a second launch forms dk and dv from the exact delta.
#include "attention.h"

namespace fx {
namespace net {
namespace {

constexpr int SHORT = 128;  // queries and keys
constexpr int SHORT_WAVES = 4, SHORT_NT = 64 * SHORT_WAVES;

template <class T, int DP>
constexpr size_t short_tile() {
  return (size_t)SHORT * Tile<T, DP>::STRIDE * sizeof(T);
}

template <class T, int DP>
constexpr size_t short_lds(size_t view, int buckets, bool table, bool own) {
  const size_t sums = table ? SHORT_WAVES * 256 * (size_t)buckets : 0, ps = !own ? 0 : short_tile<T, SHORT>();
  return 2 * short_tile<T, DP>() + 544 + view + (sums > ps ? sums : ps);
}

// OWN: heads have K and V of their own; else dk and dv are left to the launch that adds up those that share them.
template <class T, int DP, bool GEN, bool OWN>
__global__ __launch_bounds__(SHORT_NT, DP <= 64 ? 2 : 1) void attention_short_grad_kernel(const AttArgs a) {
  extern __shared__ __align__(16) unsigned char smem[];
  using M = Mma<T>;
  const fx_attention& p = a.p;
  constexpr int DB = DP / 32, ST = Tile<T, DP>::STRIDE;
  T* const t0 = reinterpret_cast<T*>(smem);  // K, then the queries
  T* const t1 = t0 + SHORT * ST;             // V, then the cotangent
  unsigned char* rest = reinterpret_cast<unsigned char*>(t1 + SHORT * ST);
  int* const kpos = reinterpret_cast<int*>(rest);
  unsigned long long* const kok = reinterpret_cast<unsigned long long*>(rest + 512);
  float* const tops = reinterpret_cast<float*>(rest + 528);  // float16: [wave]
  rest += 544;
  const BiasView bv(GEN, rest, p.radius);
  rest += view_lds(GEN, p.radius);
  float* const ds_sums = reinterpret_cast<float*>(rest);  // [wave][bucket][64]
  T* const ps = reinterpret_cast<T*>(rest);               // then [query][key]

  const Place at(a, p.heads, true);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
  const int qi = 32 * wave + (lane & 31);
  const int qlen = p.q_lengths ? max(0, min(p.q_lengths[at.b], p.nq)) : p.nq;
  const int klen = p.lengths ? max(0, min(p.lengths[at.b], p.nk)) : p.nk;
  const bool in = qi < qlen;
  const int qpos = p.q_pos ? (qi < p.nq ? p.q_pos[at.b * p.nq + qi] : 0) : counted_pos(p, qi);
  const int64_t row = (at.b * p.nq + qi) * p.heads + at.h;

  // K and V, 64 rows at a time, and the wave's own rows
  RowFrags<T, DP> q, g;
  {
    const int kh = OWN ? at.h : at.h / (p.heads / p.kv_heads);
    const T* kbase = static_cast<const T*>(p.k) + at.b * p.kb + kh * p.kh;
    const T* vbase = static_cast<const T*>(p.v) + at.b * p.vb + kh * p.vh;
    TileLoad<T, DP, SHORT_NT> kl[2], vl[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int k0 = i * ATT_TILE;
      auto live = [&](int r) { return !GEN || !p.mask || p.mask[at.b * p.nk + k0 + r]; };
      kl[i].fetch(kbase + (int64_t)k0 * p.kn, p.kn, klen - k0, p.dim, a.whole, live);
      vl[i].fetch(vbase + (int64_t)k0 * p.vn, p.vn, klen - k0, p.dim, a.whole, live);
    }
    q.load(static_cast<const T*>(p.q) + at.b * p.qb + (int64_t)qi * p.qn + at.h * p.qh, in, p.dim, a.whole, half);
    g.load(static_cast<const T*>(p.grad_out) + row * p.dim, in, p.dim, a.whole, half);
    load_bias<GEN, SHORT_NT>(p, at.h, bv, a.inv_scale);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      kl[i].put(t0 + i * ATT_TILE * ST);
      vl[i].put(t1 + i * ATT_TILE * ST);
    }
    if (GEN && wave < 2)
      put_keys(key_of(p, at.b, wave * ATT_TILE, klen, lane), KeyView{kpos + wave * ATT_TILE, kok + wave}, lane);
  }
  Sums sums{ds_sums + wave * p.buckets * 64 + lane, nullptr, 0.0f, {}, {}};
  if (p.grad_table)
    for (int t = 0; t < p.buckets; ++t) sums.ds[64 * t] = 0.0f;
  const float2 ml = in ? reinterpret_cast<const float2*>(p.stats)[(at.b * p.heads + at.h) * p.nq + qi]
                       : make_float2(0.0f, INFINITY);
  const float base = ml.x * a.c + ml.y;
  const bool exact = __any(fabsf(ml.x * a.c) > BASE_MAX);
  __syncthreads();
  if (!GEN) {
    lay_bias<GEN, SHORT_NT>(bv);
    __syncthreads();
  }

  // P and dP of all keys, delta
  const int64_t last = !in ? 0 : p.causal ? min((int64_t)klen, (int64_t)p.offset + qi + 1) : (int64_t)klen;
  v16f s[4], dp[4];
  float delta = 0.0f;
  int far[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) far[i] = GEN ? 0 : far_side(i * ATT_TILE - counted_pos(p, 32 * wave), ATT_TILE, 32, p.radius);
#pragma unroll
  for (int kb = 0; kb < 4; ++kb) {
    s[kb] = dp[kb] = v16f{};
    if (32 * kb >= klen) continue;
    const int k0 = kb / 2 * ATT_TILE;
    const KeyView kv{kpos + k0, kok + kb / 2};
    s[kb] = bias_block<GEN>(p, bv, kv, kb & 1, k0, qpos, half, far[kb / 2]);
    s[kb] = row_product<T, DP>(t0, 32 * kb, q, s[kb], lane, p.dim);
    dp[kb] = row_product<T, DP>(t1, 32 * kb, g, dp[kb], lane, p.dim);
    if (exact) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[kb][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][i] - ml.x, a.c, -ml.y));
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[kb][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][i], a.c, -base));
    }
    const int left = (int)last - 32 * kb - 4 * half;
    if (!__all(left >= 28)) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[kb][i] = acc_row(i) < left ? s[kb][i] : 0.0f;
    }
    if (GEN && p.mask) {
      const unsigned ok = (unsigned)(kok[kb / 2] >> (32 * (kb & 1))) >> (4 * half);
#pragma unroll
      for (int i = 0; i < 16; ++i) s[kb][i] = (ok >> acc_row(i)) & 1 ? s[kb][i] : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) delta += s[kb][i] * dp[kb][i];
  }
  delta = half_sum(delta);

  // float16: dS scaled so that the head's largest is just below 2^15. (A scale for each query would serve dq alone: dk's
  // products are over the queries.)
  float fit = 1.0f;
  if constexpr (IS_F16<T>) {
    float top = 0.0f;
#pragma unroll
    for (int kb = 0; kb < 4; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(s[kb][i] * (dp[kb][i] - delta)));
    top = stride_join<1, MaxOp>(top);
    if (lane == 0) tops[wave] = top;
    __syncthreads();
    fit = power_to(fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])), 15);
  }

  // dS, its bucket sums, dq; P and dS rounded for the second half
  v16f dq[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) dq[d] = v16f{};
  typename M::frag pr[4][2], sr[4][2];
#pragma unroll
  for (int kb = 0; kb < 4; ++kb) {
#pragma unroll
    for (int i = 0; i < 2; ++i) pr[kb][i] = M::from_acc(in_units<T>(s[kb]), i);
#pragma unroll
    for (int i = 0; i < 16; ++i) dp[kb][i] = s[kb][i] * (dp[kb][i] - delta);
    const v16f ds = IS_F16<T> ? dp[kb] * fit : dp[kb];
#pragma unroll
    for (int i = 0; i < 2; ++i) sr[kb][i] = M::from_acc(ds, i);
    if (32 * kb >= klen) continue;
    const int k0 = kb / 2 * ATT_TILE;
    if (p.grad_table)
      bucket_add<GEN>(bv, KeyView{kpos + k0, nullptr}, sums, dp[kb], s[kb], kb & 1, k0, qpos, half, far[kb / 2], false);
    column_product<T, DP>(t0, 32 * kb, ds, dq, lane, p.dim);
  }
  const float unit = p.scale / fit;  // of dq and dk
  store_rows<T, DP>(static_cast<T*>(p.grad_q) + row * p.dim, qi < p.nq, dq, unit, p.dim, a.whole, half);
  if (!GEN && p.grad_table) add_pair(sums.ds, bv.map[0], sums.far_ds[0], bv.map[2 * p.radius + 128], sums.far_ds[1]);
  __syncthreads();
  if (p.grad_table) {
    float* out = a.part + (at.h * p.batch + at.b) * p.buckets;
    // four lanes a bucket, one for each wave's sums
    for (int t = threadIdx.x / SHORT_WAVES; t < p.buckets; t += SHORT_NT / SHORT_WAVES) {
      const float* w = ds_sums + ((threadIdx.x % SHORT_WAVES) * p.buckets + t) * 64;
      float x = 0.0f;
#pragma unroll 8
      for (int l = 0; l < 64; ++l) x += w[(l + threadIdx.x) & 63];  // rotated: no shared bank
      x = group_sum<SHORT_WAVES>(x);
      if (threadIdx.x % SHORT_WAVES == 0) out[t] = x;
    }
  }

  if (!OWN) {
    if (qi < p.nq && half == 0) a.delta[(at.b * p.heads + at.h) * p.nq + qi] = delta;
    return;
  }

  // the wave's rows of q and dO for K and V; P
#pragma unroll
  for (int i = 0; i < RowFrags<T, DP>::STEPS; ++i) {
    const int o = Tile<T, DP>::at(qi, M::KS * i + M::KS / 2 * half);
    *reinterpret_cast<typename M::frag*>(t0 + o) = q.f[i];
    *reinterpret_cast<typename M::frag*>(t1 + o) = g.f[i];
  }
  auto put = [&](const typename M::frag(&x)[4][2]) {
#pragma unroll
    for (int kb = 0; kb < 4; ++kb)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        // registers 8 i ..: keys 16 i + 4 half + 0..3, then those 8 on
        const int c = 32 * kb + 16 * i + 4 * half;
        using P = Tile<T, SHORT>;
        *reinterpret_cast<vec_t<T, 4>*>(ps + P::at(qi, c)) = __builtin_shufflevector(x[kb][i], x[kb][i], 0, 1, 2, 3);
        *reinterpret_cast<vec_t<T, 4>*>(ps + P::at(qi, c + 8)) = __builtin_shufflevector(x[kb][i], x[kb][i], 4, 5, 6, 7);
      }
  };
  // rows: the tile's columns; columns: the wave's keys; contracted over the queries
  auto over_queries = [&](const T* tile, v16f(&acc)[DB]) {
#pragma unroll
    for (int d = 0; d < DB; ++d) acc[d] = v16f{};
#pragma unroll
    for (int s = 0; s < SHORT / M::KS; ++s) {
      if (M::KS * s >= qlen) break;
      const typename M::frag b = M::template columns<SHORT>(ps, M::KS * s, 32 * wave, lane);
#pragma unroll
      for (int d = 0; d < DB; ++d) acc[d] = M::mma(M::template columns<DP>(tile, M::KS * s, 32 * d, lane), b, acc[d]);
    }
  };
  __syncthreads();  // the bucket sums have been read
  put(pr);
  __syncthreads();
  v16f acc[DB];
  const int ki = 32 * wave + (lane & 31);
  const int64_t krow = ((at.b * p.nk + ki) * p.kv_heads + at.h) * p.dim;
  over_queries(t1, acc);
  __syncthreads();
  put(sr);
  store_rows<T, DP>(static_cast<T*>(p.grad_v) + krow, ki < p.nk, acc, WEIGHT_UNIT<T>, p.dim, a.whole, half);
  __syncthreads();
  over_queries(t0, acc);
  store_rows<T, DP>(static_cast<T*>(p.grad_k) + krow, ki < p.nk, acc, unit, p.dim, a.whole, half);
}

}  // namespace

bool attention_grad_short_fits(const fx_attention& p) {
  return p.dtype != FX_F32 && p.nq >= 1 && p.nq <= SHORT && p.nk >= 1 && p.nk <= SHORT;
}

int launch_attention_grad_short(const AttArgs& args, hipStream_t s) {
  const fx_attention& p = args.p;
  auto go = [&](auto t, auto dp, auto gen) {
    using T = decltype(t);
    constexpr int DP = decltype(dp)::value;
    constexpr bool GEN = decltype(gen)::value != 0;
    const bool own = p.heads == p.kv_heads;
    const size_t lds = short_lds<T, DP>(view_lds(GEN, p.radius), p.buckets, p.grad_table != nullptr, own);
    launch_items(args, 1, p.batch * p.heads, SHORT_NT, [&](const AttArgs& a) {
      const dim3 grid((unsigned)a.items), block(SHORT_NT);
      if (own)
        hipLaunchKernelGGL((attention_short_grad_kernel<T, DP, GEN, true>), grid, block, lds, s, a);
      else
        hipLaunchKernelGGL((attention_short_grad_kernel<T, DP, GEN, false>), grid, block, lds, s, a);
    });
  };
  return attention_shape(p, [&](auto t, auto dp, auto gen) {
    if constexpr (sizeof(t) == 2) go(t, dp, gen);
  });
}

}  // namespace net
}  // namespace fx
