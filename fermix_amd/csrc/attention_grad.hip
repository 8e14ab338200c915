// Attention's gradient from the forward's statistics and out, in two launches that form the scores again:
//   P = exp2(c (S' - m) - log2 l),  delta = sum_d out dO,  dP = dO v^T,  dS = P (dP - delta),
//   dq = scale dS k  and the bias' bucket sums of dS     (a workgroup: 128 queries, over the keys),
//   dv = P^T dO,  dk = scale dS^T q                      (a workgroup: 128 keys, over the queries of
//                                                         all heads that share them).
// MI355X: causal, 2 x 16 heads x 8192, head dimension 128, bfloat16, 1157 + 1880 us (450 TFLOP/s of the five products
// that a gradient needs); bound by the waits of two waves a SIMD at the tiles' barriers (products 29 % of the second
// launch's time, LDS and vector instructions some 30 % each). float32, 48 x 6 heads x 302 ragged, 136 + 160 us.
//
// Seven products where one launch would need five, but no sum crosses workgroups: nothing is added
// by atomics in memory, every order is fixed. The first launch also leaves delta for the second.
//
// Bucket sums: each lane adds its dS to sums of its own in LDS, [bucket][lane] (no two lanes share a
// bank or an address, a wave's LDS operations complete in order); tiles past the radius add up in
// registers; the workgroups' sums are joined by a last launch. delta as out gives it is off by what P and out lost to
// rounding (16-bit types: some 1e-3, out_low takes most of it), which a bucket's sum would keep. A query's dS
// then add up to that error instead of to 0, so the launch also sums P by query and bucket, and takes
// (sum of the query's dS) x (sum of its P in the bucket) off at the end. As the correction is small, P is summed
// in fixed point (units of 2^-30), whose order does not matter, the two halves of a wave in one place.
#include "attention.h"

namespace fx {
namespace net {
namespace {

template <class T, int DP>
constexpr size_t tiles_lds() {
  return 2 * (size_t)ATT_TILE * Tile<T, DP>::STRIDE * sizeof(T);
}
// WAVES: of a workgroup.
template <class T, int DP, bool GEN, int WAVES>
__global__ __launch_bounds__(64 * WAVES, DP * (int)sizeof(T) <= 256 && !(DP == 128 && WAVES == 4) ? 2 : 1) void attention_dq_kernel(
    const AttArgs a) {
  constexpr int NT = 64 * WAVES;
  extern __shared__ __align__(16) unsigned char smem[];
  using M = Mma<T>;
  const fx_attention& p = a.p;
  constexpr int DB = DP / 32, TS = ATT_TILE * Tile<T, DP>::STRIDE;
  T* const kt = reinterpret_cast<T*>(smem);
  T* const vt = kt + TS;
  unsigned char* rest = reinterpret_cast<unsigned char*>(vt + TS);
  KeyView kv{reinterpret_cast<int*>(rest), reinterpret_cast<unsigned long long*>(rest + 256)};
  rest += 272;
  const BiasView bv(GEN, rest, p.radius);
  const bool weights_on = p.grad_table && (sizeof(T) == 2 || a.weights);
  float* const row_sum = reinterpret_cast<float*>(rest + view_lds(GEN, p.radius));  // [wave][32]
  float* const ds_sums = row_sum + 32 * WAVES;                                             // [wave][bucket][64]
  unsigned* const weights = reinterpret_cast<unsigned*>(ds_sums + 64 * WAVES * p.buckets);  // [wave][bucket][32]

  const Place at(a, p.heads, true);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
  const int q0 = at.tile * 32 * WAVES, qi = q0 + 32 * wave + (lane & 31);
  const int qlen = p.q_lengths ? max(0, min(p.q_lengths[at.b], p.nq)) : p.nq;
  const int klen = p.lengths ? max(0, min(p.lengths[at.b], p.nk)) : p.nk;
  const bool in = qi < qlen;
  const int qpos = p.q_pos ? (qi < p.nq ? p.q_pos[at.b * p.nq + qi] : 0) : counted_pos(p, qi);
  int keys = q0 < qlen ? klen : 0;
  if (p.causal) keys = (int)min((int64_t)keys, (int64_t)p.offset + min(q0 + 32 * WAVES, qlen));
  const int kh = at.h / (p.heads / p.kv_heads);
  const T* kbase = static_cast<const T*>(p.k) + at.b * p.kb + kh * p.kh;
  const T* vbase = static_cast<const T*>(p.v) + at.b * p.vb + kh * p.vh;
  const int64_t row = (at.b * p.nq + qi) * p.heads + at.h, stat = (at.b * p.heads + at.h) * p.nq + qi;

  Sums sums{ds_sums + wave * p.buckets * 64 + lane, weights + wave * p.buckets * 32 + (lane & 31), 0.0f, {}, {}};
  if (p.grad_table)
    for (int t = 0; t < p.buckets; ++t) {
      sums.ds[64 * t] = 0.0f;
      if (weights_on) sums.weight[32 * t] = 0u;
    }
  RowFrags<T, DP> q, g;
  q.load(static_cast<const T*>(p.q) + at.b * p.qb + (int64_t)qi * p.qn + at.h * p.qh, in, p.dim, a.whole, half);
  g.load(static_cast<const T*>(p.grad_out) + row * p.dim, in, p.dim, a.whole, half);
  float delta = 0.0f;
  {
    RowFrags<T, DP> o;
    o.load(static_cast<const T*>(p.out) + row * p.dim, in, p.dim, a.whole, half);
#pragma unroll
    for (int s = 0; s < RowFrags<T, DP>::STEPS; ++s)
#pragma unroll
      for (int e = 0; e < M::KS / 2; ++e) delta += (float)o.f[s][e] * (float)g.f[s][e];
    if constexpr (sizeof(T) == 2) {
      if (p.out_low) {
        RowFrags<_Float16, DP> low;
        low.load(static_cast<const _Float16*>(p.out_low) + row * p.dim, in, p.dim, a.whole, half);
        float d = 0.0f;
#pragma unroll
        for (int s = 0; s < RowFrags<T, DP>::STEPS; ++s)
#pragma unroll
          for (int e = 0; e < M::KS / 2; ++e) d += (float)low.f[s][e] * (float)g.f[s][e];
        delta += d * (1.0f / LOW_SCALE<T>);
      }
    }
    delta = half_sum(delta);
  }
  const float2 ml = in ? reinterpret_cast<const float2*>(p.stats)[stat] : make_float2(0.0f, INFINITY);
  const float base = ml.x * a.c + ml.y;
  const bool exact = sizeof(T) == 4 || __any(fabsf(ml.x * a.c) > BASE_MAX);

  v16f dq[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) dq[d] = v16f{};
  float fit = IS_F16<T> ? SCALE_START : 1.0f;
  TileLoad<T, DP, NT> kl, vl;
  KeyOf key{};  // of wave 0's lanes (GEN)
  auto fetch = [&](int k0) {
    if (GEN && wave == 0) key = key_of(p, at.b, k0, klen, lane);
    auto live = [&](int r) { return !GEN || !p.mask || p.mask[at.b * p.nk + k0 + r]; };
    kl.fetch(kbase + (int64_t)k0 * p.kn, p.kn, keys - k0, p.dim, a.whole, live);
    vl.fetch(vbase + (int64_t)k0 * p.vn, p.vn, keys - k0, p.dim, a.whole, live);
  };
  if (keys > 0) fetch(0);
  load_bias<GEN, NT>(p, at.h, bv, a.inv_scale);
  __syncthreads();
  lay_bias<GEN, NT>(bv);
  const int64_t wave_last = p.causal ? (int64_t)p.offset + q0 + 32 * wave + 31 : (int64_t)p.nk;
  for (int k0 = 0; k0 < keys; k0 += ATT_TILE) {
    __syncthreads();
    kl.put(kt);
    vl.put(vt);
    if (GEN && wave == 0) put_keys(key, kv, lane);
    __syncthreads();
    if (k0 + ATT_TILE < keys) fetch(k0 + ATT_TILE);
    if (k0 > wave_last) continue;
    const int64_t last = !in ? 0 : p.causal ? min((int64_t)klen, (int64_t)p.offset + qi + 1) : (int64_t)klen;
    const int left = (int)max((int64_t)0, min((int64_t)ATT_TILE, last - k0)) - 4 * half;
    const bool edge = k0 + ATT_TILE > klen || q0 + 32 * wave + 32 > qlen ||
                      (p.causal && k0 + ATT_TILE - 1 > wave_last - 31);
    const int far = GEN ? 0 : far_side(k0 - counted_pos(p, q0 + 32 * wave), ATT_TILE, 32, p.radius);
#pragma unroll 1  // both blocks at once spill at DP = 128: 1269 us at 2 x 16 x 8192 queries, one by one 1120
    for (int kb = 0; kb < 2; ++kb) {
      v16f s = bias_block<GEN>(p, bv, kv, kb, k0, qpos, half, far);
      s = row_product<T, DP>(kt, 32 * kb, q, s, lane, p.dim);
      v16f dp = row_product<T, DP>(vt, 32 * kb, g, v16f{}, lane, p.dim);
      if (exact) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i] - ml.x, a.c, -ml.y));
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], a.c, -base));
      }
      if (edge) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = 32 * kb + acc_row(i) < left ? s[i] : 0.0f;
      }
      if (GEN && p.mask) {
        const unsigned ok = (unsigned)(*kv.ok >> (32 * kb)) >> (4 * half);
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = (ok >> acc_row(i)) & 1 ? s[i] : 0.0f;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) dp[i] = s[i] * (dp[i] - delta);
      if (sizeof(T) == 2 || weights_on) {
#pragma unroll
        for (int i = 0; i < 16; ++i) sums.all += dp[i];
      }
      if (p.grad_table) bucket_add<GEN>(bv, kv, sums, dp, s, kb, k0, qpos, half, far, weights_on);
      if constexpr (IS_F16<T>) {
        fit_scale(fit, dp, dq);
        dp *= fit;
      }
      column_product<T, DP>(kt, 32 * kb, dp, dq, lane, p.dim);
    }
  }
  store_rows<T, DP>(static_cast<T*>(p.grad_q) + row * p.dim, qi < p.nq, dq, p.scale / fit, p.dim, a.whole, half);
  // what dS add up to is delta's error: the second launch gets delta without it
  const float all = sizeof(T) == 2 || weights_on ? half_sum(sums.all) : 0.0f;
  if (qi < p.nq && half == 0) a.delta[stat] = delta + all;
  if (p.grad_table) {
    if (!GEN) {
      const int t[2] = {bv.map[0], bv.map[2 * p.radius + 128]};
      add_pair(sums.ds, t[0], sums.far_ds[0], t[1], sums.far_ds[1]);
      for (int i = 0; weights_on && i < 2; ++i) atomicAdd(sums.weight + 32 * t[i], fixed_weight(sums.far_weight[i]));
    }
    if (half == 0) row_sum[32 * wave + lane] = all;
    __syncthreads();
    float* out = a.part + ((at.h * p.batch + at.b) * a.tiles + at.tile) * p.buckets;
    for (int t = threadIdx.x; t < p.buckets; t += NT) {
      float x = 0.0f, y = 0.0f;
      for (int w = 0; w < WAVES; ++w) {
#pragma unroll 4
        for (int l = 0; l < 64; ++l) x += ds_sums[(w * p.buckets + t) * 64 + ((l + t) & 63)];  // rotated: no shared bank
        if (weights_on)
#pragma unroll 4
          for (int l = 0; l < 32; ++l) {
            const int r = (l + t) & 31;
            y += row_sum[32 * w + r] * (float)weights[(w * p.buckets + t) * 32 + r];
          }
      }
      out[t] = x - 0x1p-30f * y;
    }
  }
}

// A tile's queries: positions (GEN), maximum (exact), c maximum + log2 sum, or log2 sum (exact), and delta.
struct QueryView {
  int* pos;
  float *max, *log, *delta;
  unsigned* exact;  // some |c maximum| of the tile is over BASE_MAX
};

template <bool GEN>
__device__ __forceinline__ v16f bias_block_t(const BiasView& bv, const QueryView& qv, int qb, int at0, int kpos,
                                             int half, int far) {
  v16f x;
  if (!GEN && far) {
    const float v = bv.lut[far > 0 ? 2 * bv.radius + 128 : 0];
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = v;
  } else if constexpr (GEN) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int4 qp = *reinterpret_cast<const int4*>(qv.pos + 32 * qb + 8 * g + 4 * half);
      const int q[4] = {qp.x, qp.y, qp.z, qp.w};
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        x[4 * g + r] = bv.table[distance_bucket(bv.map, bv.radius, kpos, q[r])];
      }
    }
  } else {
    const int d = max(-bv.radius, min(bv.radius + 64, kpos - at0));
    const float* l = bv.lut + d + bv.radius + 64 - 32 * qb - 4 * half;
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = l[-acc_row(i)];
  }
  return x;
}

// Four waves have 32 keys each. SPLIT: eight do, the first four for dv and the others for dk of the same keys; both
// form the scores (five products for four), but neither has to hold the other's sums, so that two waves fit a
// SIMD where the rows are long. (Not for float32, whose products take longest: 204 us for 175 at 48 x 302.)
template <class T, int DP, bool GEN, bool SPLIT>
__global__ __launch_bounds__(SPLIT ? 512 : 256, sizeof(T) == 2 || DP == 32 ? 2 : 1) void attention_dkv_kernel(
    const AttArgs a) {
  constexpr int NT = SPLIT ? 512 : 256;
  extern __shared__ __align__(16) unsigned char smem[];
  const fx_attention& p = a.p;
  constexpr int DB = DP / 32, TS = ATT_TILE * Tile<T, DP>::STRIDE;
  T* const qt = reinterpret_cast<T*>(smem);
  T* const gt = qt + TS;
  unsigned char* rest = reinterpret_cast<unsigned char*>(gt + TS);
  float* const f = reinterpret_cast<float*>(rest);
  QueryView qv{reinterpret_cast<int*>(rest), f + 64, f + 128, f + 192, reinterpret_cast<unsigned*>(f + 256)};
  rest += 1040;
  const BiasView bv(GEN, rest, p.radius);

  const Place at(a, p.kv_heads, false);  // heads: those of k and v
  const int lane = threadIdx.x & 63, wave = (threadIdx.x >> 6) & 3, half = lane >> 5;
  const bool do_v = !SPLIT || threadIdx.x < 256, do_k = !SPLIT || threadIdx.x >= 256;
  const int k0 = at.tile * 128, kw = k0 + 32 * wave, ki = kw + (lane & 31);
  const int qlen = p.q_lengths ? max(0, min(p.q_lengths[at.b], p.nq)) : p.nq;
  const int klen = p.lengths ? max(0, min(p.lengths[at.b], p.nk)) : p.nk;
  const bool in = ki < klen && !(GEN && p.mask && !p.mask[at.b * p.nk + ki]);
  const int kpos = p.k_pos ? (ki < p.nk ? p.k_pos[at.b * p.nk + ki] : 0) : ki;
  const int group = p.heads / p.kv_heads;
  RowFrags<T, DP> k, v;
  k.load(static_cast<const T*>(p.k) + at.b * p.kb + (int64_t)ki * p.kn + at.h * p.kh, in, p.dim, a.whole, half);
  v.load(static_cast<const T*>(p.v) + at.b * p.vb + (int64_t)ki * p.vn + at.h * p.vh, in && do_k, p.dim, a.whole, half);
  const bool whole = __all(in);  // every lane's key is left
  v16f sum[SPLIT ? 1 : 2][DB];   // dk (SPLIT: or dv), dv
#pragma unroll
  for (int d = 0; d < DB; ++d) {
    sum[0][d] = v16f{};
    if (!SPLIT) sum[SPLIT ? 0 : 1][d] = v16f{};
  }
  float fit = IS_F16<T> ? SCALE_START : 1.0f;
  // queries that some key of the workgroup is seen by
  const int first = p.causal ? max(0, k0 - p.offset) / ATT_TILE * ATT_TILE : 0;
  const int queries = k0 < klen ? qlen : 0;

  for (int j = 0; j < group; ++j) {
    const int h = at.h * group + j;
    const T* qbase = static_cast<const T*>(p.q) + at.b * p.qb + h * p.qh;
    const T* gbase = static_cast<const T*>(p.grad_out) + (at.b * p.nq * p.heads + h) * p.dim;
    const int64_t stat = (at.b * p.heads + h) * p.nq;
    TileLoad<T, DP, NT> ql, gl;
    float2 ml;  // of query threadIdx.x of the tile: statistics, delta, position
    float de;
    int qp = 0;
    auto fetch = [&](int q0) {
      if (threadIdx.x < ATT_TILE) {
        const int i = q0 + threadIdx.x;
        const bool q_in = i < queries;
        ml = q_in ? reinterpret_cast<const float2*>(p.stats)[stat + i] : make_float2(0.0f, INFINITY);
        de = q_in ? a.delta[stat + i] : 0.0f;
        if (GEN) qp = !q_in ? 0 : p.q_pos ? p.q_pos[at.b * p.nq + i] : p.offset + i;
      }
      auto live = [](int) { return true; };
      ql.fetch(qbase + (int64_t)q0 * p.qn, p.qn, queries - q0, p.dim, a.whole, live);
      gl.fetch(gbase + (int64_t)q0 * p.heads * p.dim, (int64_t)p.heads * p.dim, queries - q0, p.dim, a.whole, live);
    };
    if (first < queries) fetch(first);
    __syncthreads();  // the last head's view has been read
    load_bias<GEN, NT>(p, h, bv, a.inv_scale);
    __syncthreads();
    lay_bias<GEN, NT>(bv);
    for (int q0 = first; q0 < queries; q0 += ATT_TILE) {
      __syncthreads();
      ql.put(qt);
      gl.put(gt);
      if (threadIdx.x < ATT_TILE) {
        const bool exact = sizeof(T) == 4 || __any(fabsf(ml.x * a.c) > BASE_MAX);
        qv.max[threadIdx.x] = ml.x;
        qv.log[threadIdx.x] = exact ? ml.y : ml.x * a.c + ml.y;
        if (threadIdx.x == 0) *qv.exact = exact;
        qv.delta[threadIdx.x] = de;
        if (GEN) qv.pos[threadIdx.x] = qp;
      }
      __syncthreads();
      if (q0 + ATT_TILE < queries) fetch(q0 + ATT_TILE);
      if (p.causal && (int64_t)p.offset + q0 + ATT_TILE - 1 < kw) continue;
      // first row of the tile that sees the lane's key, counted from its half's first row
      const int from = (p.causal ? (int)max((int64_t)0, min((int64_t)ATT_TILE, (int64_t)ki - p.offset - q0)) : 0) - 4 * half;
      const bool edge = p.causal && (int64_t)p.offset + q0 < kw + 31;
      const int far = GEN ? 0 : far_side(kw - counted_pos(p, q0), 32, ATT_TILE, p.radius);
      const bool exact = sizeof(T) == 4 || *qv.exact;
#pragma unroll sizeof(T) == 4 && DP == 128 ? 1 : 2  // (both blocks at once do not fit the registers there)
      for (int qb = 0; qb < 2; ++qb) {
        v16f s = bias_block_t<GEN>(bv, qv, qb, p.offset + q0, kpos, half, far);
        s = row_product<T, DP>(qt, 32 * qb, k, s, lane, p.dim);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int at4 = 32 * qb + 8 * g + 4 * half;
          const float4 log = *reinterpret_cast<const float4*>(qv.log + at4);
          const float lo[4] = {log.x, log.y, log.z, log.w};
          if (exact) {
            const float4 max = *reinterpret_cast<const float4*>(qv.max + at4);
            const float ma[4] = {max.x, max.y, max.z, max.w};
#pragma unroll
            for (int r = 0; r < 4; ++r) s[4 * g + r] -= ma[r];
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) s[4 * g + r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[4 * g + r], a.c, -lo[r]));
        }
        if (edge) {
#pragma unroll
          for (int i = 0; i < 16; ++i) s[i] = 32 * qb + acc_row(i) >= from ? s[i] : 0.0f;
        }
        if (!whole) {
#pragma unroll
          for (int i = 0; i < 16; ++i) s[i] = in ? s[i] : 0.0f;
        }
        if (do_v) column_product<T, DP>(gt, 32 * qb, in_units<T>(s), sum[SPLIT ? 0 : 1], lane, p.dim);
        if (!do_k) continue;
        const v16f dp = row_product<T, DP>(gt, 32 * qb, v, v16f{}, lane, p.dim);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float4 delta = *reinterpret_cast<const float4*>(qv.delta + 32 * qb + 8 * g + 4 * half);
          const float de[4] = {delta.x, delta.y, delta.z, delta.w};
#pragma unroll
          for (int r = 0; r < 4; ++r) s[4 * g + r] *= dp[4 * g + r] - de[r];
        }
        if constexpr (IS_F16<T>) {
          fit_scale(fit, s, sum[0]);
          s *= fit;
        }
        column_product<T, DP>(qt, 32 * qb, s, sum[0], lane, p.dim);
      }
    }
  }
  const int64_t row = ((at.b * p.nk + ki) * p.kv_heads + at.h) * p.dim;
  if (do_k)
    store_rows<T, DP>(static_cast<T*>(p.grad_k) + row, ki < p.nk, sum[0], p.scale / fit, p.dim, a.whole, half);
  if (do_v)
    store_rows<T, DP>(static_cast<T*>(p.grad_v) + row, ki < p.nk, sum[SPLIT ? 0 : 1], WEIGHT_UNIT<T>, p.dim, a.whole, half);
}

// Whether P is summed beside dS. For float32, whose delta is off by float32's roundings only, where these add up over many
// keys (3000 keys: the bucket sums' error 1.8e-6 without, 0.9e-6 with; at 302 it is 0.7e-6, and 190 us for 133, as
// the sums leave LDS for one workgroup a CU), and not for rows of 128 with more buckets than LDS holds both for.
bool sums_weights(const fx_attention& p) {
  return p.dtype != FX_F32 || (p.nk > 1024 && (p.dim <= 64 || p.buckets <= 32));
}

// Bytes of a workgroup's bucket sums in the first launch.
size_t sums_lds(const fx_attention& p, int waves) {
  return waves * (128 + (sums_weights(p) ? 384 : 256) * (size_t)p.buckets);
}

// Waves of a workgroup of the first launch: eight where the rows are long (they leave the registers for two waves a
// SIMD only if the tile's loads are shared by eight) and the bucket sums of eight fit, else four.
int dq_waves(const fx_attention& p) {
  return p.dim > 64 && p.dtype != FX_F32 && p.nq > 128 && p.buckets <= 32 && p.radius <= 1024 ? 8 : 4;
}

int64_t delta_floats(const fx_attention& p) { return cdiv(p.batch * p.heads * p.nq, 4) * 4; }

}  // namespace
}  // namespace net
}  // namespace fx

using namespace fx;
using namespace fx::net;

extern "C" {

size_t fx_attention_grad_workspace(const fx_attention* p) {
  if (!attention_sizes_ok(p) || p->batch == 0 || p->nq == 0) return 0;
  const int64_t tiles = cdiv(p->nq, 32 * dq_waves(*p));
  return sizeof(float) * (size_t)(delta_floats(*p) + (p->table ? p->batch * p->heads * tiles * p->buckets : 0));
}

int fx_attention_grad(const fx_attention* p, void* workspace, size_t workspace_bytes, fx_stream_t stream) {
  if (!attention_sizes_ok(p) || (p->grad_table && !p->table)) return FX_ERR_INVALID_ARGUMENT;
  if (p->batch == 0) {
    if (!p->grad_table) return FX_OK;
    return launch_bucket_join(nullptr, 0, p->buckets, p->heads, p->grad_table, (hipStream_t)stream);
  }
  const hipStream_t s = (hipStream_t)stream;
  if (p->nq > 0) {
    if (!attention_pointers_ok(*p) || !p->stats || !p->grad_out || !p->grad_q) return FX_ERR_INVALID_ARGUMENT;
    if (!workspace || !aligned(workspace, 16) || workspace_bytes < fx_attention_grad_workspace(p))
      return FX_ERR_WORKSPACE;
  }
  if (p->nk > 0 && (!p->k || !p->v || !p->grad_k || !p->grad_v)) return FX_ERR_INVALID_ARGUMENT;
  AttArgs args = attention_args(*p);
  args.delta = static_cast<float*>(workspace);
  args.part = args.delta + delta_floats(*p);
  args.weights = sums_weights(*p);
  const bool in_short = attention_grad_short_fits(*p), own = p->heads == p->kv_heads;
  if (in_short) {
    const int st = launch_attention_grad_short(args, s);
    if (st != FX_OK) return st;
  }
  const int waves = dq_waves(*p), qtiles = (int)cdiv(p->nq, 32 * waves), ktiles = (int)cdiv(p->nk, 128);
  const int st = attention_shape(*p, [&](auto t, auto dp, auto gen) {
    using T = decltype(t);
    constexpr int DP = decltype(dp)::value;
    constexpr bool GEN = decltype(gen)::value != 0;
    const size_t tiles = tiles_lds<T, DP>(), view = view_lds(GEN, p->radius);
    const size_t lds_q = tiles + 272 + view + (p->grad_table ? sums_lds(*p, waves) : 0);
    const size_t lds_kv = tiles + 1040 + view;
    constexpr bool LONG_ROWS = DP == 128 && sizeof(T) == 2;
    if (qtiles && !in_short) {
      auto go = [&](auto w) {
        constexpr int WAVES = decltype(w)::value;
        launch_items(args, qtiles, p->batch * p->heads * qtiles, 64 * WAVES, [&](const AttArgs& a) {
          hipLaunchKernelGGL((attention_dq_kernel<T, DP, GEN, WAVES>), dim3((unsigned)a.items), dim3(64 * WAVES), lds_q,
                             s, a);
        });
      };
      if constexpr (LONG_ROWS) {
        if (waves == 8)
          go(ic<8>{});
        else
          go(ic<4>{});
      } else {
        go(ic<4>{});
      }
    }
    if (ktiles && !(in_short && own)) {
      constexpr int NT = LONG_ROWS ? 512 : 256;
      launch_items(args, ktiles, p->batch * p->kv_heads * ktiles, NT, [&](const AttArgs& a) {
        hipLaunchKernelGGL((attention_dkv_kernel<T, DP, GEN, LONG_ROWS>), dim3((unsigned)a.items), dim3(NT), lds_kv, s,
                           a);
      });
    }
  });
  if (st != FX_OK || !p->grad_table) return st;
  return launch_bucket_join(args.part, p->batch * qtiles, p->buckets, p->heads, p->grad_table, s);
}

}  // extern "C"
