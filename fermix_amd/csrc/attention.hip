// Attention forward: one pass over the keys with the running maximum and sum of the softmax.
//
// A workgroup has 128 queries of one head, a wave 32 of them, one to a lane (both halves of the wave hold
// it, each half of the keys). Scores are formed transposed, S^T = K q^T, so that a lane has all of its
// query's scores in registers: maximum, sum and rescaling need one exchange between the halves, and the
// rounded weights are the next product's operand as they are (attention.h). K and V tiles of 64 keys
// go through LDS, the next tile's loads in flight while one is worked on.
//
// Bound by vector instructions beside the products (a score costs some nine, an exponential four of them) for long
// sequences, by memory and the workgroups' latency for short ones. MI355X: causal, 2 x 16 heads x 8192, head dimension
// 128, bfloat16, 817 us (670 TFLOP/s); 1024 x 8 heads x 128, head dimension 64, 138 us (3.9 TB/s); float32, 48 x 6
// heads x 302 ragged, 94 us.
#include "attention.h"

namespace fx {
namespace net {
namespace {

template <class T, int DP>
constexpr size_t forward_lds(bool gen, int radius) {
  return 2 * (size_t)ATT_TILE * Tile<T, DP>::STRIDE * sizeof(T) + (gen ? 272 : 0) + view_lds(gen, radius);
}

// WAVES: of a workgroup. Two waves a SIMD hide each other's waits (head dimension 128: 1411 -> 820 us at
// 2 x 16 x 8192 queries); float32 rows of 128 do not fit their registers then.
template <class T, int DP, bool GEN, int WAVES>
__global__ __launch_bounds__(64 * WAVES, DP * (int)sizeof(T) <= 256 ? 2 : 1) void attention_kernel(const AttArgs a) {
  constexpr int NT = 64 * WAVES;
  extern __shared__ __align__(16) unsigned char smem[];
  const fx_attention& p = a.p;
  constexpr int DB = DP / 32, TS = ATT_TILE * Tile<T, DP>::STRIDE;
  T* const kt = reinterpret_cast<T*>(smem);
  T* const vt = kt + TS;
  unsigned char* rest = reinterpret_cast<unsigned char*>(vt + TS);
  KeyView kv{reinterpret_cast<int*>(rest), reinterpret_cast<unsigned long long*>(rest + 256)};
  if (GEN) rest += 272;
  const BiasView bv(GEN, rest, p.radius);

  const Place at(a, p.heads, true);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
  const int q0 = at.tile * 32 * WAVES, qi = q0 + 32 * wave + (lane & 31);
  const int qlen = p.q_lengths ? max(0, min(p.q_lengths[at.b], p.nq)) : p.nq;
  const int klen = p.lengths ? max(0, min(p.lengths[at.b], p.nk)) : p.nk;
  const bool in = qi < qlen;
  const int qpos = p.q_pos ? (qi < p.nq ? p.q_pos[at.b * p.nq + qi] : 0) : counted_pos(p, qi);
  // keys that any query of the workgroup can see
  int keys = q0 < qlen ? klen : 0;
  if (p.causal) keys = (int)min((int64_t)keys, (int64_t)p.offset + min(q0 + 32 * WAVES, qlen));
  const int kh = at.h / (p.heads / p.kv_heads);
  const T* kbase = static_cast<const T*>(p.k) + at.b * p.kb + kh * p.kh;
  const T* vbase = static_cast<const T*>(p.v) + at.b * p.vb + kh * p.vh;

  RowFrags<T, DP> q;
  q.load(static_cast<const T*>(p.q) + at.b * p.qb + (int64_t)qi * p.qn + at.h * p.qh, in, p.dim, a.whole, half);
  v16f o[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) o[d] = v16f{};
  float m = -INFINITY, m_base = -INFINITY, l = 0.0f;  // maximum of the raw scores, that times c, sum

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
  // last key that some query of the wave can see
  const int64_t wave_last = p.causal ? (int64_t)p.offset + q0 + 32 * wave + 31 : (int64_t)p.nk;
  for (int k0 = 0; k0 < keys; k0 += ATT_TILE) {
    __syncthreads();
    kl.put(kt);
    vl.put(vt);
    if (GEN && wave == 0) put_keys(key, kv, lane);
    __syncthreads();
    if (k0 + ATT_TILE < keys) fetch(k0 + ATT_TILE);
    if (k0 > wave_last) continue;

    const int far = GEN ? 0 : far_side(k0 - counted_pos(p, q0 + 32 * wave), ATT_TILE, 32, p.radius);
    v16f s[2];
    float top = -INFINITY;
    // keys of this tile left to the lane, counted from its half's first row
    const int64_t last = !in ? 0 : p.causal ? min((int64_t)klen, (int64_t)p.offset + qi + 1) : (int64_t)klen;
    const int left = (int)max((int64_t)0, min((int64_t)ATT_TILE, last - k0)) - 4 * half;
    const bool edge = k0 + ATT_TILE > klen || q0 + 32 * wave + 32 > qlen ||
                      (p.causal && k0 + ATT_TILE - 1 > wave_last - 31);
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      s[kb] = bias_block<GEN>(p, bv, kv, kb, k0, qpos, half, far);
      s[kb] = row_product<T, DP>(kt, 32 * kb, q, s[kb], lane, p.dim);
      if (edge) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[kb][i] = 32 * kb + acc_row(i) < left ? s[kb][i] : -INFINITY;
      }
      if (GEN && p.mask) {
        const unsigned ok = (unsigned)(*kv.ok >> (32 * kb)) >> (4 * half);
#pragma unroll
        for (int i = 0; i < 16; ++i) s[kb][i] = (ok >> acc_row(i)) & 1 ? s[kb][i] : -INFINITY;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, s[kb][i]);
    }
    const float next = fmaxf(m, half_max(top));
    const float ref = next == -INFINITY ? 0.0f : next, base = ref * a.c;
    const bool exact = sizeof(T) == 4 || __any(fabsf(base) > BASE_MAX);
    const float keep = __builtin_amdgcn_exp2f(exact ? (m - ref) * a.c : m_base - base);
    m = next;
    m_base = next == -INFINITY ? -INFINITY : base;
    float sum = 0.0f;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      exp_block(s[kb], a.c, ref, base, exact);
#pragma unroll
      for (int i = 0; i < 16; ++i) sum += s[kb][i];
    }
    l = l * keep + sum;
    if (__any(keep != 1.0f)) {
#pragma unroll
      for (int d = 0; d < DB; ++d) o[d] *= keep;
    }
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) column_product<T, DP>(vt, 32 * kb, in_units<T>(s[kb]), o, lane, p.dim);
  }

  const bool out_in = qi < p.nq;
  l = half_sum(l);
  const float inv = l > 0.0f ? WEIGHT_UNIT<T> / l : (l != l ? l : 0.0f);
  const int64_t row = (at.b * p.nq + qi) * p.heads + at.h;
  store_rows<T, DP>(static_cast<T*>(p.out) + row * p.dim, out_in, o, inv, p.dim, a.whole, half);
  if constexpr (sizeof(T) == 2)
    if (p.out_low)
      store_low<T, DP>(static_cast<_Float16*>(p.out_low) + row * p.dim, out_in, o, inv, p.dim, a.whole, half);
  if (p.stats && out_in && half == 0)
    reinterpret_cast<float2*>(p.stats)[(at.b * p.heads + at.h) * p.nq + qi] =
        l == 0.0f ? make_float2(0.0f, INFINITY) : make_float2(m, __builtin_amdgcn_logf(l));
}

int forward_waves(const fx_attention& p) { return p.dim > 64 && p.dtype != FX_F32 && p.nq > 128 ? 8 : 4; }

}  // namespace

bool attention_sizes_ok(const fx_attention* p) {
  if (!p || p->batch < 0 || p->nq < 0 || p->nq > FX_MAX_POSITIONS || p->nk < 0 || p->nk > FX_MAX_POSITIONS ||
      p->heads < 1 || p->kv_heads < 1 || p->heads % p->kv_heads || p->dim < 1 || p->dim > 128)
    return false;
  if (p->dtype != FX_F32 && p->dtype != FX_BF16 && p->dtype != FX_F16) return false;
  if (!scale_ok(p->scale)) return false;
  if (p->offset < 0 || p->offset > 0x7fffffff - (p->nq > p->nk ? p->nq : p->nk)) return false;
  if (p->table ? p->buckets < 1 || p->buckets > FX_MAX_ATTENTION_BUCKETS || p->radius < 0 || p->radius > FX_MAX_RADIUS
               : p->buckets != 0 || p->radius != 0)
    return false;
  return !p->q_pos == !p->k_pos;
}

bool attention_pointers_ok(const fx_attention& p) {
  const size_t e = dtype_size(p.dtype);
  for (const void* q : {p.q, p.k, p.v, (const void*)p.out, p.grad_out, (const void*)p.grad_q, (const void*)p.grad_k,
                        (const void*)p.grad_v, (const void*)p.out_low})
    if (!aligned(q, e)) return false;
  for (const void* q : {(const void*)p.table, (const void*)p.q_pos, (const void*)p.k_pos, (const void*)p.lengths,
                        (const void*)p.q_lengths, (const void*)p.grad_table})
    if (!aligned(q, 4)) return false;
  if (!aligned(p.stats, 8)) return false;
  return p.q && (p.nk == 0 || (p.k && p.v)) && p.out && (!p.table || p.map);
}

AttArgs attention_args(const fx_attention& p) {
  AttArgs a{};
  a.p = p;
  const int64_t e = (int64_t)dtype_size(p.dtype), v = 16 / e;
  const int64_t strides = p.dim | p.qb | p.qn | p.qh | p.kb | p.kn | p.kh | p.vb | p.vn | p.vh;
  const uintptr_t in = (uintptr_t)p.q | (uintptr_t)p.k | (uintptr_t)p.v | (uintptr_t)p.grad_out | (uintptr_t)p.out |
                       (uintptr_t)p.out_low | (uintptr_t)p.grad_q | (uintptr_t)p.grad_k | (uintptr_t)p.grad_v;
  a.whole = strides % v == 0 && !(in & 15);
  a.c = p.scale * LOG2E;
  a.inv_scale = 1.0f / p.scale;
  return a;
}

}  // namespace net
}  // namespace fx

using namespace fx;
using namespace fx::net;

extern "C" int32_t fx_attention_keeps_low(const fx_attention* p) {
  return attention_sizes_ok(p) && p->dtype != FX_F32 && !attention_grad_short_fits(*p);
}

extern "C" int fx_attention_forward(const fx_attention* p, fx_stream_t stream) {
  if (!attention_sizes_ok(p)) return FX_ERR_INVALID_ARGUMENT;
  if (p->batch == 0 || p->nq == 0) return FX_OK;
  if (!attention_pointers_ok(*p)) return FX_ERR_INVALID_ARGUMENT;
  const AttArgs args = attention_args(*p);
  const int waves = forward_waves(*p), tiles = (int)cdiv(p->nq, 32 * waves);
  return attention_shape(*p, [&](auto t, auto dp, auto gen) {
    using T = decltype(t);
    constexpr int DP = decltype(dp)::value;
    constexpr bool GEN = decltype(gen)::value != 0;
    const size_t lds = forward_lds<T, DP>(GEN, p->radius);
    auto go = [&](auto w) {
      constexpr int WAVES = decltype(w)::value;
      launch_items(args, tiles, p->batch * p->heads * tiles, 64 * WAVES, [&](const AttArgs& a) {
        hipLaunchKernelGGL((attention_kernel<T, DP, GEN, WAVES>), dim3((unsigned)a.items), dim3(64 * WAVES), lds,
                           (hipStream_t)stream, a);
      });
    };
    if constexpr (DP == 128 && sizeof(T) == 2)
      if (waves == 8) return go(ic<8>{});
    go(ic<4>{});
  });
}
