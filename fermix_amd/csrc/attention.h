// Attention with a relative position bias: what its forward and gradient kernels share.
//
// Products run on the 32 x 32 MFMA. Lane l = 32 h + c (h the half, c the column) of a wave holds
//   A or B operand: row (column) c, the KS / 2 contraction indices KS s + (KS / 2) h .. of step s:
//     16 bytes of a row, eight 16-bit or four float32 elements (four K = 2 products);
//   accumulator: column c, rows 8 g + 4 h + r (g, r = 0..3) in register 4 g + r.
// A product's accumulator, rounded to the type, is the B operand of the next product that contracts
// over its rows, without a move between lanes: float32's indices agree, and for 16-bit types
// the A operand takes the rows in the accumulator's order (16 s + 4 h + r, then 16 s + 8 + 4 h + r).
// That A operand is a column read of a row-major tile: four float32 reads, or two transposing
// 64-bit LDS reads (16 lanes read 4 rows of 16 columns, each gets one column).
#pragma once
#include "net.h"

namespace fx {
namespace net {

typedef float v16f __attribute__((ext_vector_type(16)));

// Rows of DP elements in LDS, padded by 16 bytes. For the 16-bit types the rows of each sixteen are stored
// transposed as 4 x 4, so that a column operand's four consecutive rows lie four apart: 16 banks apart for every DP,
// where in order they were 4 (6 clk more for each read). A row operand's lanes meet all banks either way.
template <class T, int DP>
struct Tile {
  static constexpr int STRIDE = DP + 16 / (int)sizeof(T);
  static __device__ __forceinline__ int row_at(int row) {
    return sizeof(T) == 2 ? (row & ~15) | ((row & 3) << 2) | ((row >> 2) & 3) : row;
  }
  // Place of an element; the rest of its row follows.
  static __device__ __forceinline__ int at(int row, int col) { return row_at(row) * STRIDE + col; }
};

template <class T>
struct Mma;

template <>
struct Mma<float> {
  static constexpr int KS = 8;
  using frag = v4f;
  static __device__ __forceinline__ v16f mma(frag a, frag b, v16f c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
    return c;
  }
  template <int DP>
  static __device__ __forceinline__ frag columns(const float* tile, int row, int col, int lane) {
    constexpr int S = Tile<float, DP>::STRIDE;
    const float* p = tile + (row + 4 * (lane >> 5)) * S + col + (lane & 31);
    return frag{p[0], p[S], p[2 * S], p[3 * S]};
  }
  static __device__ __forceinline__ frag from_acc(const v16f& x, int s) {
    return frag{x[4 * s], x[4 * s + 1], x[4 * s + 2], x[4 * s + 3]};
  }
};

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

// Columns of four rows of a row-major 16-bit tile for 16 lanes at a time.
__device__ __forceinline__ s16x4 read_columns4(const void* p) {
  typedef __attribute__((address_space(3))) s16x4 lds_t;
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t*)(const s16x4*)p);
}

template <class T>
struct Mma16 {
  static constexpr int KS = 16;
  using frag = vec_t<T, 8>;
  template <int DP>
  static __device__ __forceinline__ frag columns(const T* tile, int row, int col, int lane) {
    // rows row + 4 half + 0..3 and those 8 on, row a multiple of 16, where Tile::row_at has them
    constexpr int S = Tile<T, DP>::STRIDE;
    const T* const p = tile + row * S + (((lane & 12) + (lane >> 5)) * S + (lane & 16) + 4 * (lane & 3)) + col;
    const s16x4 a = read_columns4(p), b = read_columns4(p + 2 * S);
    return __builtin_bit_cast(frag, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
  }
  static __device__ __forceinline__ frag from_acc(const v16f& x, int s) {
    frag f;
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = (T)x[8 * s + j];
    return f;
  }
};
template <>
struct Mma<__bf16> : Mma16<__bf16> {
  static __device__ __forceinline__ v16f mma(frag a, frag b, v16f c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mma<_Float16> : Mma16<_Float16> {
  static __device__ __forceinline__ v16f mma(frag a, frag b, v16f c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};

// Row of register i of an accumulator in its half's lanes.
__device__ __forceinline__ constexpr int acc_row(int i) { return 8 * (i >> 2) + (i & 3); }

constexpr float LOG2E = 1.4426950408889634f;
constexpr float F32_MAX = 3.402823466e38f;

// Scales whose reciprocal and product with log2 e are far from float32's ends (at which a bias of 0 would become NaN).
inline bool scale_ok(float scale) { return scale >= FX_MIN_SCALE && scale <= FX_MAX_SCALE; }

// A bias in the unit of the raw product q k (scores are c acc, c = scale log2 e): finite entries stay
// finite, so that the type's lowest value weighs like any other and only -inf forbids.
__device__ __forceinline__ float scaled_bias(float b, float inv_scale) {
  const float x = b * inv_scale;
  return isinf(b) || !(fabsf(x) > F32_MAX) ? x : copysignf(F32_MAX, b);
}

// float16 loses digits below 2^-14 and has nothing below 2^-25, where weights of long rows lie (some 1 / keys, and beside
// a dominant key far less) and dS of a small cotangent. Its weights, at most 1, are rounded as 2^15 of them (in
// units of WEIGHT_UNIT), and dS are brought up by a power of two (fit_scale). A product for each weight: 4 % of a long
// forward (699 -> 726 us at 2 x 16 heads x 8192, head dimension 128). In the exponent the 15 would cost nothing, but
// rounds it at 2^-20, which doubled the error of d table.
template <class T>
constexpr bool IS_F16 = __is_same(T, _Float16);
template <class T>
constexpr float WEIGHT_UNIT = IS_F16<T> ? 0x1p-15f : 1.0f;
template <class T>
__device__ __forceinline__ v16f in_units(const v16f& weights) {
  if constexpr (IS_F16<T>) return weights * (1.0f / WEIGHT_UNIT<T>);
  return weights;
}

// The power of two that brings top to [2^(to - 1), 2^to), at most 2^100; 2^to for 0 and what is not finite.
__device__ __forceinline__ float power_to(float top, int to) {
  return __builtin_ldexpf(1.0f, min(to - __builtin_amdgcn_frexp_expf(top), 100));
}

// Scale of a lane's column of dS for a float16 product: dS f is at most 2^15. Starts at SCALE_START and comes down where
// a block's largest asks for it, and what has been summed with it: once for most rows, as it then leaves a factor of 2
// to 4. What is below the largest by 2^-28 keeps its digits. A call with gradients takes 8 % more (3390 -> 3660 us at 2 x 16
// heads x 8192, head dimension 128; 2 % for short sequences), of which the weights' units are a tenth; without it dk of
// cotangents of 1e-4 was 3 % off.
constexpr float SCALE_START = 0x1p60f;
template <int DB>
__device__ __forceinline__ void fit_scale(float& f, const v16f& ds, v16f (&acc)[DB]) {
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(ds[i]));
  top = join32<MaxOp>(top);
  const bool over = top * f > 0x1p15f;
  if (__any(over)) {
    const float next = over ? power_to(top, 14) : f, keep = next * (1.0f / f);
#pragma unroll
    for (int d = 0; d < DB; ++d) acc[d] *= keep;
    f = next;
  }
}

// exp2(c (s - m)) for a block of raw scores. One fma each while c m is small; past BASE_MAX (entries of the
// table like the type's lowest value), where c m's own rounding would be a factor, and always for float32,
// the difference is formed first.
constexpr float BASE_MAX = 1024.0f;
__device__ __forceinline__ void exp_block(v16f& s, float c, float m, float base, bool exact) {
  if (exact) {
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f((s[i] - m) * c);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], c, -base));
  }
}

constexpr int ATT_TILE = 64;  // rows of a staged tile

// A tile of up to 64 rows of dim elements, through registers into LDS: fetch starts the loads, put
// stores them. Rows at or past `rows`, and those that `live` refuses, become zero, so that nothing a
// masked row holds enters a product; columns dim .. DP too.
template <class T, int DP, int NT>
struct TileLoad {
  static constexpr int V = VEC16<T>, CHUNKS = DP / V, PER = ATT_TILE * CHUNKS / NT;
  static_assert(PER >= 1 && PER * NT == ATT_TILE * CHUNKS, "whole turns");
  vec_t<T, V> x[PER];

  template <class L>
  __device__ __forceinline__ void fetch(const T* base, int64_t row_stride, int rows, int dim, bool whole, L&& live) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int at = i * NT + threadIdx.x, r = at / CHUNKS, c = (at % CHUNKS) * V;
      x[i] = {};
      if (r < rows && c < dim && live(r)) {
        const T* p = base + r * row_stride + c;
        if (whole) {
          x[i] = *reinterpret_cast<const vec_t<T, V>*>(p);
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e)
            if (c + e < dim) x[i][e] = p[e];
        }
      }
    }
  }
  __device__ __forceinline__ void put(T* tile) const {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int at = i * NT + threadIdx.x, r = at / CHUNKS, c = (at % CHUNKS) * V;
      *reinterpret_cast<vec_t<T, V>*>(tile + Tile<T, DP>::at(r, c)) = x[i];
    }
  }
};

// The operand of a wave's own rows straight from memory: row c of the lane, all steps.
template <class T, int DP>
struct RowFrags {
  using M = Mma<T>;
  static constexpr int STEPS = DP / M::KS, V = M::KS / 2;
  typename M::frag f[STEPS];
  __device__ __forceinline__ void load(const T* row, bool in, int dim, bool whole, int half) {
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const int c = M::KS * s + V * half;
      typename M::frag x = {};
      if (in && c < dim) {
        if (whole) {
          x = *reinterpret_cast<const typename M::frag*>(row + c);
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e)
            if (c + e < dim) x[e] = row[c + e];
        }
      }
      f[s] = x;
    }
  }
};

// acc += (rows row0 .. row0 + 31 of the tile, row0 a multiple of 16) x (the wave's rows): the tile's rows are the accumulator's.
template <class T, int DP>
__device__ __forceinline__ v16f row_product(const T* tile, int row0, const RowFrags<T, DP>& b, v16f acc, int lane,
                                            int dim) {
  using M = Mma<T>;
  const T* p = tile + row0 * Tile<T, DP>::STRIDE + Tile<T, DP>::at(lane & 31, (M::KS / 2) * (lane >> 5));
#pragma unroll
  for (int s = 0; s < RowFrags<T, DP>::STEPS; ++s) {
    if (sizeof(T) == 4 && M::KS * s >= dim) break;  // float32's products take eight times as long as the branch
    acc = M::mma(*reinterpret_cast<const typename M::frag*>(p + M::KS * s), b.f[s], acc);
  }
  return acc;
}

// acc[d] += (columns 32 d .. of the tile's rows row0 .. row0 + 31, transposed) x p, contracted over the rows.
template <class T, int DP>
__device__ __forceinline__ void column_product(const T* tile, int row0, const v16f& p, v16f (&acc)[DP / 32], int lane,
                                               int dim) {
  using M = Mma<T>;
#pragma unroll
  for (int s = 0; s < 32 / M::KS; ++s) {
    const typename M::frag b = M::from_acc(p, s);
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) {
      if (sizeof(T) == 4 && 32 * d >= dim) break;
      acc[d] = M::mma(M::template columns<DP>(tile, row0 + M::KS * s, 32 * d, lane), b, acc[d]);
    }
  }
}

// Maximum and sum of the lane's value and that of the lane 32 away.
__device__ __forceinline__ float half_max(float x) { return join32<MaxOp>(x); }
__device__ __forceinline__ float half_sum(float x) { return join32<AddOp>(x); }

// A transposed accumulator (rows: 32 d + .. columns of the result; column: the lane's row) times f, as
// rows of memory, 16 bytes a store: the halves of a wave swap what they hold of two groups of eight columns.
// Call with the whole wave; row and in are the lane's (both halves the same).
template <class T, int DP>
__device__ __forceinline__ void store_rows(T* row, bool in, const v16f (&acc)[DP / 32], float f, int dim, bool whole,
                                           int half) {
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int g = 0; g < 4; g += 2) {
      vec_t<T, 4> x[2];  // rounded in one place, so that the ways to store agree
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) x[i][r] = (T)(acc[d][4 * (g + i) + r] * f);
      if constexpr (sizeof(T) == 2) {
        if (whole) {
          typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
          const u32x2 y = __builtin_bit_cast(u32x2, x[0]), z = __builtin_bit_cast(u32x2, x[1]);
          // lanes 0..31 get the even group's eight columns, 32..63 the odd one's
          const auto a = __builtin_amdgcn_permlane32_swap(y[0], z[0], false, false);
          const auto b = __builtin_amdgcn_permlane32_swap(y[1], z[1], false, false);
          const int c = 32 * d + 8 * (g + half);
          if (in && c < dim) *reinterpret_cast<uint4*>(row + c) = make_uint4(a[0], b[0], a[1], b[1]);
          continue;
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int c = 32 * d + 8 * (g + i) + 4 * half;
        if (whole) {
          if (in && c < dim) *reinterpret_cast<vec_t<T, 4>*>(row + c) = x[i];
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (in && c + r < dim) row[c + r] = x[i][r];
        }
      }
    }
}

// What a rounding to T loses, as float16 of LOW_SCALE times it: with the rounded value 19 bits or more.
template <class T>
constexpr float LOW_SCALE = __is_same(T, __bf16) ? 256.0f : 2048.0f;

template <class T, int DP>
__device__ __forceinline__ void store_low(_Float16* row, bool in, const v16f (&acc)[DP / 32], float f, int dim,
                                          bool whole, int half) {
  if (!in) return;
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int c = 32 * d + 8 * g + 4 * half;
      vec_t<_Float16, 4> x;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float v = acc[d][4 * g + r] * f, low = (v - (float)(T)v) * LOW_SCALE<T>;
        x[r] = (_Float16)fmaxf(-65504.0f, fminf(65504.0f, low));
      }
      if (whole) {
        if (c < dim) *reinterpret_cast<vec_t<_Float16, 4>*>(row + c) = x;
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (c + r < dim) row[c + r] = x[r];
      }
    }
}

// Bias of one head. Two forms:
//  - positions that count up (GEN = false): the bias depends on key - query alone, so LDS holds it laid
//    out over the distances -(R + 64) .. R + 64, saturated past R. A lane clamps once a tile, and
//    the tile's values follow at constant offsets; a tile that lies past R as a whole has one value.
//  - positions from memory (GEN = true): each pair's distance is clamped and looked up, map then table.
constexpr int MAX_BUCKETS = FX_MAX_ATTENTION_BUCKETS;
__device__ __host__ constexpr int bias_entries(bool gen, int radius) { return gen ? 2 * radius + 1 : 2 * radius + 129; }
struct BiasView {
  float* table;        // [MAX_BUCKETS]
  float* lut;          // (not GEN) [2 R + 129] over distances
  unsigned char* map;  // GEN: [2 R + 1]; else [2 R + 129] buckets over distances
  int radius;
  __device__ __forceinline__ BiasView(bool gen, unsigned char* at, int r)
      : table(reinterpret_cast<float*>(at)), lut(table + MAX_BUCKETS),
        map(at + 4 * (MAX_BUCKETS + (gen ? 0 : bias_entries(false, r)))), radius(r) {}
};
// Bytes of a BiasView.
constexpr size_t view_lds(bool gen, int radius) {
  return (4 * (size_t)(MAX_BUCKETS + (gen ? 0 : bias_entries(false, radius))) + bias_entries(gen, radius) + 15) / 16 * 16;
}

// Fills the view from `head` of the table (NULL: no bias) in two steps, so that the loads are all on their way at
// once: load (from memory; a barrier follows), lay (within LDS; a barrier follows). All threads.
template <bool GEN, int NT>
__device__ __forceinline__ void load_bias(const fx_attention& p, int head, const BiasView& b, float inv_scale) {
  float x = 0.0f;
  if (p.table && (int)threadIdx.x < p.buckets)
    x = scaled_bias(p.table[(int64_t)threadIdx.x * p.heads + head], inv_scale);
  const int n = bias_entries(GEN, b.radius);
  for (int i = threadIdx.x; i < n; i += NT) {
    const int d = GEN ? i : max(0, min(2 * b.radius, i - 64));
    b.map[i] = p.table ? (unsigned char)min((int)p.map[d], p.buckets - 1) : 0;
  }
  if ((int)threadIdx.x < MAX_BUCKETS) b.table[threadIdx.x] = x;
}
template <bool GEN, int NT>
__device__ __forceinline__ void lay_bias(const BiasView& b) {
  if constexpr (!GEN)
    for (int i = threadIdx.x; i < bias_entries(false, b.radius); i += NT) b.lut[i] = b.table[b.map[i]];
}

// A workgroup's place: items are laid out so that those of one kv head follow each other, and each of
// the eight XCDs (workgroups go to them in turn) gets a contiguous part, whose K and V then stay
// in its L2.
__device__ __forceinline__ int64_t xcd_item(int64_t block, int64_t total) {
  const int64_t per = total / 8, rest = total % 8, x = block % 8;
  return x * per + (x < rest ? x : rest) + block / 8;
}

struct AttArgs {
  fx_attention p;
  int whole;   // rows are whole 16-byte vectors
  float c;     // scale log2(e)
  float inv_scale;
  int weights;  // gradient: whether P is summed beside dS
  int tiles;   // items of a head
  int64_t first, items;  // of a launch
  float* delta;  // gradient: [batch][heads][nq] sum_d out grad_out
  float* part;   // gradient: bucket sums [head][batch * tiles][buckets]
};

// Launches for all items, each of at most as many as its lanes are counted in 32 bits. f(a) launches a.items workgroups.
template <class F>
void launch_items(const AttArgs& args, int tiles, int64_t items, int threads, F&& f) {
  AttArgs a = args;
  a.tiles = tiles;
  const int64_t most = 0xffffffffll / threads;
  for (a.first = 0; a.first < items; a.first += most) {
    a.items = items - a.first < most ? items - a.first : most;
    f(a);
  }
}

// An item's place: sample, head and tile. The heads that share K and V follow each other; within a head the tile with
// the most work under causal comes first: the last of the queries (last_first), the first of the keys.
struct Place {
  int64_t b;
  int h, tile;
  __device__ __forceinline__ Place(const AttArgs& a, int heads, bool last_first) {
    const int64_t item = a.first + xcd_item(blockIdx.x, a.items), bh = item / a.tiles;
    tile = (int)(item - bh * a.tiles);
    if (last_first) tile = a.tiles - 1 - tile;
    b = bh / heads;
    h = (int)(bh - b * heads);
  }
};

// What is left of a tile of keys: bit j of `ok` (GEN: mask), and a position for each key (GEN).
struct KeyView {
  int* pos;                // [64]
  unsigned long long* ok;  // [1]
};
// By one wave, lane j for key k0 + j: from memory with the tile's loads, and into LDS with its stores (a barrier follows).
struct KeyOf {
  int pos;
  bool ok;
};
__device__ __forceinline__ KeyOf key_of(const fx_attention& p, int64_t b, int k0, int len, int lane) {
  const int j = k0 + lane;
  const bool in = j < len;
  return KeyOf{!in ? 0 : p.k_pos ? p.k_pos[b * p.nk + j] : j, in && (!p.mask || p.mask[b * p.nk + j])};
}
__device__ __forceinline__ void put_keys(const KeyOf& key, const KeyView& kv, int lane) {
  kv.pos[lane] = key.pos;
  const unsigned long long m = __ballot(key.ok);
  if (lane == 0) *kv.ok = m;
}

// Position of query i where positions count up. Saturates for the rows past the last query that fill a tile.
__device__ __forceinline__ int counted_pos(const fx_attention& p, int i) {
  return __builtin_elementwise_add_sat(p.offset, i);
}

// Whether a block of keys x queries pairs whose first distance (first key - first query) is d lies past the
// radius as a whole: 1 above, -1 below, 0 neither. Distances run d - (queries - 1) .. d + (keys - 1), which may pass
// the lowest int32 where d does not: the sums are on the radius' side.
__device__ __forceinline__ int far_side(int d, int keys, int queries, int radius) {
  return d >= radius + (queries - 1) ? 1 : d <= -radius - (keys - 1) ? -1 : 0;
}

// Start of a score block of 32 keys (rows k0 + 32 kb + ..) for the lane's query: the bias.
template <bool GEN>
__device__ __forceinline__ v16f bias_block(const fx_attention& p, const BiasView& bv, const KeyView& kv, int kb,
                                           int k0, int qpos, int half, int far) {
  v16f x;
  if (!GEN && far) {
    const float v = bv.lut[far > 0 ? 2 * bv.radius + 128 : 0];
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = v;
  } else if constexpr (GEN) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int4 kp = *reinterpret_cast<const int4*>(kv.pos + 32 * kb + 8 * g + 4 * half);
      const int k[4] = {kp.x, kp.y, kp.z, kp.w};
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        x[4 * g + r] = bv.table[distance_bucket(bv.map, bv.radius, k[r], qpos)];
      }
    }
  } else {
    const int d = max(-(bv.radius + 64), min(bv.radius, k0 - qpos));
    const float* l = bv.lut + d + bv.radius + 64 + 32 * kb + 4 * half;
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = l[acc_row(i)];
  }
  return x;
}

int launch_bucket_join(const float* part, int64_t n, int buckets, int heads, float* out, hipStream_t s);

bool attention_sizes_ok(const fx_attention* p);
bool attention_pointers_ok(const fx_attention& p);
AttArgs attention_args(const fx_attention& p);

// f(type, padded dim, positions or mask from memory)
template <class F>
int attention_shape(const fx_attention& p, F&& f) {
  return with_type<false>(p.dtype, [&](auto t) {
    auto by_gen = [&](auto dp) {
      if (p.q_pos || p.mask)
        f(t, dp, ic<1>{});
      else
        f(t, dp, ic<0>{});
      return launched();
    };
    if (p.dim <= 32) return by_gen(ic<32>{});
    if (p.dim <= 64) return by_gen(ic<64>{});
    return by_gen(ic<128>{});
  });
}

// ------------------------------------------------------------------ gradient

// Buckets of a block's pairs (as bias_block has them).
template <bool GEN>
__device__ __forceinline__ void buckets_of(const BiasView& bv, const KeyView& kv, int kb, int k0, int qpos, int half,
                                           int (&t)[16]) {
  if constexpr (GEN) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int4 kp = *reinterpret_cast<const int4*>(kv.pos + 32 * kb + 8 * g + 4 * half);
      const int k[4] = {kp.x, kp.y, kp.z, kp.w};
#pragma unroll
      for (int r = 0; r < 4; ++r) t[4 * g + r] = distance_bucket(bv.map, bv.radius, k[r], qpos);
    }
  } else {
    const int d = max(-(bv.radius + 64), min(bv.radius, k0 - qpos));
    const unsigned char* l = bv.map + d + bv.radius + 64 + 32 * kb + 4 * half;
#pragma unroll
    for (int i = 0; i < 16; ++i) t[i] = l[acc_row(i)];
  }
}

// The lane's bucket sums: of dS, of its query's P (weights), and what tiles past the
// radius add to the first and the last distance's bucket.
struct Sums {
  float* ds;
  unsigned* weight;
  float all;                    // of dS over all buckets
  float far_ds[2], far_weight[2];  // below, above
};
__device__ __forceinline__ unsigned fixed_weight(float p) { return (unsigned)(p * 0x1p30f); }

// Adds a block's dS and P (rows: keys; column: the lane's query).
template <bool GEN>
__device__ __forceinline__ void bucket_add(const BiasView& bv, const KeyView& kv, Sums& sums, const v16f& ds,
                                           const v16f& w, int kb, int k0, int qpos, int half, int far,
                                           bool weights) {
  if (!GEN && far) {
    float total = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) total += ds[i];
    sums.far_ds[far > 0] += total;
    if (weights) {
#pragma unroll
      for (int i = 0; i < 16; ++i) sums.far_weight[far > 0] += w[i];
    }
    return;
  }
  int t[16];  // all lookups before the first add: the compiler keeps a read that follows one behind it
  buckets_of<GEN>(bv, kv, kb, k0, qpos, half, t);
#pragma unroll
  for (int i = 0; i < 16; i += 2) {
    add_pair(sums.ds, t[i], ds[i], t[i + 1], ds[i + 1]);
  }
  if (weights) {
#pragma unroll
    for (int i = 0; i < 16; ++i) atomicAdd(sums.weight + 32 * t[i], fixed_weight(w[i]));
  }
}

// The gradient of short sequences (attention_short.hip): where it applies. Where heads share K and V it gives dq, the bucket
// sums and delta, and the general second launch dk and dv.
bool attention_grad_short_fits(const fx_attention& p);
int launch_attention_grad_short(const AttArgs& a, hipStream_t s);

}  // namespace net
}  // namespace fx
