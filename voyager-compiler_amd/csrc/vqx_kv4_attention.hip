// Attention over a 4-bit cache of keys and values.
//
// The scores of 16 query rows are formed transposed, S^T = K Q^T, so that a
// lane of the accumulator has one row's scores of several tokens, and the
// output likewise, O^T = V^T P^T: a row's running maximum and sum are then
// values of its lanes, and the weights P leave the first product in the very
// layout the second one takes them in.
//
// Both products are bf16 matrix products with fp32 sums.  Keys and values are
// turned into bf16, which holds every code times its scale exactly.  A query is
// 1, 2 or 3 bf16 terms (bf16, fp16, fp32), which hold it exactly; the weights
// are 2, 3 for fp32 outputs, off by 2^-16 or 2^-24 of themselves: well below
// the half step of their output (2^-8 and 2^-11, 2^-24).  Everything else
// (scores, maxima, sums, outputs until their one rounding) is fp32.
// The scaled product that takes fp4 as it is stored would save the keys'
// conversion (32 of some 250 vector instructions a step), but its other operand
// holds 4 bits, and what is 2^7 and more below the largest product of an
// instruction is cut off: with a query as two e4m3 terms the scores were off by
// 2^-17 of their sums' magnitude in the mean, against 2^-25 here.
#include "vqx_kv4.h"

namespace vqx {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

struct Bf16 {};
struct F16 {};
// What becomes of scores: nothing but the mask of a prompt; a cap or slopes too;
// all that of new tokens that are a tree.  A tree's rows cost little more than a
// prompt's: its masks matter to the last steps only (drafted and plain on the same
// rows, bf16 heads of 128, from a graph: 16 sequences of 4000 with 24 new tokens 59
// and 57 us, 8 of 2000 with 16 23 and 22, 32 of 2000 with 8 28 and 26, 4 of 8000
// with 64 75 and 70; of 400 to 4000 with 24, where trees begin with the longest, 50
// and 55).
enum Mode { kPlain, kCurved, kTreed };
template <typename T>
struct Terms;
template <>
struct Terms<Bf16> {
  static constexpr int kQ = 1, kP = 2;
};
template <>
struct Terms<F16> {
  static constexpr int kQ = 2, kP = 2;
};
template <>
struct Terms<float> {
  static constexpr int kQ = 3, kP = 3;
};

constexpr int kRows = 16;       // query rows of a tile
constexpr int kStep = 32;       // tokens of a wave's step
constexpr int kWaves = 4;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.693147180559945309417f;
constexpr float kLowest = -3.0e38f;  // below every finite score, and finite: no inf - inf
// A row's reference stays until a score passes it by this (in powers of two):
// the weights then stay below 2^8, and the sums are rescaled a few times only.
constexpr float kSlack = 8.0f;
// Values in blocks with a scale byte from here on, 2^88 and up, are taken, as all
// that are summed with them, 2^-40 times as large: the largest codes times the
// largest scales are then within bf16, no weight of 0 meets an infinity, and
// 2^30 weights of 2^8 keep their sums within fp32 (so they do below 2^88).
// Blocks below 2^-87 beside such ones count as 2^-87.
constexpr uint32_t kLargeScale = 215, kDown = 40;
constexpr float kDownFactor = 0x1p-40f, kUpFactor = 0x1p40f;

// 8 values from element i of p as bf16 terms, their sum the value.
__device__ __forceinline__ void load_terms(const void* p, int64_t i, Bf16, u32x4 (&t)[1]) {
  t[0] = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p) + i);
}
template <int kTerms>
__device__ __forceinline__ void split_terms(float (&x)[8], u32x4 (&t)[kTerms]) {
#pragma unroll
  for (int k = 0; k < kTerms; ++k)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t w = pack_bf16x2(x[2 * j], x[2 * j + 1]);
      t[k][j] = w;
      if (k + 1 < kTerms) x[2 * j] -= u2f(w << 16), x[2 * j + 1] -= u2f(w & 0xFFFF0000u);
    }
}
__device__ __forceinline__ void load_terms(const void* p, int64_t i, F16, u32x4 (&t)[2]) {
  const u32x4 a = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p) + i);
  float x[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) x[2 * j] = h2f_exact(a[j] & 0xFFFFu), x[2 * j + 1] = h2f_exact(a[j] >> 16);
  split_terms(x, t);
}
__device__ __forceinline__ void load_terms(const void* p, int64_t i, float, u32x4 (&t)[3]) {
  const f32x4* q = reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + i);
  const f32x4 a = q[0], b = q[1];
  float x[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  split_terms(x, t);
}

// The order of a row's elements in the first product.  Lane (token or row, g)
// of product i has the 8 elements from key_element(i, g): those of a lane are
// 16 bytes of codes for each 128 elements of a head (8 bytes of 64).
template <int D>
__device__ __forceinline__ int key_element(int i, int g) {
  return D == 64 ? 16 * g + 8 * i : 128 * (i / 4) + 32 * g + 8 * (i % 4);
}

// 8 elements of a row's query from element i as the B operand's terms, a
// negative scale's sign included; zeros where the scale is 0.
template <typename T, int kTerms>
__device__ __forceinline__ void load_query(const Kv4Query& q, int64_t i, bool live, T, u32x4 (&t)[kTerms]) {
  const uint32_t flip = q.scale < 0.0f ? 0x80008000u : 0u, keep = q.scale == 0.0f ? 0u : ~0u;
  if (live) {
    load_terms(q.q, i, T(), t);
#pragma unroll
    for (int k = 0; k < kTerms; ++k) t[k] = (t[k] & keep) ^ flip;
  } else {
#pragma unroll
    for (int k = 0; k < kTerms; ++k) t[k] = u32x4{0, 0, 0, 0};
  }
}

// One row's query as that product's B operand.
template <int D, typename T>
struct QueryTerms {
  u32x4 v[D / 32][Terms<T>::kQ];

  __device__ __forceinline__ void load(const Kv4Query& q, int64_t at, bool live, int g) {
#pragma unroll
    for (int i = 0; i < D / 32; ++i) load_query(q, at + key_element<D>(i, g), live, T(), v[i]);
  }
};

// How a call is cut up.  A tile is `rows` query rows of one kv head (row r is
// new token r / group, head r % group); each split of a tile's tokens leaves
// its results in the workspace: rows * D outputs, rows references and rows sums.
struct Kv4Plan {
  int32_t rows, tiles, chunk, splits;
  int32_t listed;  // tiles of a kv head that the workgroups are handed one by one; 0: tiles of every sequence
  bool ranked;     // sequences in the order of their lengths
};

// Where the rows of one tile stand.
struct TileRows {
  int first, count;  // the sequence's first new token and their number
  int base;          // position of new token 0
  int rows;          // count * group
  int lo, hi;        // tokens that any row of the tile sees: [lo, hi), lo a multiple of a step
  int pos_min, pos_max;
};

template <bool kTree = false>
__host__ __device__ __forceinline__ TileRows tile_rows(const Kv4View& c, const Kv4Query& q, uint32_t b, int tile,
                                                       int tile_size, int step) {
  TileRows r;
  kv4_span(q.tokens, b, r.first, r.count);
  // room, new tokens and windows are below 2^30 (checked by the host), a length
  // is kept there, so that no place overflows
  int length = c.lengths[b];
  length = length < 0 ? 0 : (length > (1 << 30) ? 1 << 30 : length);
  r.base = length - r.count;
  const int n = r.count < q.most ? r.count : q.most;
  r.rows = n * q.group;
  const int r0 = tile * tile_size, r1 = r0 + tile_size < r.rows ? r0 + tile_size : r.rows;
  r.pos_min = r.base + r0 / q.group;
  r.pos_max = r1 > r0 ? r.base + (r1 - 1) / q.group : -1;
  if constexpr (kTree) {
    // a row is at a place from base - 1 (of no ancestors, itself not among them)
    // to base + n - 1, and may see any of the n new tokens that the call was told of
    r.pos_min = r.base - 1;
    if (r1 > r0) r.pos_max = r.base + n - 1;
  }
  r.hi = r.pos_max + 1 < 0 ? 0 : ((uint32_t)(r.pos_max + 1) > c.cap ? (int)c.cap : r.pos_max + 1);
  r.lo = 0;
  if (q.window && r.pos_min >= q.window) r.lo = (r.pos_min - q.window + 1) & ~(step - 1);
  if (r.lo > r.hi) r.lo = r.hi & ~(step - 1);
  return r;
}

// The splits of a tile that have sums: as many as the workspace has room for, or
// fewer.
__host__ __device__ __forceinline__ int joined_splits(const TileRows& rows, const Kv4Plan& plan) {
  const int n = rows.hi > rows.lo ? (rows.hi - rows.lo + plan.chunk - 1) / plan.chunk : 1;
  return n < plan.splits ? n : plan.splits;
}

// Sequences and tiles counted through: where tile t of all that there are lies.
__device__ __forceinline__ bool listed_tile(const Kv4View& c, const Kv4Query& q, const Kv4Plan& plan, uint32_t t,
                                            uint32_t& b, int& tile) {
  const int lane = threadIdx.x & 63;
  uint32_t before = 0;
  for (uint32_t b0 = 0; b0 < c.seqs; b0 += 64) {
    int first, count = 0;
    if (b0 + lane < c.seqs) kv4_span(q.tokens, b0 + lane, first, count);
    if (count > q.most) count = q.most;
    // no more than there are at all, whatever the offsets say: below 2^25
    uint32_t mine = ((uint32_t)count * q.group + plan.rows - 1) / (uint32_t)plan.rows;
    if (mine > (uint32_t)plan.listed) mine = plan.listed;
    uint32_t sum = mine;
    for (int d = 1; d < 64; d *= 2) {
      const uint32_t x = (uint32_t)__shfl_up((int)sum, d);
      if (lane >= d) sum += x;
    }
    const uint64_t past = __ballot(before + sum > t);
    if (past) {
      const int l = __builtin_ctzll(past);
      b = b0 + l;
      tile = (int)(t - before - (uint32_t)__builtin_amdgcn_readlane((int)(sum - mine), l));
      return true;
    }
    before += (uint32_t)__builtin_amdgcn_readlane((int)sum, 63);
  }
  return false;
}

// What a workgroup has to do.
struct Place {
  uint32_t b, h, split;
  int tile;
  int64_t at;  // of its sums in the workspace
};

// The i-th longest of up to 64 sequences, for all lanes.
__device__ __forceinline__ uint32_t longest(const Kv4View& c, uint32_t i) {
  const int lane = threadIdx.x & 63, there = lane < (int)c.seqs, length = there ? kv4_length(c, lane) : 0;
  // no two the same: the lane below the length
  const uint32_t mine = there ? (uint32_t)(length < 1 << 25 ? length : (1 << 25) - 1) << 6 | (uint32_t)(63 - lane) : 0;
  uint32_t rank = 0;
  for (int b = 0; b < (int)c.seqs; ++b) rank += (uint32_t)__builtin_amdgcn_readlane((int)mine, b) > mine;
  return (uint32_t)__builtin_ctzll(__ballot(there && rank == i));
}

// Heads first, so that with 8 of them each XCD's L2 has the cache of one (of
// other numbers each XCD gets all in turn, or a long sequence would be one
// XCD's: 4 ragged prompts of 300, 4 heads: 35 and 32 us); then the splits, then
// the tiles from the last, which sees the most.  (Splits and tiles first put
// the first tile of every sequence, often the only one, on one XCD: 64 sequences
// with 128 new tokens at most, all but one with one: 242 and 50 us.)
template <bool kTree = false>
__device__ __forceinline__ bool place_of(const Kv4View& c, const Kv4Query& q, const Kv4Plan& plan, Place& p) {
  if (kTree && plan.ranked) {
    const uint32_t each = c.kv * (uint32_t)(plan.tiles * plan.splits), in = blockIdx.x % each, rest = in / c.kv;
    p.b = longest(c, blockIdx.x / each);
    p.h = (in + (c.kv % 8 ? rest : 0u)) % c.kv, p.split = rest % (uint32_t)plan.splits;
    p.tile = plan.tiles - 1 - (int)(rest / (uint32_t)plan.splits);
    p.at = (((int64_t)p.b * c.kv + p.h) * plan.tiles + p.tile) * plan.splits + p.split;
    return true;
  }
  const uint32_t heads = plan.listed ? c.kv : c.seqs * c.kv, rest = blockIdx.x / heads;
  const uint32_t slot = (blockIdx.x + (c.kv % 8 ? rest : 0u)) % heads;
  p.split = rest % (uint32_t)plan.splits;
  const int t = (plan.listed ? plan.listed : plan.tiles) - 1 - (int)(rest / (uint32_t)plan.splits);
  if (plan.listed) {
    p.h = slot;
    p.at = ((int64_t)t * c.kv + slot) * plan.splits + p.split;
    return listed_tile(c, q, plan, (uint32_t)t, p.b, p.tile);
  }
  p.b = slot / c.kv, p.h = slot % c.kv, p.tile = t;
  p.at = (((int64_t)p.b * c.kv + p.h) * plan.tiles + t) * plan.splits + p.split;
  return true;
}

// What a score becomes, in powers of two: capped by a tanh, less its slope for
// each token of distance.
struct Curve {
  float scale;          // of a plain score, positive: the queries carry its sign
  float inner, outer;   // capped: outer * tanh(score * inner)
  float slope;
  bool capped, sloped;
};

__device__ __forceinline__ Curve curve_of(const Kv4Query& q, int head) {
  Curve k;
  // not 0: a masked score, -inf, stays one (the queries are 0 where the scale is)
  k.scale = __builtin_fmaxf(__builtin_fabsf(q.scale) * kLog2e, 0x1p-126f);
  k.capped = q.softcap != 0.0f;
  k.inner = k.capped ? __builtin_fabsf(q.scale) / q.softcap : 0.0f;
  k.outer = q.softcap * kLog2e;
  k.sloped = q.slopes != nullptr;
  k.slope = q.slopes ? q.slopes[head] * kLog2e : 0.0f;
  return k;
}

// Capped scores of a lane's 8 tokens.  tanh to fp32's own error: up to 0.75 an odd
// polynomial (fitted to 2^-25 of tanh), beyond by the exponential, which no wave
// computes whose scores are all within the polynomial's range: a cap is mostly
// well above.
__device__ __forceinline__ void cap_scores(const Curve& k, float (&x)[8]) {
  if (k.capped) {
    float most = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[j] *= k.inner;
      most = __builtin_fmaxf(most, __builtin_fabsf(x[j]));
    }
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float z = x[j] * x[j];
      float p = __builtin_fmaf(z, -0.00476948991f, 0.0196649131f);
      p = __builtin_fmaf(z, p, -0.0533902584f);
      p = __builtin_fmaf(z, p, 0.133265212f);
      p = __builtin_fmaf(z, p, -0.333330684f);
      y[j] = __builtin_fmaf(x[j] * z, p, x[j]);
    }
    if (__ballot(!(most <= 0.75f))) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float r = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x[j] * (2.0f * kLog2e)));
        y[j] = __builtin_fabsf(x[j]) <= 0.75f ? y[j] : __builtin_fmaf(-2.0f, r, 1.0f);
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = y[j] * k.outer;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] *= k.scale;
  }
}

// Capped and sloped scores of a lane's 8 tokens, of which token j is t0 + (j / 4)
// 16 + j % 4.
__device__ __forceinline__ void curve_scores(const Curve& k, float (&x)[8], int pos, int t0) {
  cap_scores(k, x);
  if (k.sloped) {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] -= k.slope * (float)(pos - (t0 + (j >> 2) * 16 + (j & 3)));
  }
}

// A row among drafted tokens: what it sees of them and where that puts it.
struct Line {
  uint64_t mask;  // its ancestors and itself, as bits of the new tokens
  int base;       // the first new token's place
  int pos;        // the row's: as far behind the cached tokens as it has ancestors
  bool live;
};

__device__ __forceinline__ Line line_of(const Kv4Query& q, const TileRows& rows, int token, bool live) {
  Line l;
  l.live = live;
  l.base = rows.base;
  // bits of tokens beyond `most` lie outside the range that the plan is made for
  const int n = rows.count < q.most ? rows.count : q.most;
  const uint64_t all = n < 64 ? (1ull << n) - 1 : ~0ull;
  l.mask = live ? (uint64_t)q.tree[rows.first + token] & all : 0;
  l.pos = rows.base + __popcll(l.mask) - 1;
  return l;
}

// How far before the row token t is: of the new tokens only the row's ancestors
// count.  -1: it is not seen.
__device__ __forceinline__ int distance(const Line& l, int t) {
  const int d = t - l.base;
  if (d < 0) return l.live ? l.pos - t : -1;
  return d < 64 && (l.mask >> d & 1u) ? (int)__popcll(l.mask >> d >> 1) : -1;
}

// Slopes and mask of a row among drafted tokens on its capped scores; which of
// the 8 it sees, as bits.  Token j is t0 + (j / 4) 16 + j % 4, bit u + 16 (j / 4) + j
// % 4 of valid says that it is there.
__device__ __forceinline__ uint32_t line_scores(const Curve& k, const Line& l, float (&x)[8], uint32_t valid, int u, int t0,
                                                int window) {
  uint32_t seen = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int i = (j >> 2) * 16 + (j & 3), away = distance(l, t0 + i);
    const bool in = (valid >> (u + i) & 1u) && away >= 0 && (window == 0 || away < window);
    x[j] = in ? x[j] - k.slope * (float)away : -__builtin_huge_valf();
    seen |= (uint32_t)in << j;
  }
  return seen;
}

// The keys and values of one step of 32 tokens as a wave's loads leave them.
// Keys: lane (token & 15, g) has key_element's codes of its token, twice, and
// the scales they need.  Values: lane
// (m, g) has the D / 16 elements from m D / 16 of tokens 4 g .. 4 g + 3 and
// 16 + 4 g .. 16 + 4 g + 3, and all scale bytes of those tokens.
template <int D>
struct Loaded {
  static constexpr int kGroups = (D + 127) / 128;
  static constexpr int kWords = D == 256 ? 2 : 1;     // of a token's values
  static constexpr int kScaleWords = D / 32;          // of four tokens' scales
  uint32_t k[2][D / 32];
  uint32_t ks[2][kGroups];
  uint32_t v[8][kWords];
  uint32_t vs[2][kScaleWords];
  uint32_t valid;  // bit t: token t of the step is there
  int t0;
};

// codes + at, scales + scale_at: a token's key; the offsets apart, so that a
// common base stays in scalar registers.
template <int D>
__device__ __forceinline__ void load_keys(const uint8_t* codes, const uint8_t* scales, uint32_t at, uint32_t scale_at,
                                          int g, uint32_t (&k)[D / 32], uint32_t (&s)[Loaded<D>::kGroups]) {
  if constexpr (D == 64) {
    const u32x2 a = *reinterpret_cast<const u32x2*>(codes + (at + 8 * g));
    k[0] = a[0], k[1] = a[1];
    s[0] = scales[scale_at + (g >> 1)];
  } else {
#pragma unroll
    for (int a = 0; a < D / 128; ++a) {
      const u32x4 w = *reinterpret_cast<const u32x4*>(codes + (at + 16 * g) + 64 * a);
#pragma unroll
      for (int i = 0; i < 4; ++i) k[4 * a + i] = w[i];
      s[a] = scales[(scale_at + g) + 4 * a];
    }
  }
}

template <int D>
__device__ __forceinline__ void load_values(const uint8_t* p, uint32_t (&w)[Loaded<D>::kWords]) {
  if constexpr (D == 64) {
    w[0] = *reinterpret_cast<const uint16_t*>(p);
  } else if constexpr (D == 128) {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else {
    const u32x2 a = *reinterpret_cast<const u32x2*>(p);
    w[0] = a[0], w[1] = a[1];
  }
}

struct __attribute__((packed, aligned(1))) Raw16 {
  u32x4 v;
};
struct __attribute__((packed, aligned(1))) Raw8 {
  u32x2 v;
};

// A whole step on one page: one base, and offsets that are constants.  `row` is
// its first token's.
template <int D>
__device__ __forceinline__ void load_whole(const Kv4View& c, uint32_t page, uint32_t row, int t0, int lane,
                                           Loaded<D>& s) {
  constexpr int kRow = D / 2, kScales = D / 32;
  const int m = lane & 15, g = lane >> 4;
  s.t0 = t0;
  s.valid = page < c.pages ? 0xFFFFFFFFu : 0u;
  const uint8_t* kc = c.codes + (uint64_t)row * kRow;
  const uint8_t* ks = c.scales + (uint64_t)row * kScales;
#pragma unroll
  for (int i = 0; i < 2; ++i)
    load_keys<D>(kc, ks, (uint32_t)((i * 16 + m) * kRow), (uint32_t)((i * 16 + m) * kScales), g, s.k[i], s.ks[i]);
  const uint64_t vrow = c.plane_rows + row;
  const uint8_t* vc = c.codes + vrow * kRow;
  const uint8_t* vs = c.scales + vrow * kScales;
#pragma unroll
  for (int j = 0; j < 8; ++j)
    load_values<D>(vc + (uint32_t)(4 * g * kRow + m * (kRow / 16)) + ((j >> 2) * 16 + (j & 3)) * kRow, s.v[j]);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    // four tokens' scales are next to each other, not always on 16 bytes
    const uint8_t* p = vs + (uint32_t)(4 * g * kScales) + i * 16 * kScales;
    if constexpr (D == 64) {
      const u32x2 a = reinterpret_cast<const Raw8*>(p)->v;
      s.vs[i][0] = a[0], s.vs[i][1] = a[1];
    } else {
#pragma unroll
      for (int k = 0; k < kScales / 4; ++k) {
        const u32x4 a = reinterpret_cast<const Raw16*>(p)[k].v;
#pragma unroll
        for (int x = 0; x < 4; ++x) s.vs[i][4 * k + x] = a[x];
      }
    }
  }
}

// Any step: lane l (and l + 32) has the page of token l and finds its row; past
// the end that is the last token's, which no row counts.
template <int D, bool kValues>
__device__ __forceinline__ void load_any(const Kv4View& c, uint32_t h, uint32_t page, int t0, int end, int lane,
                                         Loaded<D>& s) {
  constexpr int kRow = D / 2, kScales = D / 32;
  const int m = lane & 15, g = lane >> 4;
  const int t = t0 + (lane & 31);
  const uint32_t mine = kv4_row(c, page, h, (uint32_t)(t < end ? t : end - 1));
  s.t0 = t0;
  s.valid = (uint32_t)__ballot(t < end && page < c.pages);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint64_t row = (uint32_t)__shfl((int)mine, 16 * i + m);
    load_keys<D>(c.codes + row * kRow, c.scales + row * kScales, 0u, 0u, g, s.k[i], s.ks[i]);
  }
  if constexpr (kValues) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint64_t row = c.plane_rows + (uint32_t)__shfl((int)mine, (j >> 2) * 16 + 4 * g + (j & 3));
      load_values<D>(c.codes + row * kRow + m * (kRow / 16), s.v[j]);
      const uint8_t* p = c.scales + row * kScales;
      if constexpr (D == 64) {
        const uint32_t w = *reinterpret_cast<const uint16_t*>(p);
        s.vs[j >> 2][(j & 3) >> 1] = (j & 1) ? s.vs[j >> 2][(j & 3) >> 1] | w << 16 : w;
      } else if constexpr (D == 128) {
        s.vs[j >> 2][j & 3] = *reinterpret_cast<const uint32_t*>(p);
      } else {
        const u32x2 a = *reinterpret_cast<const u32x2*>(p);
        s.vs[j >> 2][2 * (j & 3)] = a[0], s.vs[j >> 2][2 * (j & 3) + 1] = a[1];
      }
    }
  }
}

// bf16x2 words of the two values whose codes are byte kByte of w.  The scale's
// exponent counts: 0 is 2^-127, that of an infinity makes a NaN.
template <int kByte>
__device__ __forceinline__ uint32_t fp4_pair(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, kByte));
}

// Scores of the step's tokens 16 i + 4 g + r in x[4 i + r], lane (row, g).
template <int D, typename T>
__device__ __forceinline__ void step_scores(const QueryTerms<D, T>& q, const Loaded<D>& s, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    f32x4 acc = {0, 0, 0, 0};
#pragma unroll
    for (int a = 0; a < D / 32; ++a) {
      const float scale = u2f(s.ks[i][a / 4] << 23);
      const uint32_t w = s.k[i][a];
      const u32x4 k = {fp4_pair<0>(w, scale), fp4_pair<1>(w, scale), fp4_pair<2>(w, scale), fp4_pair<3>(w, scale)};
#pragma unroll
      for (int t = 0; t < Terms<T>::kQ; ++t)
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, k), __builtin_bit_cast(bf16x8, q.v[a][t]),
                                                      acc, 0, 0, 0);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) x[4 * i + r] = acc[r];
  }
}

// The row's curve and mask on those scores; seen: bit 4 i + r.
template <Mode kMode>
__device__ __forceinline__ void finish_scores(const Curve& k, const Line& line, float (&x)[8], uint32_t valid, int t0, int g,
                                              int pos, int window, bool masked, uint32_t& seen) {
  seen = 0xFFu;
  if constexpr (kMode == kTreed) {
    if (masked) {
      cap_scores(k, x);
      seen = line_scores(k, line, x, valid, 4 * g, t0 + 4 * g, window);
    } else {
      curve_scores(k, x, pos, t0 + 4 * g);
    }
    return;
  }
  if (kMode == kCurved) {
    curve_scores(k, x, pos, t0 + 4 * g);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] *= k.scale;
  }
  if (masked) {
    seen = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int u = (j >> 2) * 16 + 4 * g + (j & 3), t = t0 + u;
      const bool in = (valid >> u & 1u) && t <= pos && (window == 0 || t > pos - window);
      x[j] = in ? x[j] : -__builtin_huge_valf();
      seen |= (uint32_t)in << j;
    }
  }
}

__device__ __forceinline__ bool needs_mask(const TileRows& r, uint32_t valid, int t0, int window) {
  return valid != 0xFFFFFFFFu || t0 + kStep - 1 > r.pos_min || (window && t0 <= r.pos_max - window);
}

__device__ __forceinline__ void put(void* out, int64_t i, float v, float) { static_cast<float*>(out)[i] = v; }
__device__ __forceinline__ void put(void* out, int64_t i, float v, Bf16) {
  static_cast<uint16_t*>(out)[i] = (uint16_t)f2bf(v);
}
__device__ __forceinline__ void put(void* out, int64_t i, float v, F16) {
  static_cast<uint16_t*>(out)[i] = (uint16_t)f2h_exact(v);
}
// 4 consecutive elements, i a multiple of 4
__device__ __forceinline__ void put4(void* out, int64_t i, f32x4 v, float) {
  *reinterpret_cast<f32x4*>(static_cast<float*>(out) + i) = v;
}
__device__ __forceinline__ void put4(void* out, int64_t i, f32x4 v, Bf16) {
  *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(out) + i) = u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
}
__device__ __forceinline__ void put4(void* out, int64_t i, f32x4 v, F16) {
  *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(out) + i) =
      u32x2{f2h_exact(v[0]) | f2h_exact(v[1]) << 16, f2h_exact(v[2]) | f2h_exact(v[3]) << 16};
}

// A sequence with more new tokens than the call was told of: their rows have
// no result.
template <int D, typename T>
__device__ __forceinline__ void fill_beyond(const Kv4Query& q, const TileRows& rows, uint32_t h, void* out,
                                            float* lse) {
  const int64_t extra = (int64_t)(rows.count - q.most) * q.group;
  for (int64_t e = threadIdx.x; e < extra; e += 256) {
    const int64_t row = (int64_t)(rows.first + q.most + e / q.group) * q.heads + (int64_t)h * q.group + e % q.group;
    lse[row] = __builtin_nanf("");
    for (int d = 0; d < D; ++d) put(out, row * D + d, __builtin_nanf(""), T());
  }
}

// Few rows, many tokens: the cache is read once for each tile of 16 rows, and
// that reading is the bound.  A workgroup has one tile, one kv head and one
// run of tokens; its four waves take steps of 32 tokens in turn, each straight
// from memory into the operands' registers, one step ahead, and are joined at
// the end.  64 sequences of 4096 tokens, 32 kv heads of 128, bf16: 178 us, 5.6
// TB/s.  With fewer tokens a workgroup's own time shows: 4.5 us and 0.7 us for
// each step of its waves (one sequence of 131073 tokens, 8 kv heads: 33 us, 4.3
// TB/s; 16 of 4000 at most: 19 us).
template <int D, typename T, Mode kMode, bool kWhole>
__global__ __launch_bounds__(256, D == 64 ? 3 : (D == 128 ? 2 : 1)) void kv4_rows_kernel(Kv4View c, Kv4Query q,
                                                                                        Kv4Plan plan, void* out,
                                                                                        float* lse, float* ws) {
  constexpr int kTiles = D / 16;  // of 16 output elements
  constexpr int kPer = D / 4;     // output elements of a lane
  constexpr int kPad = D + 4;
  __shared__ __align__(16) float part[2][kRows][kPad];
  __shared__ float part_m[2][kRows], part_l[2][kRows];
  __shared__ uint32_t part_bad[2][kRows];
  __shared__ int part_down[2];
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  Place place;
  if (!place_of<kMode == kTreed>(c, q, plan, place)) return;
  const uint32_t b = place.b, h = place.h, split = place.split;
  const int tile = place.tile;
  const TileRows rows = tile_rows<kMode == kTreed>(c, q, b, tile, kRows, kStep);
  const int r = tile * kRows + n;
  const bool live = r < rows.rows;
  const int token = r / q.group, head = (int)h * q.group + r % q.group;
  const int64_t at_row = (int64_t)(rows.first + token) * q.heads + head;
  if (rows.count > q.most && tile == 0 && split == 0) fill_beyond<D, T>(q, rows, h, out, lse);
  if (tile * kRows >= rows.rows) return;
  const int begin = rows.lo + (int)split * plan.chunk;
  int end = begin + plan.chunk;
  if (end > rows.hi) end = rows.hi;
  if (begin >= end && split > 0) return;
  const int steps = begin < end ? (end - begin + kStep - 1) / kStep : 0;
  Line line = {};
  if constexpr (kMode == kTreed) line = line_of(q, rows, token, live);
  const int pos = kMode == kTreed ? line.pos : (live ? rows.base + token : -1);
  const Curve curve = curve_of(q, live ? head : (int)h * q.group);

  float m = kLowest, l = 0.0f;
  uint32_t bad = 0;  // blocks of values that are NaN in a token the row sees
  bool down = false;  // the wave's outputs are 2^-kDown of themselves
  f32x4 acc[kTiles];
#pragma unroll
  for (int j = 0; j < kTiles; ++j) acc[j] = f32x4{0, 0, 0, 0};

  if (wave < steps) {
    QueryTerms<D, T> terms;
    terms.load(q, (int64_t)(rows.first + token) * q.sn + (int64_t)head * q.sh, live, g);

    // the page of this lane's token in step s
    auto page_of = [&](int s) -> uint32_t {
      const int t = begin + s * kStep + (lane & 31);
      return kv4_page(c, b, (uint32_t)(t < end ? t : end - 1));
    };
    auto work = [&](const Loaded<D>& s) {
      float x[8];
      step_scores<D, T>(terms, s, x);
      const bool masked = needs_mask(rows, s.valid, s.t0, q.window);
      uint32_t seen;
      finish_scores<kMode>(curve, line, x, s.valid, s.t0, g, pos, q.window, masked, seen);
      float top = x[0];
#pragma unroll
      for (int j = 1; j < 8; ++j) top = __builtin_fmaxf(top, x[j]);
      if (__ballot(top > m + kSlack)) {
        top = __builtin_fmaxf(top, __shfl_xor(top, 16));
        top = __builtin_fmaxf(top, __shfl_xor(top, 32));
        const float next = __builtin_fmaxf(m, top), f = __builtin_amdgcn_exp2f(m - next);
        m = next;
        l *= f;
#pragma unroll
        for (int j = 0; j < kTiles; ++j) acc[j] *= f;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = __builtin_amdgcn_exp2f(x[j] - m), l += x[j];
      u32x4 p[Terms<T>::kP];
      split_terms(x, p);
      // this lane's block of each token's scales
      uint32_t vs[8];
      const uint32_t block = (uint32_t)n * (D / 16) / 32;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        uint32_t w;
        if constexpr (D == 64)
          w = s.vs[j >> 2][(j & 3) >> 1] >> (16 * (j & 1));
        else if constexpr (D == 128)
          w = s.vs[j >> 2][j & 3];
        else
          w = block >= 4 ? s.vs[j >> 2][2 * (j & 3) + 1] : s.vs[j >> 2][2 * (j & 3)];
        vs[j] = w >> (8 * (block & 3)) & 0xFFu;
      }
      uint32_t most = vs[0];
#pragma unroll
      for (int j = 1; j < 8; ++j) most = umax32(most, vs[j]);
      if (__ballot(most >= kLargeScale) || down) {
        // 255: a weight of 0 must not meet a NaN.  The value is taken as tiny, and
        // the rows that see the token note its blocks.  A token that is not there
        // has the scales of another one, or of none.
        most = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          uint32_t nan = 0;
#pragma unroll
          for (int k = 0; k < D / 32; ++k) {
            const int byte = (j & 3) * (D / 32) + k;
            nan |= (uint32_t)((s.vs[j >> 2][byte >> 2] >> (8 * (byte & 3)) & 0xFFu) == 255u) << k;
          }
          if (seen >> j & 1u) bad |= nan;
          if (vs[j] == 255u || !(s.valid >> ((j >> 2) * 16 + 4 * g + (j & 3)) & 1u)) vs[j] = 0;
          most = umax32(most, vs[j]);
        }
        if (!down && __ballot(most >= kLargeScale)) {
          down = true;
#pragma unroll
          for (int j = 0; j < kTiles; ++j) acc[j] *= kDownFactor;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) vs[j] = __builtin_elementwise_sub_sat(vs[j], down ? kDown : 0u);
      }
      float f[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = u2f(vs[j] << 23);
#pragma unroll
      for (int w = 0; w < Loaded<D>::kWords; ++w) {
        // byte by byte: two elements of two tokens in one word each, then the
        // halves exchanged so that a word has two tokens of one element
        auto product = [&](auto which) {
          constexpr int kByte = decltype(which)::value;
          u32x4 even, odd;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t x0 = fp4_pair<kByte>(s.v[2 * j][w], f[2 * j]),
                           x1 = fp4_pair<kByte>(s.v[2 * j + 1][w], f[2 * j + 1]);
            even[j] = __builtin_amdgcn_perm(x1, x0, 0x05040100u);
            odd[j] = __builtin_amdgcn_perm(x1, x0, 0x07060302u);
          }
          constexpr int kTile = 2 * kByte;
#pragma unroll
          for (int t = 0; t < Terms<T>::kP; ++t) {
            const bf16x8 pt = __builtin_bit_cast(bf16x8, p[t]);
            acc[8 * w + kTile] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, even), pt,
                                                                         acc[8 * w + kTile], 0, 0, 0);
            acc[8 * w + kTile + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, odd), pt,
                                                                             acc[8 * w + kTile + 1], 0, 0, 0);
          }
        };
        product(std::integral_constant<int, 0>());
        product(std::integral_constant<int, 1>());
        if constexpr (D > 64) {
          product(std::integral_constant<int, 2>());
          product(std::integral_constant<int, 3>());
        }
      }
    };

    // steps that lie whole on a page go round this loop, two of them in flight
    const int round = kWhole ? (end - begin) / kStep : steps;
    Loaded<D> one, two;
    uint32_t page = 0;
    auto load = [&](int s, Loaded<D>& to) {
      const int t0 = begin + s * kStep;
      if constexpr (kWhole) {
        const uint32_t pg = (uint32_t)__builtin_amdgcn_readfirstlane((int)page);
        load_whole<D>(c, pg, (uint32_t)__builtin_amdgcn_readfirstlane((int)kv4_row(c, pg, h, (uint32_t)t0)), t0, lane, to);
      } else {
        load_any<D, true>(c, h, page, t0, end, lane, to);
      }
      page = page_of(s + kWaves);
    };
    if (wave < round) {
      page = page_of(wave);
      load(wave, one);
      int s = wave;
      while (true) {
        // the last round loads its own step again
        load(s + kWaves < round ? s + kWaves : s, two);
        work(one);
        s += kWaves;
        if (s >= round) break;
        load(s + kWaves < round ? s + kWaves : s, one);
        work(two);
        s += kWaves;
        if (s >= round) break;
      }
    }
    if (kWhole && round < steps && wave == round % kWaves) {
      load_any<D, true>(c, h, page_of(round), begin + round * kStep, end, lane, one);
      work(one);
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    bad |= (uint32_t)__shfl_xor((int)bad, 16);
    bad |= (uint32_t)__shfl_xor((int)bad, 32);
  }

  // join the waves: 2 and 3 into 0 and 1, then 1 into 0
#pragma unroll
  for (int half = 2; half >= 1; half /= 2) {
    if (wave >= half && wave < 2 * half) {
      const int z = wave - half;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < kTiles; j += 4)
          *reinterpret_cast<f32x4*>(&part[z][n][g * kPer + i * kTiles + j]) =
              f32x4{acc[j][i], acc[j + 1][i], acc[j + 2][i], acc[j + 3][i]};
      if (g == 0) part_m[z][n] = m, part_l[z][n] = l, part_bad[z][n] = bad;
      if (lane == 0) part_down[z] = down;
    }
    __syncthreads();
    if (wave < half) {
      const float m1 = part_m[wave][n], top = __builtin_fmaxf(m, m1);
      const float f0 = __builtin_amdgcn_exp2f(m - top), f1 = __builtin_amdgcn_exp2f(m1 - top);
      m = top;
      l = l * f0 + part_l[wave][n] * f1;
      bad |= part_bad[wave][n];
      const bool down1 = part_down[wave] != 0;
      const float a0 = down1 && !down ? f0 * kDownFactor : f0, a1 = down && !down1 ? f1 * kDownFactor : f1;
      down = down || down1;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < kTiles; j += 4) {
          const f32x4 o = *reinterpret_cast<const f32x4*>(&part[wave][n][g * kPer + i * kTiles + j]);
#pragma unroll
          for (int x = 0; x < 4; ++x) acc[j + x][i] = acc[j + x][i] * a0 + o[x] * a1;
        }
    }
    __syncthreads();
  }
  if (wave != 0) return;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l, up = down ? kUpFactor : 1.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < kTiles; ++j) {
      const uint32_t block = (uint32_t)(g * kPer + i * kTiles + j) / 32;
      acc[j][i] = bad >> block & 1u ? __builtin_nanf("") : acc[j][i] * inv * up;
    }
  if (plan.splits > 1) {
    float* o = ws + place.at * (kRows * D + 2 * kRows);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < kTiles; j += 4)
        *reinterpret_cast<f32x4*>(o + n * D + g * kPer + i * kTiles + j) =
            f32x4{acc[j][i], acc[j + 1][i], acc[j + 2][i], acc[j + 3][i]};
    if (g == 0) o[kRows * D + n] = m, o[kRows * D + kRows + n] = l;
    return;
  }
  if (!live) return;
  if (g == 0) lse[at_row] = l == 0.0f ? -__builtin_huge_valf() : (m + __builtin_amdgcn_logf(l)) * kLn2;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < kTiles; j += 4)
      put4(out, at_row * D + g * kPer + i * kTiles + j, f32x4{acc[j][i], acc[j + 1][i], acc[j + 2][i], acc[j + 3][i]},
           T());
}


// Tokens of a step of the kernel for many rows.
constexpr int kBlockStep = 64;
// Tiles of 16 rows of a wave: 2, and 1 where the registers do not hold the
// queries' terms and the outputs of 2.
constexpr int block_sub(int dim, int q_terms) { return dim * q_terms > 256 ? 1 : 2; }
// Many rows: a workgroup has 128 rows of one kv head, 32 of them a wave (64 and
// 16 where a wave has one tile), and walks over the tokens by 64.  Keys and
// values of a step are turned into bf16 once, the values transposed, into LDS
// (two buffers, one barrier a step), and read by all four waves.  Bound by the
// matrix instructions (busy for 46% of the SIMDs' cycles) and the vector ones of
// the softmax (issuing for 56%), which two waves a SIMD overlap a little: a prompt
// of 8192 tokens, 32 heads over 8 of 128, 740 us; its 824 GFLOP with both terms
// of the weights at 1.11 PFLOP/s, where a large library product reaches 1.21.
//
// Weights of bf16 outputs are two bf16 terms here as in the other kernel, a
// third of the matrix work more than one.  As one fp16 term, with the values as
// fp16 relative to the largest scale that the workgroup had met, the same prompt
// took 660 us; but values 2^36 below that scale came back as zeros, also where
// it was another block's, or that of a token that the row does not see.
template <int D, typename T, Mode kMode, bool kWhole>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void kv4_block_kernel(Kv4View c, Kv4Query q, Kv4Plan plan, void* out,
                                                                         float* lse, float* ws) {
  constexpr int kTiles = D / 16;
  constexpr int kVWords = Loaded<D>::kWords, kKWords = D / 32, kRow = D / 2, kScales = D / 32;
  constexpr int kKScales = D == 256 ? 2 : 1;  // of a thread's keys
  constexpr int kP = Terms<T>::kP;
  constexpr int kSub = block_sub(D, Terms<T>::kQ), kBlockRows = 64 * kSub;
  // rows a 16-byte bank group off each other's
  __shared__ __align__(16) uint16_t kt[2][kBlockStep][D + 8];
  __shared__ __align__(16) uint16_t vt[2][D][kBlockStep + 8];
  // the last even and odd step with a NaN block of values, and with a large one
  __shared__ int notes[2][2];
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  Place place;
  if (!place_of<kMode == kTreed>(c, q, plan, place)) return;
  const uint32_t b = place.b, h = place.h, split = place.split;
  const int tile = place.tile;
  constexpr bool kTree = kMode == kTreed;
  const TileRows rows = tile_rows<kTree>(c, q, b, tile, kBlockRows, kBlockStep);
  if (rows.count > q.most && tile == 0 && split == 0) fill_beyond<D, T>(q, rows, h, out, lse);
  if (tile * kBlockRows >= rows.rows) return;
  const int begin = rows.lo + (int)split * plan.chunk;
  int end = begin + plan.chunk;
  if (end > rows.hi) end = rows.hi;
  if (begin >= end && split > 0) return;
  const int steps = begin < end ? (end - begin + kBlockStep - 1) / kBlockStep : 0;

  // the wave's own rows
  const int r0 = tile * kBlockRows + wave * kSub * 16;
  const TileRows mine = tile_rows<kTree>(c, q, b, tile * kWaves + wave, 16 * kSub, kStep);
  int row[kSub], pos[kSub];
  Line line[kSub];
  Curve curve[kSub];
  u32x4 terms[kSub][kKWords][Terms<T>::kQ];
#pragma unroll
  for (int y = 0; y < kSub; ++y) {
    row[y] = r0 + 16 * y + n;
    const bool live = row[y] < rows.rows;
    const int token = row[y] / q.group, head = (int)h * q.group + row[y] % q.group;
    pos[y] = live ? rows.base + token : -1;
    if constexpr (kTree) line[y] = line_of(q, rows, token, live), pos[y] = line[y].pos;
    curve[y] = curve_of(q, live ? head : (int)h * q.group);
    const int64_t at = (int64_t)(rows.first + token) * q.sn + (int64_t)head * q.sh;
#pragma unroll
    for (int a = 0; a < kKWords; ++a) load_query(q, at + 32 * a + 8 * g, live, T(), terms[y][a]);
  }
  float m[kSub], l[kSub];
  uint32_t bad[kSub];
  f32x4 acc[kSub][kTiles];
#pragma unroll
  for (int y = 0; y < kSub; ++y) {
    m[y] = kLowest, l[y] = 0.0f, bad[y] = 0;
#pragma unroll
    for (int j = 0; j < kTiles; ++j) acc[y][j] = f32x4{0, 0, 0, 0};
  }
  uint32_t down = 0;  // kDown: values and outputs are 2^-kDown of themselves
  if (tid < 4) notes[tid >> 1][tid & 1] = -1;

  // Loads go round without a branch, so that each wait is for its own: a token
  // past the end is the last one, which no row counts.  Where pages hold whole
  // steps (kWhole) a step has one base, its page looked up a step ahead;
  // otherwise every thread looks its tokens' pages up, a step ahead too.
  // Keys: thread (token, part) has D / 4 elements of a token; values: thread
  // (quad, part) has D / 16 of four tokens.
  const int k_token = tid >> 2, k_part = tid & 3;
  const int quad = tid & 15, element = (tid >> 4) * (D / 16);
  struct Pages {
    uint32_t k, v[4], all;  // kWhole: k only
  };
  auto clamped = [&](int t) { return (uint32_t)(t < end ? t : end - 1); };
  auto pages_of = [&](int step, Pages& p) {
    const int t0 = begin + step * kBlockStep;
    if constexpr (kWhole) {
      p.k = kv4_page(c, b, clamped(t0));
    } else {
      p.k = kv4_page(c, b, clamped(t0 + k_token));
      p.all = kv4_page(c, b, clamped(t0 + lane));
#pragma unroll
      for (int i = 0; i < 4; ++i) p.v[i] = kv4_page(c, b, clamped(t0 + 4 * quad + i));
    }
  };
  uint32_t k[kKWords], ks[kKScales], v[4][kVWords], vs[4], v_pages;
  auto take_keys = [&](const uint8_t* codes, const uint8_t* scales, uint32_t at, uint32_t scale_at) {
    if constexpr (D == 64) {
      const u32x2 a = *reinterpret_cast<const u32x2*>(codes + (at + 8 * k_part));
      k[0] = a[0], k[1] = a[1];
      ks[0] = scales[scale_at + k_part / 2];
    } else {
#pragma unroll
      for (int i = 0; i < kKScales; ++i) {
        const u32x4 a = *reinterpret_cast<const u32x4*>(codes + (at + 16 * kKScales * k_part) + 16 * i);
#pragma unroll
        for (int j = 0; j < 4; ++j) k[4 * i + j] = a[j];
        ks[i] = scales[(scale_at + kKScales * k_part) + i];
      }
    }
  };
  // returns bit t: token t of the step is there
  auto load = [&](int step, const Pages& p) -> uint64_t {
    const int t0 = begin + step * kBlockStep;
    if constexpr (kWhole) {
      const uint32_t page = (uint32_t)__builtin_amdgcn_readfirstlane((int)p.k);
      const int first = t0 < end ? t0 : end - 1, last = end - 1 - first;
      const uint64_t at = kv4_row(c, page, h, (uint32_t)first), v_at = c.plane_rows + at;
      const uint32_t u = (uint32_t)(k_token < last ? k_token : last);
      take_keys(c.codes + at * kRow, c.scales + at * kScales, u * kRow, u * kScales);
      const uint8_t* codes = c.codes + v_at * kRow;
      const uint8_t* scales = c.scales + v_at * kScales;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t w = (uint32_t)(4 * quad + i < last ? 4 * quad + i : last);
        load_values<D>(codes + (w * kRow + element / 2), v[i]);
        vs[i] = scales[w * kScales + element / 32];
      }
      v_pages = page < c.pages ? 0xFu : 0u;
      const int left = end - t0;
      const uint64_t there = left >= kBlockStep ? ~0ull : (left > 0 ? (1ull << left) - 1 : 0ull);
      return page < c.pages ? there : 0ull;
    } else {
      const uint64_t at = kv4_row(c, p.k, h, clamped(t0 + k_token));
      take_keys(c.codes + at * kRow, c.scales + at * kScales, 0u, 0u);
      v_pages = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint64_t v_at = c.plane_rows + kv4_row(c, p.v[i], h, clamped(t0 + 4 * quad + i));
        load_values<D>(c.codes + v_at * kRow + element / 2, v[i]);
        vs[i] = c.scales[v_at * kScales + element / 32];
        v_pages |= (uint32_t)(p.v[i] < c.pages) << i;
      }
      return __ballot(t0 + lane < end && p.all < c.pages);
    }
  };
  // The scales of the step whose values were loaded last.
  auto note_scales = [&](int step) {
    if (umax32(umax32(vs[0], vs[1]), umax32(vs[2], vs[3])) < kLargeScale) return;
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (!(v_pages >> i & 1u)) vs[i] = 0;  // a token without a page has another's scales, or none's
      if (vs[i] == 255) notes[step & 1][0] = step, vs[i] = 0;
      most = umax32(most, vs[i]);
    }
    if (most >= kLargeScale) notes[step & 1][1] = step;
  };
  // A step's place in LDS: a lane of the second product takes tokens
  // 4 g .. 4 g + 3 and 16 + 4 g .. of 32 as 16 bytes.
  auto store_keys = [&](int step) {
    uint16_t* kto = &kt[step & 1][k_token][k_part * (D / 4)];
#pragma unroll
    for (int i = 0; i < kKWords; ++i) {
      const float f = u2f(ks[i / 4] << 23);
      *reinterpret_cast<u32x4*>(kto + 8 * i) =
          u32x4{fp4_pair<0>(k[i], f), fp4_pair<1>(k[i], f), fp4_pair<2>(k[i], f), fp4_pair<3>(k[i], f)};
    }
  };
  auto store_values = [&](int step) {
    uint16_t* to = &vt[step & 1][element][32 * (quad >> 3) + 8 * (quad & 3) + 4 * (quad >> 2 & 1)];
    constexpr int kNext = kBlockStep + 8;
    float f[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = u2f(__builtin_elementwise_sub_sat(vs[i], down) << 23);
#pragma unroll
    for (int w = 0; w < kVWords; ++w) {
      auto pair = [&](auto which) {
        constexpr int kByte = decltype(which)::value;
        uint32_t x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = fp4_pair<kByte>(v[i][w], f[i]);
        const u32x2 even = {__builtin_amdgcn_perm(x[1], x[0], 0x05040100u), __builtin_amdgcn_perm(x[3], x[2], 0x05040100u)};
        const u32x2 odd = {__builtin_amdgcn_perm(x[1], x[0], 0x07060302u), __builtin_amdgcn_perm(x[3], x[2], 0x07060302u)};
        *reinterpret_cast<u32x2*>(to + (8 * w + 2 * kByte) * kNext) = even;
        *reinterpret_cast<u32x2*>(to + (8 * w + 2 * kByte + 1) * kNext) = odd;
      };
      pair(std::integral_constant<int, 0>());
      pair(std::integral_constant<int, 1>());
      if constexpr (D > 64) {
        pair(std::integral_constant<int, 2>());
        pair(std::integral_constant<int, 3>());
      }
    }
  };

  // Scores of the half step's tokens 16 i + 4 g + r in x[y][4 i + r].
  auto scores = [&](int step, int half, float (&x)[kSub][8]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      f32x4 s[kSub];
#pragma unroll
      for (int y = 0; y < kSub; ++y) s[y] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int a = 0; a < kKWords; ++a) {
        const bf16x8 key = *reinterpret_cast<const bf16x8*>(&kt[step & 1][32 * half + 16 * i + n][32 * a + 8 * g]);
#pragma unroll
        for (int t = 0; t < Terms<T>::kQ; ++t)
#pragma unroll
          for (int y = 0; y < kSub; ++y)
            s[y] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(key, __builtin_bit_cast(bf16x8, terms[y][a][t]), s[y], 0, 0, 0);
      }
#pragma unroll
      for (int y = 0; y < kSub; ++y)
#pragma unroll
        for (int r = 0; r < 4; ++r) x[y][4 * i + r] = s[y][r];
    }
  };
  // which of a half step's scores the row sees, as bits
  auto seen_of = [&](uint32_t valid, int t0, int y) {
    uint32_t seen = 0;
    const int at = pos[y];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int u = (j >> 2) * 16 + 4 * g + (j & 3), t = t0 + u;
      if constexpr (kTree) {
        const int away = distance(line[y], t);
        seen |= (uint32_t)((valid >> u & 1u) && away >= 0 && (q.window == 0 || away < q.window)) << j;
      } else {
        seen |= (uint32_t)((valid >> u & 1u) && t <= at && (q.window == 0 || t > at - q.window)) << j;
      }
    }
    return seen;
  };
  const float scale = kMode != kPlain ? 1.0f : curve[0].scale;
  // curve and mask, and the references moved where a score passes them
  auto settle = [&](float (&x)[kSub][8], uint32_t valid, int t0) {
    const bool masked = needs_mask(mine, valid, t0, q.window);
    if constexpr (kTree) {
#pragma unroll
      for (int y = 0; y < kSub; ++y) {
        if (masked)
          cap_scores(curve[y], x[y]), line_scores(curve[y], line[y], x[y], valid, 4 * g, t0 + 4 * g, q.window);
        else
          curve_scores(curve[y], x[y], pos[y], t0 + 4 * g);
      }
    } else {
      if (kMode == kCurved) {
#pragma unroll
        for (int y = 0; y < kSub; ++y) curve_scores(curve[y], x[y], pos[y], t0 + 4 * g);
      }
      if (masked) {
#pragma unroll
        for (int y = 0; y < kSub; ++y) {
          const uint32_t seen = seen_of(valid, t0, y);
#pragma unroll
          for (int j = 0; j < 8; ++j) x[y][j] = seen >> j & 1u ? x[y][j] : -__builtin_huge_valf();
        }
      }
    }
    float top[kSub];
    bool above = false;
#pragma unroll
    for (int y = 0; y < kSub; ++y) {
      top[y] = x[y][0];
#pragma unroll
      for (int j = 1; j < 8; ++j) top[y] = __builtin_fmaxf(top[y], x[y][j]);
      top[y] *= scale;
      above |= top[y] > m[y] + kSlack;
    }
    if (__ballot(above)) {
#pragma unroll
      for (int y = 0; y < kSub; ++y) {
        float t = __builtin_fmaxf(top[y], __shfl_xor(top[y], 16));
        t = __builtin_fmaxf(t, __shfl_xor(t, 32));
        const float next = __builtin_fmaxf(m[y], t), f = __builtin_amdgcn_exp2f(m[y] - next);
        m[y] = next;
        l[y] *= f;
#pragma unroll
        for (int j = 0; j < kTiles; ++j) acc[y][j] *= f;
      }
    }
  };
  auto weights = [&](float (&x)[kSub][8]) {
#pragma unroll
    for (int y = 0; y < kSub; ++y) {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[y][j] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[y][j], scale, -m[y]));
      l[y] += ((x[y][0] + x[y][1]) + (x[y][2] + x[y][3])) + ((x[y][4] + x[y][5]) + (x[y][6] + x[y][7]));
    }
  };
  auto gather = [&](int step, int half, float (&x)[kSub][8]) {
    u32x4 p[kSub][kP];
#pragma unroll
    for (int y = 0; y < kSub; ++y) split_terms(x[y], p[y]);
#pragma unroll
    for (int j = 0; j < kTiles; ++j) {
      const bf16x8 a = *reinterpret_cast<const bf16x8*>(&vt[step & 1][16 * j + n][32 * half + 8 * g]);
#pragma unroll
      for (int t = 0; t < kP; ++t)
#pragma unroll
        for (int y = 0; y < kSub; ++y)
          acc[y][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, __builtin_bit_cast(bf16x8, p[y][t]), acc[y][j], 0, 0, 0);
    }
  };
  // the blocks of values that were taken as tiny, for the rows that see them
  auto note_nan = [&](uint64_t valid, int t0) {
#pragma clang loop unroll(disable)
    for (int half = 0; half < 2; ++half) {
#pragma unroll
      for (int y = 0; y < kSub; ++y) {
        const uint32_t seen = seen_of((uint32_t)(valid >> (32 * half)), t0 + 32 * half, y);
#pragma clang loop unroll(disable)
        for (int j = 0; j < 8; ++j) {
          const int t = t0 + 32 * half + (j >> 2) * 16 + 4 * g + (j & 3);
          if (seen >> j & 1u) {
            const uint64_t at = c.plane_rows + kv4_row(c, kv4_page(c, b, (uint32_t)t), h, (uint32_t)t);
#pragma clang loop unroll(disable)
            for (int x = 0; x < kScales; ++x) bad[y] |= (uint32_t)(c.scales[at * kScales + x] == 255) << x;
          }
        }
      }
    }
  };

  // The second half's scores beside the first half's exponentials.
  auto work = [&](int step, uint64_t valid) {
    const int t0 = begin + step * kBlockStep;
    float x0[kSub][8], x1[kSub][8];
    scores(step, 0, x0);
    settle(x0, (uint32_t)valid, t0);
    scores(step, 1, x1);
    weights(x0);
    gather(step, 0, x0);
    settle(x1, (uint32_t)(valid >> 32), t0 + kStep);
    weights(x1);
    gather(step, 1, x1);
  };
  // Noted in the iteration before the step's store, read in the one of the store.
  auto noted = [&](int step, int what) { return notes[step & 1][what] == step; };
  if (steps > 0) {
    Pages next, later;  // of the step whose loads come next and of the one after
    pages_of(0, next);
    pages_of(1, later);
    uint64_t valid = load(0, next), valid_next;
    __syncthreads();
    note_scales(0);
    __syncthreads();
    bool nan = noted(0, 0);
    if (__ballot(noted(0, 1))) down = kDown;
    store_keys(0);
    store_values(0);
    next = later;
    valid_next = load(1, next);
    pages_of(2, next);
    note_scales(1);
    for (int step = 0; step < steps; ++step) {
      const int t0 = begin + step * kBlockStep;
      __syncthreads();
      const bool nan_next = noted(step + 1, 0), large = noted(step + 1, 1);
      store_keys(step + 1);
      const bool lower = down == 0 && __ballot(large);
      if (lower) down = kDown;
      store_values(step + 1);
      const uint64_t valid_later = load(step + 2, next);
      pages_of(step + 3, next);
      if (t0 < mine.hi && t0 + kBlockStep > mine.lo) {
        work(step, valid);
        if (nan) note_nan(valid, t0);
      }
      valid = valid_next, valid_next = valid_later, nan = nan_next;
      if (lower) {
#pragma unroll
        for (int y = 0; y < kSub; ++y)
#pragma unroll
          for (int j = 0; j < kTiles; ++j) acc[y][j] *= kDownFactor;
      }
      note_scales(step + 2);
    }
  }

#pragma unroll
  for (int y = 0; y < kSub; ++y) {
    l[y] += __shfl_xor(l[y], 16);
    l[y] += __shfl_xor(l[y], 32);
    bad[y] |= (uint32_t)__shfl_xor((int)bad[y], 16);
    bad[y] |= (uint32_t)__shfl_xor((int)bad[y], 32);
    if (row[y] >= rows.rows) continue;
    const float inv = l[y] == 0.0f ? 0.0f : 1.0f / l[y], up = down ? kUpFactor : 1.0f;
#pragma unroll
    for (int j = 0; j < kTiles; ++j)
      acc[y][j] = bad[y] >> (j / 2) & 1u ? acc[y][j] * __builtin_nanf("") : acc[y][j] * inv * up;
    if (plan.splits > 1) {
      float* o = ws + place.at * (kBlockRows * D + 2 * kBlockRows);
      const int r = row[y] - tile * kBlockRows;
#pragma unroll
      for (int j = 0; j < kTiles; ++j) *reinterpret_cast<f32x4*>(o + r * D + 16 * j + 4 * g) = acc[y][j];
      if (g == 0) o[kBlockRows * D + r] = m[y], o[kBlockRows * D + kBlockRows + r] = l[y];
      continue;
    }
    const int64_t at = (int64_t)(rows.first + row[y] / q.group) * q.heads + (int64_t)h * q.group + row[y] % q.group;
    if (g == 0) lse[at] = l[y] == 0.0f ? -__builtin_huge_valf() : (m[y] + __builtin_amdgcn_logf(l[y])) * kLn2;
#pragma unroll
    for (int j = 0; j < kTiles; ++j) put4(out, at * D + 16 * j + 4 * g, acc[y][j], T());
  }
}

// Splits of a row that one wave joins.
constexpr int kFewSplits = 16;

// The splits of one row joined, in their order: kShare waves of a workgroup a
// row, which take its splits in turn.  One where there are few splits, as for
// the many rows of a prompt: 20480 rows of 5 splits took 33 us with four.
template <int D, typename T, int kShare>
__global__ __launch_bounds__(256) void kv4_join_kernel(Kv4View c, Kv4Query q, Kv4Plan plan, void* out, float* lse,
                                                       const float* ws) {
  constexpr int kPer = D / 64;
  __shared__ float sum[kWaves][D];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t id = kShare == 1 ? blockIdx.x * kWaves + wave : blockIdx.x;
  const uint32_t slot = id / (uint32_t)plan.rows;
  uint32_t b = slot / (uint32_t)plan.tiles / c.kv, h = slot / (uint32_t)plan.tiles % c.kv;
  int tile = (int)(slot % (uint32_t)plan.tiles);
  if (plan.listed) {
    h = slot % c.kv;
    if (!listed_tile(c, q, plan, slot / c.kv, b, tile)) return;
  }
  if (b >= c.seqs) return;
  const int n = (int)(id % (uint32_t)plan.rows), r = tile * plan.rows + n;
  const int step = plan.rows == kRows ? kStep : kBlockStep;
  const TileRows rows = q.tree ? tile_rows<true>(c, q, b, tile, plan.rows, step) : tile_rows(c, q, b, tile, plan.rows, step);
  if (r >= rows.rows) return;
  const int splits = joined_splits(rows, plan);
  const int64_t size = (int64_t)plan.rows * (D + 2);
  const float* o_n = ws + (int64_t)slot * plan.splits * size + (int64_t)n * D;
  const float* m_n = ws + (int64_t)slot * plan.splits * size + (int64_t)plan.rows * D + n;
  // the first sums are on their way while the references are compared
  constexpr int kAhead = 4;
  const int first = kShare == 1 ? 0 : wave;
  float part[kAhead][kPer], part_m[kAhead], part_l[kAhead];
  auto fetch = [&](int s0) {
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      const int s = s0 + a * kShare < splits ? s0 + a * kShare : splits - 1;
      part_m[a] = m_n[s * size], part_l[a] = m_n[s * size + plan.rows];
#pragma unroll
      for (int k = 0; k < kPer; ++k) part[a][k] = o_n[s * size + lane * kPer + k];
    }
  };
  fetch(first);
  // where there are few, lanes a row of them apart take the same split
  constexpr int kLanes = kShare == 1 ? kFewSplits : 64;
  float m = kLowest, l = 0.0f;
  for (int s = lane & (kLanes - 1); s < splits; s += kLanes) {
    const float m1 = m_n[s * size], top = __builtin_fmaxf(m, m1);
    l = l * __builtin_amdgcn_exp2f(m - top) + m_n[s * size + plan.rows] * __builtin_amdgcn_exp2f(m1 - top);
    m = top;
  }
  const float mine = m;
  for (int d = 1; d < kLanes; d *= 2) m = __builtin_fmaxf(m, __shfl_xor(m, d));
  l *= __builtin_amdgcn_exp2f(mine - m);
  for (int d = 1; d < kLanes; d *= 2) l += __shfl_xor(l, d);
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  float o[kPer];
#pragma unroll
  for (int k = 0; k < kPer; ++k) o[k] = 0.0f;
  for (int s = first; s < splits; s += kAhead * kShare) {
    if (s > first) fetch(s);
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      if (s + a * kShare >= splits) break;
      const float f = part_l[a] * __builtin_amdgcn_exp2f(part_m[a] - m) * inv;  // a split's share
#pragma unroll
      for (int k = 0; k < kPer; ++k) o[k] += part[a][k] * f;
    }
  }
  if constexpr (kShare > 1) {
#pragma unroll
    for (int k = 0; k < kPer; ++k) sum[wave][lane * kPer + k] = o[k];
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int d = lane * kPer + k;
      o[k] = (sum[0][d] + sum[1][d]) + (sum[2][d] + sum[3][d]);
    }
  }
  const int64_t row = (int64_t)(rows.first + r / q.group) * q.heads + (int)h * q.group + r % q.group;
  if (lane == 0) lse[row] = l == 0.0f ? -__builtin_huge_valf() : (m + __builtin_amdgcn_logf(l)) * kLn2;
#pragma unroll
  for (int k = 0; k < kPer; ++k) put(out, row * D + lane * kPer + k, o[k], T());
}

// Tokens of a wave that weighs.
constexpr int weigh_tokens(int dim) { return dim == 256 ? 32 : 64; }
// Bytes of a tile's queries and statistics in LDS.
constexpr int weigh_tile(int dim, int q_terms) { return kRows * (q_terms * (dim + 8) * 2 + 4); }

// The attention weights of every row added to its kv head's tokens.  A wave
// owns 64 tokens (32 of a head of 256), holds their keys as bf16 and walks over
// all rows, so that a token's sum has one order and one writer; the rows'
// statistics are known (lse), so the values are not read.  The rows' terms lie
// in LDS, as many tiles at a time as fit, for the four waves (read tile by tile
// from memory, 260 rows over 16385 tokens took 64 us).  One tile of rows is
// bound by the reading of the keys (8 sequences of 2000: 8 us, its own latency),
// many by vector instructions (260 rows over 16385 tokens, 16 heads: 44 us).
template <int D, typename T, bool kExtra>
__global__ __launch_bounds__(256) void kv4_weigh_kernel(Kv4View c, Kv4Query q, int most_tiles, const float* lse,
                                                        float* weights, int64_t weights_len) {
  constexpr int kRow = D / 2, kScales = D / 32, kWords = D / 32;
  constexpr int kParts = weigh_tokens(D) / 16;
  constexpr int kQ = Terms<T>::kQ;
  struct Tile {  // rows a 16-byte bank group off each other's
    uint16_t q[kRows][kQ][D + 8];
    float lse[kRows];
  };
  extern __shared__ __align__(16) uint8_t shared[];
  Tile* held = reinterpret_cast<Tile*>(shared);  // [most_tiles]
  static_assert(sizeof(Tile) == weigh_tile(D, kQ), "");
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t heads = c.seqs * c.kv, chunk = blockIdx.x / heads;
  const uint32_t slot = (blockIdx.x + (c.kv % 8 ? chunk : 0u)) % heads;
  const uint32_t b = slot / c.kv, h = slot % c.kv;
  const TileRows all = tile_rows(c, q, b, 0, 0x40000000, kStep);
  const int end = all.hi < weights_len ? all.hi : (int)weights_len;
  const int w0 = all.lo + (int)chunk * kWaves * weigh_tokens(D);
  if (w0 >= end) return;
  const int t0 = w0 + wave * weigh_tokens(D);
  u32x4 key[kParts][kWords];
  uint64_t valid = 0;
  {
    uint32_t k[kParts][kWords], s[kParts][Loaded<D>::kGroups], page[kParts];
#pragma unroll
    for (int i = 0; i < kParts; ++i) {
      const int t = t0 + 16 * i + n;
      page[i] = kv4_page(c, b, (uint32_t)(t < end ? t : end - 1));
    }
#pragma unroll
    for (int i = 0; i < kParts; ++i) {
      const int t = t0 + 16 * i + n;
      const uint64_t row = kv4_row(c, page[i], h, (uint32_t)(t < end ? t : end - 1));
      valid |= (__ballot(t < end && page[i] < c.pages) & 0xFFFFull) << (16 * i);
      load_keys<D>(c.codes + row * kRow, c.scales + row * kScales, 0u, 0u, g, k[i], s[i]);
    }
#pragma unroll
    for (int i = 0; i < kParts; ++i)
#pragma unroll
      for (int a = 0; a < kWords; ++a) {
        const float f = u2f(s[i][a / 4] << 23);
        key[i][a] = u32x4{fp4_pair<0>(k[i][a], f), fp4_pair<1>(k[i][a], f), fp4_pair<2>(k[i][a], f), fp4_pair<3>(k[i][a], f)};
      }
  }
  float add[4 * kParts];
#pragma unroll
  for (int j = 0; j < 4 * kParts; ++j) add[j] = 0.0f;
  const int tokens = all.rows / q.group, tiles = (all.rows + kRows - 1) / kRows;
  // tiles from the first whose rows are not all before the workgroup's tokens
  const int skip = w0 > all.base ? (int)((uint32_t)(w0 - all.base) * (uint32_t)q.group / kRows) : 0;
  const int step_token = kRows / q.group, step_which = kRows % q.group;
  for (int first = skip; first < tiles; first += most_tiles) {
    const int batch = tiles - first < most_tiles ? tiles - first : most_tiles;
    if (first > skip) __syncthreads();
    // the terms of these rows: 8 elements of a row a thread, four rows' loads in
    // flight (one at a time, 260 rows over 16385 tokens took 61 us)
    constexpr int kAhead = 4, kEach = 256 / (D / 8);  // rows of a round of the threads
    const int e = tid % (D / 8) * 8;
    for (int i0 = tid / (D / 8); i0 < batch * kRows; i0 += kAhead * kEach) {
      u32x4 t[kAhead][kQ];
      float statistic[kAhead];
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        const int r = first * kRows + i0 + a * kEach, rc = r < all.rows ? r : all.rows - 1;
        const int64_t at = all.first + rc / q.group;
        const int head = (int)h * q.group + rc % q.group;
        load_query(q, at * q.sn + (int64_t)head * q.sh + e, true, T(), t[a]);
        statistic[a] = lse[at * q.heads + head];
      }
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        const int i = i0 + a * kEach;
        if (i >= batch * kRows) break;
#pragma unroll
        for (int k = 0; k < kQ; ++k) *reinterpret_cast<u32x4*>(&held[i / kRows].q[i % kRows][k][e]) = t[a][k];
        if (e == 0) held[i / kRows].lse[i % kRows] = statistic[a] * kLog2e;
      }
    }
    __syncthreads();
    if (t0 >= end) continue;
    // row n of a tile: its token and the head of its group, kept up by steps of
    // 16 rows (a division is some 25 instructions)
    int token = (first * kRows + n) / q.group, which = (first * kRows + n) % q.group;
#pragma clang loop unroll(disable)
    for (int tile = 0; tile < batch; ++tile) {
      const float base = held[tile].lse[n];
      const int pos = token < tokens ? all.base + token : -1;
      // the last tile may be a part of one; rows before the sequence's beginning
      // have negative places, so that a place does not tell
      const bool part = (first + tile + 1) * kRows > all.rows;
      const int pos_first = __builtin_amdgcn_readfirstlane(pos);
      const int pos_last = part ? all.base + tokens - 1 : __builtin_amdgcn_readlane(pos, 15);
      const Curve curve = curve_of(q, (int)h * q.group + which);
      token += step_token, which += step_which;
      if (which >= q.group) which -= q.group, ++token;
      // a window that has passed these tokens, or rows that have not come to them
      if (q.window && pos_first - q.window >= t0 + weigh_tokens(D) - 1) continue;
      if (pos_last < t0) continue;
      const bool masked = valid != (kParts == 4 ? ~0ull : 0xFFFFFFFFull) || t0 + weigh_tokens(D) - 1 > pos_first ||
                          (q.window && t0 <= pos_last - q.window) || part;
      float x[4 * kParts];
#pragma unroll
      for (int i = 0; i < kParts; ++i) {
        f32x4 acc = {0, 0, 0, 0};
#pragma unroll
        for (int a = 0; a < kWords; ++a)
#pragma unroll
          for (int t = 0; t < kQ; ++t)
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                __builtin_bit_cast(bf16x8, key[i][a]),
                *reinterpret_cast<const bf16x8*>(&held[tile].q[n][t][key_element<D>(a, g)]), acc, 0, 0, 0);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[4 * i + j] = acc[j];
      }
      if (kExtra) {
#pragma unroll
        for (int i = 0; i < kParts / 2; ++i)
          curve_scores(curve, *reinterpret_cast<float(*)[8]>(&x[8 * i]), pos, t0 + 32 * i + 4 * g);
      }
      const float scale = kExtra ? 1.0f : curve.scale;
#pragma unroll
      for (int j = 0; j < 4 * kParts; ++j) x[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[j], scale, -base));
      if (masked) {
#pragma unroll
        for (int j = 0; j < 4 * kParts; ++j) {
          const int u = (j >> 2) * 16 + 4 * g + (j & 3), t = t0 + u;
          const bool seen = (valid >> u & 1u) && t <= pos && (q.window == 0 || t > pos - q.window);
          x[j] = seen ? x[j] : 0.0f;
        }
      }
#pragma unroll
      for (int j = 0; j < 4 * kParts; ++j) add[j] += x[j];
    }
  }
  if (t0 >= end) return;
  float* w = weights + (int64_t)slot * weights_len + t0;
  // lane (n, g) of the 16 of a group keeps token (n / 4) 16 + 4 g + n % 4
  float sum = 0.0f;
#pragma unroll
  for (int j = 0; j < 4 * kParts; ++j) {
    float a = add[j];
    for (int d = 1; d < 16; d *= 2) a += __shfl_xor(a, d);
    sum = n == j ? a : sum;
  }
  const int u = (n >> 2) * 16 + 4 * g + (n & 3);
  if (n < 4 * kParts && (valid >> u & 1u)) w[u] += sum;
}

// When the kernel for many rows is taken.  Its workgroups have 4 or 8 times the
// rows and a time of their own of some 20 us with the join, so that they have to
// be full and to fill the card.  Full: in the mean a sequence has 128 rows, or
// the most that any has (bf16, heads of 128, with it and with the other: 32
// sequences of up to 4000 tokens, one with 512 new tokens and the others with
// one, 140 and 37 us; of up to 1000, 8 with 300 and 24 with one, 80 and 86).  To
// fill the card, either so many tiles of 16 rows by 32 tokens that its splits are
// long enough (twice as many where a workgroup has 64 rows): 256 new tokens of
// 2000 (32000 tiles) 43 and 27 us, 2 x 350 of 2000 (90112) 85 and 63, 512 of 4096
// (131072) 84 and 82, 2 x 700 of 1800 (162400) 88 and 89, 2 x 65 of 16385 (139264)
// 103 and 153, 2048 of 2048 (262144) 93 and 96; f16, heads of 256, 64 rows: 3000
// of 5000 with 4 heads over 1 (118500) 304 and 168, 2048 of 2048 288 and 463.
constexpr int64_t kManyTiles = 100000;
// Or a workgroup for every compute unit over few tokens, without splits: there
// the other kernel's time is that of its workgroups' beginnings.  bf16, heads of
// 128: 6 x 139 new tokens of 180, 8 heads each (432 workgroups), 22 and 31 us,
// 16 x 64 of 500 (256) 30 and 32, 1 x 512 of 512 (128) 28 and 16, 1 x 1000 of 1000
// (256, two splits) 64 and 33; of 256: 6 x 139 of 180 50 and 119.
constexpr int64_t kShortSpan = 2048;

// Tiles of all kv heads, each of which has all its splits.
int64_t slots_of(const Kv4View& c, const Kv4Plan& p) {
  return (int64_t)c.kv * (p.listed ? (int64_t)p.listed : (int64_t)p.tiles * c.seqs);
}

Kv4Plan kv4_plan(const Kv4View& c, int dim, const Kv4Query& q, int dtype) {
  Kv4Plan p;
  const int64_t all = (int64_t)q.most * q.group;
  // the most tokens that rows of `tokens` new ones can see
  auto span_of = [&](int64_t tokens) {
    const int64_t seen = (int64_t)q.window + tokens + kBlockStep;
    return q.window && seen < (int64_t)c.cap ? seen : (int64_t)c.cap;
  };
  // no more tiles of a kv head than these, of sequences with less than the most
  auto tiles_of = [&](int64_t rows) {
    const int64_t every = c.seqs * ((all + rows - 1) / rows);
    const int64_t there = (int64_t)q.tokens.n * q.group / rows + (q.tokens.n < (int64_t)c.seqs ? q.tokens.n : c.seqs);
    return q.tokens.cu && there < every ? there : every;
  };
  const int many = 64 * block_sub(dim, dtype == kBF16 ? 1 : (dtype == kF16 ? 2 : 3));
  const double steps = (double)c.kv * tiles_of(kRows) * (double)(span_of(q.most) / kStep);
  // new tokens of a tile of `rows`, all of a sequence's where any may see any
  auto tokens_of = [&](int64_t rows) { return q.tree ? (int64_t)q.most : rows / q.group + 2; };
  const int64_t blocks = c.kv * tiles_of(many), room = span_of(tokens_of(many));
  const bool full = (int64_t)q.tokens.n * q.group >= c.seqs * (all < 128 ? all : 128);
  const bool whole = room <= 8 * kBlockStep ? blocks >= num_cus() : room <= kShortSpan && blocks > num_cus();
  bool block = all > kRows && full && (whole || steps >= (many == 64 ? 2 : 1) * kManyTiles);
  // Drafted tokens are at most 64 of a sequence, whose last tile is often its only
  // one, and a tile of 128 rows costs what 7 or 8 of 16 do however few it has (heads
  // of 128, bf16, 8 kv heads, second kernel and first: 16 sequences of 8000 with 32
  // rows 105 and 56 us, of 4000 with 96 rows 81 and 66, 8 of 6000 with 192 110 and 95;
  // 20 of 5000, 16 kv heads with 40 rows 262 and 105): the second for those that fill
  // seven eighths of its tiles (12 of 5000 with 128 rows 85 and 81; 3 of 30000, 5 kv
  // heads with 120 rows 71 and 86, 32 of 3000 with 256 190 and 251, fp16 234 and 322).
  // Short ones aside not where it has 64 rows (fp32: 12 of 5000 with 128 rows 141 and
  // 113, 16 of 20000 with 256 963 and 989) nor with heads of 256 (16 of 9000 with 256
  // rows 869 and 799, fp16 1085 and 947).
  if (q.tree) {
    const bool filled = 8ll * q.tokens.n * q.group >= 7 * tiles_of(many) * many;
    block = filled && (whole || (many == 128 && dim <= 128 && steps >= kManyTiles));
  }
  p.rows = block ? many : kRows;
  p.tiles = (int32_t)((all + p.rows - 1) / p.rows);
  const int64_t there = tiles_of(p.rows);
  // where most tiles would have no rows (32 sequences of up to 4000 tokens, one
  // with 512 new tokens, heads of 128: 115 us with all tiles, 37 with those there are)
  p.listed = 2 * there <= (int64_t)c.seqs * p.tiles && there < 1 << 25 ? (int32_t)there : 0;
  const int64_t span = span_of(tokens_of(p.rows));
  // The tokens are cut as if every sequence filled its room, since the lengths are
  // not known here: with room for 131072, 16 sequences of 16000 take 111 us (55 with
  // room for 16000), 256 new tokens of 2000 104 (26).
  // Two workgroups for every compute unit, as many as are resident and no more,
  // and none with fewer than eight steps (of a wave, of the workgroup): one costs
  // some 5 us beside its tokens, a join 4 and its launch (4 a unit instead of 2:
  // 16 sequences of 4000 tokens 27 and 23 us, one of 131073 47 and 38; one of
  // 1000 tokens whole 10, in four splits 12)
  const int64_t heads = slots_of(c, p), want = heads > 0 && 2ll * num_cus() > heads ? 2ll * num_cus() / heads : 1;
  const int64_t least = p.rows == kRows ? 8 * kWaves * kStep : 8 * kBlockStep;
  int64_t chunk = (span + want - 1) / want;
  if (chunk < least) chunk = least;
  chunk = (chunk + kWaves * kStep - 1) / (kWaves * kStep) * (kWaves * kStep);
  p.chunk = (int32_t)chunk;
  p.splits = (int32_t)((span + chunk - 1) / chunk);
  if (p.splits < 1) p.splits = 1;
  // Where not every compute unit has just one workgroup, those of the longest
  // sequences begin first, all tiles of one together: trees of 16 sequences of up to
  // 4000, 24 new tokens, 60 us as sequences come and 49, 32 with 8 new tokens of up to
  // 2000 27 and 23; where all are as long it costs up to 3% (heads of 256 152 and 157).
  p.ranked = q.tree && !p.listed && c.seqs > 1 && c.seqs <= 64 && heads * p.splits > num_cus();
  return p;
}

}  // namespace

int64_t kv4_workspace(const Kv4View& c, int dim, const Kv4Query& q, int dtype) {
  if (q.tokens.n == 0 || c.seqs == 0 || q.most == 0) return 0;
  const Kv4Plan p = kv4_plan(c, dim, q, dtype);
  return p.splits > 1 ? slots_of(c, p) * p.splits * p.rows * (dim + 2) * 4 : 0;
}

#define VQX_KV4_DIMS(CALL, T)  \
  if (dim == 64)               \
    CALL(64, T);               \
  else if (dim == 128)         \
    CALL(128, T);              \
  else                         \
    CALL(256, T)
#define VQX_KV4_TYPES(CALL)    \
  if (dtype == kBF16) {        \
    VQX_KV4_DIMS(CALL, Bf16);  \
  } else if (dtype == kF16) {  \
    VQX_KV4_DIMS(CALL, F16);   \
  } else {                     \
    VQX_KV4_DIMS(CALL, float); \
  }

int kv4_attention(const Kv4View& c, int dim, const Kv4Query& q, int dtype, void* out, float* lse, float* ws,
                  hipStream_t st) {
  if (q.tokens.n == 0 || c.seqs == 0 || q.most == 0) return kOk;
  const Kv4Plan p = kv4_plan(c, dim, q, dtype);
  const bool curved = q.softcap != 0.0f || q.slopes;
  const bool whole = !c.table || c.size % (p.rows == kRows ? kStep : kBlockStep) == 0;
  const int64_t slots = slots_of(c, p);
  if (slots * (p.splits > p.rows ? p.splits : p.rows) >= 1ll << 31)
    return set_error(kErrUnsupported, "kv4_attention: %lld tiles of %d splits do not fit a launch", (long long)slots,
                     p.splits);
  const dim3 grid((unsigned)(slots * p.splits));
#define VQX_KV4_MODE(NAME, D, T, MODE)                                                                               \
  do {                                                                                                             \
    if (whole)                                                                                                     \
      hipLaunchKernelGGL((NAME<D, T, MODE, true>), grid, dim3(256), 0, st, c, q, p, out, lse, ws);                 \
    else                                                                                                           \
      hipLaunchKernelGGL((NAME<D, T, MODE, false>), grid, dim3(256), 0, st, c, q, p, out, lse, ws);                \
  } while (0)
#define VQX_KV4_LAUNCH(NAME, D, T)                                                                                   \
  do {                                                                                                             \
    if (q.tree)                                                                                                    \
      VQX_KV4_MODE(NAME, D, T, kTreed);                                                                            \
    else if (curved)                                                                                               \
      VQX_KV4_MODE(NAME, D, T, kCurved);                                                                           \
    else                                                                                                           \
      VQX_KV4_MODE(NAME, D, T, kPlain);                                                                            \
  } while (0)
#define VQX_KV4_ROWS(D, T)                                                                                         \
  do {                                                                                                             \
    if (p.rows == kRows)                                                                                           \
      VQX_KV4_LAUNCH(kv4_rows_kernel, D, T);                                                                       \
    else                                                                                                           \
      VQX_KV4_LAUNCH(kv4_block_kernel, D, T);                                                                      \
    if (p.splits > kFewSplits)                                                                                     \
      hipLaunchKernelGGL((kv4_join_kernel<D, T, kWaves>), dim3((unsigned)(slots * p.rows)), dim3(256), 0, st, c,   \
                         q, p, out, lse, ws);                                                                      \
    else if (p.splits > 1)                                                                                         \
      hipLaunchKernelGGL((kv4_join_kernel<D, T, 1>), dim3((unsigned)(slots * p.rows / kWaves)), dim3(256), 0, st,  \
                         c, q, p, out, lse, ws);                                                                   \
  } while (0)
  VQX_KV4_TYPES(VQX_KV4_ROWS)
#undef VQX_KV4_ROWS
#undef VQX_KV4_LAUNCH
#undef VQX_KV4_MODE
  return check_launch("kv4_attention");
}

int kv4_accumulate(const Kv4View& c, int dim, const Kv4Query& q, int dtype, const float* lse, float* weights,
                   int64_t weights_len, hipStream_t st) {
  if (q.tokens.n == 0 || c.seqs == 0 || q.most == 0) return kOk;
  int64_t span = c.cap;
  if (q.window && (int64_t)q.window + q.most + kStep < span) span = (int64_t)q.window + q.most + kStep;
  const int64_t heads = (int64_t)c.seqs * c.kv, tokens = kWaves * weigh_tokens(dim);
  const bool extra = q.softcap != 0.0f || q.slopes;
  const int64_t chunks = (span + tokens - 1) / tokens;
  if (chunks * heads >= 1ll << 31)
    return set_error(kErrUnsupported, "kv4_accumulate: %lld runs of tokens do not fit a launch", (long long)(chunks * heads));
  const dim3 grid((unsigned)(chunks * heads));
  // LDS for the rows that there are, as many as leave room for two workgroups more
  const int tile = weigh_tile(dim, dtype == kBF16 ? 1 : (dtype == kF16 ? 2 : 3));
  const int64_t tiles = ((int64_t)q.most * q.group + kRows - 1) / kRows;
  const int most = (int)(tiles < 48 * 1024 / tile ? tiles : 48 * 1024 / tile);
#define VQX_KV4_WEIGH(D, T)                                                                                          \
  do {                                                                                                               \
    if (extra)                                                                                                       \
      hipLaunchKernelGGL((kv4_weigh_kernel<D, T, true>), grid, dim3(256), most * tile, st, c, q, most,  \
                         lse, weights, weights_len);                                                                 \
    else                                                                                                             \
      hipLaunchKernelGGL((kv4_weigh_kernel<D, T, false>), grid, dim3(256), most * tile, st, c, q, most, \
                         lse, weights, weights_len);                                                                 \
  } while (0)
  VQX_KV4_TYPES(VQX_KV4_WEIGH)
#undef VQX_KV4_WEIGH
  return check_launch("kv4_accumulate");
}

}  // namespace vqx
