// The bookkeeping of a 4-bit cache's steps on the GPU: pages for new tokens, and
// which drafted tokens stay.
#include "vqx_kv4.h"

namespace vqx {
namespace {

// ---------------------------------------------------------------------------
// reserve: block table, offsets, positions and slots of the new tokens
// ---------------------------------------------------------------------------
constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kSlotsEach = 2;  // of a thread of the second launch

// The sum of the values of the threads before this one, and of all.
__device__ __forceinline__ int64_t scan_before(int64_t x, uint64_t* sums, int64_t& all) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint64_t upto = wave_scan((uint64_t)x);
  __syncthreads();  // the sums of the scan before have been read
  if (lane == 63) sums[wave] = upto;
  __syncthreads();
  static_assert(kWaves == 16, "");
  uint64_t sum = sums[lane & 15];
  sum += from_lane<0x111, 0xF>(sum);
  sum += from_lane<0x112, 0xF>(sum);
  sum += from_lane<0x114, 0xF>(sum);
  sum += from_lane<0x118, 0xF>(sum);
  all = (int64_t)lane_of(sum, 15);
  return (int64_t)((wave > 0 ? lane_of(sum, wave - 1) : 0) + upto) - x;
}

// The last sequence that begins at or before new token i; cu: offsets, in LDS or
// memory.
__device__ __forceinline__ int sequence_at(const int32_t* cu, int seqs, int64_t i) {
  int lo = 0, hi = seqs;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (cu[mid] <= i)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

__device__ __forceinline__ void fill_slot(const Kv4Pages& p, const int32_t* cu, int64_t i) {
  int32_t position = -1;
  int64_t slot = -1;
  if (i < cu[p.seqs]) {
    const int b = sequence_at(cu, p.seqs, i);
    position = p.lengths[b] - (cu[b + 1] - (int32_t)i);
    const int32_t page = p.table[(int64_t)b * p.per + position / p.size];
    slot = (int64_t)page * p.size + position % p.size;
  }
  p.positions[i] = position;
  p.slots[i] = slot;
}

// Entries of rows one after another, kChunks of them a thread, 1024 apart: which
// are marked and how many marked ones come before each.
constexpr int kChunks = 8, kGroup = kChunks * kThreads;
struct Entries {
  int row[kChunks];      // which of the rows
  int32_t* at[kChunks];  // NULL past the last
  int32_t page[kChunks];
  bool marked[kChunks];
  int32_t before[kChunks];
};

// All loads on their way together, and one barrier for all: a wave's marks are
// counted by a ballot, and each wave sums up the 128 counts itself.  Returns the
// number of marks.
// left: entries from the group's first on.
template <typename Mark>
__device__ __forceinline__ int mark_entries(Entries& e, int64_t left, int32_t (&counts)[kChunks * kWaves], Mark mark) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
  for (int k = 0; k < kChunks; ++k) e.page[k] = e.at[k] ? *e.at[k] : 0;
  __syncthreads();  // counts before have been read
#pragma unroll
  for (int k = 0; k < kChunks; ++k) {
    e.marked[k] = false;
    if (k * kThreads >= left) {
      if (lane == 0) counts[k * kWaves + wave] = 0;
      continue;
    }
    e.marked[k] = e.at[k] && mark(e.page[k]);
    const uint64_t bits = __ballot(e.marked[k]);
    e.before[k] = (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(bits >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)bits, 0));
    if (lane == 0) counts[k * kWaves + wave] = __popcll(bits);
  }
  __syncthreads();
  static_assert(kChunks * kWaves == 128, "");
  const int one = counts[2 * lane], two = counts[2 * lane + 1];
  const int upto = (int)wave_scan((uint64_t)(one + two));
#pragma unroll
  for (int k = 0; k < kChunks; ++k) {
    if (k * kThreads >= left) break;
    const int pair = (k * kWaves + wave) / 2;
    const int sum = __builtin_amdgcn_readlane(upto - one - two, pair);
    e.before[k] += wave & 1 ? sum + __builtin_amdgcn_readlane(one, pair) : sum;
  }
  return __builtin_amdgcn_readlane(upto, 63);
}

// One workgroup, a thread for each sequence: what they need depends on what
// those before them were given.  Entries of the table are read across the
// threads, in their order (a thread's own row takes a line for each lane): 512
// sequences, 51 of which end, 138 admitted with 1000 tokens in the mean, take 21.7
// us (30 with the rows of a thread each, 64 with an entry of them at a time), 16
// sequences with a token each 10.5.  Bound by its chains of loads and barriers.
__global__ __launch_bounds__(kThreads) void kv4_reserve_kernel(Kv4Pages p, bool slots) {
  __shared__ uint64_t sums[kWaves];
  __shared__ int32_t counts[kChunks * kWaves];
  __shared__ int64_t starts[kThreads + 1];             // of each sequence's entries
  __shared__ int32_t firsts[kThreads];                 // the first of them in its row
  __shared__ int64_t ranks[kThreads], ends[kThreads];  // lacking ones before the first and up to the last
  __shared__ bool serves[kThreads];
  const int tid = threadIdx.x;
  const int64_t cap = (int64_t)p.per * p.size;
  auto valid = [&](int32_t page) { return (uint32_t)page < (uint32_t)p.pages; };
  Entries e;
  int64_t stock = p.count[0];
  stock = stock < 0 ? 0 : (stock > p.pages ? p.pages : stock);
  // sequences that end give their pages back, in their order
  for (int b0 = 0; b0 < p.seqs; b0 += kThreads) {
    const int b = b0 + tid;
    const bool over = b < p.seqs && p.grow[b] < 0;
    int64_t rows;
    const int64_t at = scan_before(over, sums, rows);
    if (over) firsts[at] = b, p.lengths[b] = 0;
    __syncthreads();
    for (int64_t i0 = 0; i0 < rows * p.per; i0 += kGroup) {
#pragma unroll
      for (int k = 0; k < kChunks; ++k) {
        const int64_t n = i0 + k * kThreads + tid;
        e.at[k] = nullptr;
        if (i0 + k * kThreads >= rows * p.per) continue;
        // 32 bits, but for rows of millions
        e.row[k] = n >> 32 ? (int)(n / p.per) : (int)((uint32_t)n / (uint32_t)p.per);
        e.at[k] = n < rows * p.per ? p.table + (int64_t)firsts[e.row[k]] * p.per + (n - (int64_t)e.row[k] * p.per) : nullptr;
      }
      const int all = mark_entries(e, rows * p.per - i0, counts, valid);
#pragma unroll
      for (int k = 0; k < kChunks; ++k) {
        const int64_t to = stock + e.before[k];
        if (e.marked[k] && to < p.pages) p.free[to] = e.page[k];  // past it: one came back twice
        if (e.at[k]) *e.at[k] = -1;
      }
      stock += all;
    }
    __syncthreads();
  }
  if (stock > p.pages) stock = p.pages;
  // pages for those that grow
  int64_t needed = 0, tokens = 0, taken = 0, served_tokens = 0;
  for (int b0 = 0; b0 < p.seqs; b0 += kThreads) {
    const int b = b0 + tid;
    const bool there = b < p.seqs;
    const int32_t grow = there ? p.grow[b] : 0, length = there ? p.lengths[b] : 0;
    const int64_t wanted = grow > 0 ? grow : 0;
    const bool fits = there && length >= 0 && length + wanted <= cap;
    const int first = fits && wanted > 0 ? length / p.size : 0;
    const int last = fits && wanted > 0 ? (int)((length + wanted - 1) / p.size) + 1 : 0;
    // the entries of the new tokens of all of them, one after another
    int64_t entries;
    starts[tid] = scan_before(last - first, sums, entries);
    firsts[tid] = first, ranks[tid] = 0, ends[tid] = 0;
    if (tid == 0) starts[kThreads] = entries;
    __syncthreads();
    int most = kThreads;  // sequences of the tile, up to a power of two
    while (most / 2 >= p.seqs - b0) most /= 2;
    auto find = [&](int64_t i0) {
#pragma unroll
      for (int k = 0; k < kChunks; ++k) e.row[k] = 0;
      // the last that starts at or before each, all chunks' searches side by side
      for (int step = most / 2; step > 0; step /= 2)
#pragma unroll
        for (int k = 0; k < kChunks; ++k)
          if (i0 + k * kThreads < entries && starts[e.row[k] + step] <= i0 + k * kThreads + tid) e.row[k] += step;
#pragma unroll
      for (int k = 0; k < kChunks; ++k) {
        const int64_t n = i0 + k * kThreads + tid;
        e.at[k] = nullptr;
        if (i0 + k * kThreads >= entries) continue;
        e.at[k] = n < entries ? p.table + (int64_t)(b0 + e.row[k]) * p.per + firsts[e.row[k]] + (n - starts[e.row[k]]) : nullptr;
      }
    };
    auto lacking = [&](int32_t page) { return !valid(page); };
    int64_t found = 0;
    for (int64_t i0 = 0; i0 < entries; i0 += kGroup) {
      find(i0);
      const int all = mark_entries(e, entries - i0, counts, lacking);
#pragma unroll
      for (int k = 0; k < kChunks; ++k) {
        const int64_t n = i0 + k * kThreads + tid;
        if (!e.at[k]) continue;
        const int row = e.row[k];
        if (n == starts[row]) ranks[row] = found + e.before[k];
        if (n + 1 == starts[row + 1]) ends[row] = found + e.before[k] + e.marked[k];
      }
      found += all;
    }
    __syncthreads();
    const int64_t need = ends[tid] - ranks[tid], mine = needed + ranks[tid];
    int64_t all_tokens, all_served, all_taken;
    const int64_t upto = tokens + scan_before(fits ? wanted : 0, sums, all_tokens) + wanted;
    const bool served = fits && (need == 0 || mine + need <= stock) && upto <= p.n;
    const int64_t cu = served_tokens + scan_before(served ? wanted : 0, sums, all_served);
    scan_before(served ? need : 0, sums, all_taken);
    if (there) p.cu[b] = (int32_t)cu;
    if (served && wanted > 0) p.lengths[b] = length + (int32_t)wanted;
    serves[tid] = served;
    __syncthreads();
    int64_t rank = needed;
    for (int64_t i0 = 0; i0 < entries; i0 += kGroup) {
      int all = 0;
      if (entries > kGroup) find(i0), all = mark_entries(e, entries - i0, counts, lacking);  // one group's are still at hand
#pragma unroll
      for (int k = 0; k < kChunks; ++k)
        if (e.marked[k] && serves[e.row[k]]) e.page[k] = p.free[stock - 1 - rank - e.before[k]];
#pragma unroll
      for (int k = 0; k < kChunks; ++k)
        if (e.marked[k] && serves[e.row[k]]) *e.at[k] = e.page[k];
      rank += all;
    }
    __syncthreads();
    needed += found, tokens += all_tokens, served_tokens += all_served, taken += all_taken;
  }
  if (tid == 0) p.cu[p.seqs] = (int32_t)served_tokens, p.count[0] = (int32_t)(stock - taken);
  if (!slots) return;
  __syncthreads();
  for (int64_t i = tid; i < p.n; i += kThreads) fill_slot(p, p.cu, i);
}

// Offsets that a workgroup searches in LDS.
constexpr int kMostOffsets = 4096;

__global__ __launch_bounds__(256) void kv4_slots_kernel(Kv4Pages p) {
  __shared__ int32_t cu[kMostOffsets];
  const bool local = p.seqs < kMostOffsets;
  if (local)
    for (int b = threadIdx.x; b <= p.seqs; b += 256) cu[b] = p.cu[b];
  __syncthreads();
  const int64_t i0 = (int64_t)blockIdx.x * kSlotsEach * 256 + threadIdx.x;
#pragma unroll
  for (int a = 0; a < kSlotsEach; ++a)
    if (i0 + a * 256 < p.n) fill_slot(p, local ? cu : p.cu, i0 + a * 256);
}

// Slots that the first launch's one workgroup fills by itself.
constexpr int64_t kFewSlots = 4096;

// ---------------------------------------------------------------------------
// accept: the drafted tokens that were confirmed
// ---------------------------------------------------------------------------
constexpr int kTree = 64;  // new tokens of a sequence that are looked at

// A wave a sequence, a lane for each of its new tokens: the children of the last
// accepted one are a ballot.  Bound by its launch and a chain of loads (64
// sequences of 64: 4.2 us).
__global__ __launch_bounds__(256) void kv4_accept_kernel(Kv4Tokens q, int seqs, const int64_t* tree, const int64_t* drafts,
                                                         const int64_t* tokens, int32_t* lengths, int32_t* path,
                                                         int32_t* count, int64_t* next) {
  const int lane = threadIdx.x & 63, b = (int)blockIdx.x * 4 + (int)(threadIdx.x >> 6);
  if (b >= seqs) return;
  int first, all;
  kv4_span(q, (uint32_t)b, first, all);
  const int n = all < kTree ? all : kTree;
  const bool there = lane < n;
  const uint64_t mask = there ? (uint64_t)tree[first + lane] : 0;
  const int64_t draft = there ? drafts[first + lane] : 0, token = there ? tokens[first + lane] : 0;
  int at = 0, accepted = n > 0, mine = n > 0 && lane == 0 ? 0 : -1;
  while (n > 0) {
    const uint64_t line = (uint64_t)__shfl((long long)mask, at);
    const int64_t wanted = __shfl((long long)token, at);
    const uint64_t child = __ballot(there && lane > at && mask == (line | 1ull << lane) && draft == wanted);
    if (child == 0) break;
    at = __builtin_ctzll(child);
    if (lane == accepted) mine = at;
    ++accepted;
  }
  if (there) path[first + lane] = mine;
  for (int i = kTree + lane; i < all; i += 64) path[first + i] = -1;
  // tokens of no sequence
  if (b == 0)
    for (int i = lane; i < first; i += 64) path[i] = -1;
  if (b == seqs - 1)
    for (int i = first + all + lane; i < q.n; i += 64) path[i] = -1;
  const int64_t last = __shfl((long long)token, at);
  if (lane == 0) {
    count[b] = accepted;
    next[b] = n > 0 ? last : -1;
    lengths[b] -= all - accepted;
  }
}

// The accepted tokens of one head of one sequence moved to the front of the new
// ones.  All rows are read before any is written.  A chain of loads (offsets, path,
// pages, rows): 5.3 us for 64 sequences of 32 heads, 3.9 for 4 of 8.
template <int kDim>
__global__ __launch_bounds__(256) void kv4_pack_kernel(Kv4View c, Kv4Tokens q, const int32_t* path, const int32_t* count) {
  constexpr int kParts = kDim / 32, kUnits = 2 * kTree * kParts / 256;
  const uint32_t b = blockIdx.x / c.kv, h = blockIdx.x % c.kv;
  int first, all;
  kv4_span(q, b, first, all);
  const int n = count[b];
  const int64_t base = (int64_t)c.lengths[b] - n;  // the lengths are cut already
  u32x4 code[kUnits];
  uint8_t scale[kUnits];
  uint64_t to[kUnits];
  bool moves[kUnits];
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    const int unit = u * 256 + (int)threadIdx.x, part = unit % kParts, i = unit / kParts % kTree, plane = unit / kParts / kTree;
    const int from = i < n ? path[first + i] : i;
    const int64_t s = base + from, d = base + i;
    moves[u] = from != i && d >= 0 && d < (int64_t)c.cap;
    if (!moves[u]) continue;
    const uint32_t page = kv4_page(c, b, (uint32_t)d);
    moves[u] = page < c.pages;
    if (!moves[u]) continue;
    to[u] = ((uint64_t)plane * c.plane_rows + kv4_row(c, page, h, (uint32_t)d)) * kParts + part;
    // a token without a place reads as zeros
    code[u] = u32x4{0u, 0u, 0u, 0u}, scale[u] = 0;
    const uint32_t source = s >= 0 && s < (int64_t)c.cap ? kv4_page(c, b, (uint32_t)s) : 0xFFFFFFFFu;
    if (source < c.pages) {
      const uint64_t at = ((uint64_t)plane * c.plane_rows + kv4_row(c, source, h, (uint32_t)s)) * kParts + part;
      code[u] = reinterpret_cast<const u32x4*>(c.codes)[at], scale[u] = c.scales[at];
    }
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < kUnits; ++u)
    if (moves[u]) reinterpret_cast<u32x4*>(c.codes)[to[u]] = code[u], c.scales[to[u]] = scale[u];
}

}  // namespace

int kv4_reserve(const Kv4Pages& p, hipStream_t st) {
  const bool few = p.n <= kFewSlots;
  hipLaunchKernelGGL(kv4_reserve_kernel, dim3(1), dim3(kThreads), 0, st, p, few);
  if (!few) hipLaunchKernelGGL(kv4_slots_kernel, dim3((unsigned)((p.n + 256 * kSlotsEach - 1) / (256 * kSlotsEach))),
                               dim3(256), 0, st, p);
  return check_launch("kv4_reserve");
}

int kv4_accept(const Kv4View& c, int dim, const Kv4Tokens& q, const int64_t* tree, const int64_t* drafts,
               const int64_t* tokens, int32_t* path, int32_t* count, int64_t* next, hipStream_t st) {
  if (c.seqs == 0) return kOk;
  hipLaunchKernelGGL(kv4_accept_kernel, dim3((c.seqs + 3) / 4), dim3(256), 0, st, q, (int)c.seqs, tree, drafts, tokens,
                     const_cast<int32_t*>(c.lengths), path, count, next);
  const int rc = check_launch("kv4_accept");
  if (rc != kOk || q.n == 0) return rc;
  const dim3 grid(c.seqs * c.kv);
  if (dim == 64)
    hipLaunchKernelGGL((kv4_pack_kernel<64>), grid, dim3(256), 0, st, c, q, path, count);
  else if (dim == 128)
    hipLaunchKernelGGL((kv4_pack_kernel<128>), grid, dim3(256), 0, st, c, q, path, count);
  else
    hipLaunchKernelGGL((kv4_pack_kernel<256>), grid, dim3(256), 0, st, c, q, path, count);
  return check_launch("kv4_accept (move)");
}

}  // namespace vqx
