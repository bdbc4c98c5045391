// The bookkeeping of a 4-bit cache's steps on the GPU: pages for new tokens, and
// which drafted tokens stay.
#include "vqx_kv4.h"

namespace vqx {
namespace {

// ---------------------------------------------------------------------------
// reserve: block table, offsets, positions and slots of the new tokens
// ---------------------------------------------------------------------------
constexpr int kThreads = 1024, kWaves = kThreads / 64;

// The sum of the values of the threads before this one, and of all.
__device__ __forceinline__ int64_t scan_before(int64_t x, int64_t* sums, int64_t& all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t sum = x;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int64_t y = __shfl_up(sum, d);
    if (lane >= d) sum += y;
  }
  __syncthreads();  // the sums of the scan before have been read
  if (lane == 63) sums[wave] = sum;
  __syncthreads();
  int64_t before = 0;
  all = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    before += w < wave ? sums[w] : 0;
    all += sums[w];
  }
  return before + sum - x;
}

__device__ __forceinline__ void fill_slots(const Kv4Pages& p, int64_t i) {
  int32_t position = -1;
  int64_t slot = -1;
  if (i < p.cu[p.seqs]) {
    int lo = 0, hi = p.seqs;  // the last sequence that begins at or before i
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (p.cu[mid] <= i)
        lo = mid;
      else
        hi = mid;
    }
    position = p.lengths[lo] - (p.cu[lo + 1] - (int32_t)i);
    const int32_t page = p.table[(int64_t)lo * p.per + position / p.size];
    slot = (int64_t)page * p.size + position % p.size;
  }
  p.positions[i] = position;
  p.slots[i] = slot;
}

// One workgroup, a thread for each sequence: what they need depends on what
// those before them were given.  Bound by the chains of loads.
__global__ __launch_bounds__(kThreads) void kv4_reserve_kernel(Kv4Pages p, bool slots) {
  __shared__ int64_t sums[kWaves];
  const int tid = threadIdx.x, lane = tid & 63;
  const int64_t cap = (int64_t)p.per * p.size;
  auto valid = [&](int32_t page) { return (uint32_t)page < (uint32_t)p.pages; };
  int64_t stock = p.count[0];
  stock = stock < 0 ? 0 : (stock > p.pages ? p.pages : stock);
  // sequences that end give their pages back, in their order, a wave to a row
  for (int b0 = 0; b0 < p.seqs; b0 += kThreads) {
    const int b = b0 + tid;
    const bool ends = b < p.seqs && p.grow[b] < 0;
    const uint64_t ending = __ballot(ends);
    int64_t given = 0;
    for (uint64_t left = ending; left; left &= left - 1) {
      const int l = __builtin_ctzll(left);
      const int32_t* row = p.table + (int64_t)(b - lane + l) * p.per;
      int n = 0;
      for (int j = lane; j - lane < p.per; j += 64) n += __popcll(__ballot(j < p.per && valid(row[j < p.per ? j : 0])));
      if (lane == l) given = n;
    }
    int64_t all;
    const int64_t before = scan_before(given, sums, all);
    for (uint64_t left = ending; left; left &= left - 1) {
      const int l = __builtin_ctzll(left);
      int32_t* row = p.table + (int64_t)(b - lane + l) * p.per;
      int64_t to = stock + __shfl(before, l);
      for (int j = lane; j - lane < p.per; j += 64) {
        const int32_t page = j < p.per ? row[j] : -1;
        const bool some = j < p.per && valid(page);
        const uint64_t mask = __ballot(some);
        const int64_t at = to + __popcll(mask & ((1ull << lane) - 1));
        if (some && at < p.pages) p.free[at] = page;  // more pages than there are: one came back twice
        if (j < p.per) row[j] = -1;
        to += __popcll(mask);
      }
    }
    if (ends) p.lengths[b] = 0;
    stock += all;
  }
  if (stock > p.pages) stock = p.pages;
  __syncthreads();
  // pages for those that grow
  int64_t needed = 0, tokens = 0, taken = 0, served_tokens = 0;
  for (int b0 = 0; b0 < p.seqs; b0 += kThreads) {
    const int b = b0 + tid;
    const bool there = b < p.seqs;
    const int32_t grow = there ? p.grow[b] : 0, length = there ? p.lengths[b] : 0;
    const int64_t wanted = grow > 0 ? grow : 0;
    const bool fits = there && length >= 0 && length + wanted <= cap;
    int32_t* row = p.table + (int64_t)(there ? b : 0) * p.per;
    const int first = fits && wanted > 0 ? length / p.size : 0;
    const int last = fits && wanted > 0 ? (int)((length + wanted - 1) / p.size) + 1 : 0;
    int64_t need = 0;
    for (int j = first; j < last; ++j) need += !valid(row[j]);
    int64_t all_need, all_tokens, all_served, all_taken;
    const int64_t mine = needed + scan_before(need, sums, all_need);
    const int64_t upto = tokens + scan_before(fits ? wanted : 0, sums, all_tokens) + wanted;
    const bool served = fits && (need == 0 || mine + need <= stock) && upto <= p.n;
    const int64_t cu = served_tokens + scan_before(served ? wanted : 0, sums, all_served);
    scan_before(served ? need : 0, sums, all_taken);
    if (there) p.cu[b] = (int32_t)cu;
    if (served && wanted > 0) {
      int64_t at = stock - 1 - mine;
      for (int j = first; j < last; ++j)
        if (!valid(row[j])) row[j] = p.free[at--];
      p.lengths[b] = length + (int32_t)wanted;
    }
    needed += all_need, tokens += all_tokens, served_tokens += all_served, taken += all_taken;
  }
  if (tid == 0) p.cu[p.seqs] = (int32_t)served_tokens, p.count[0] = (int32_t)(stock - taken);
  if (!slots) return;
  __syncthreads();
  for (int64_t i = tid; i < p.n; i += kThreads) fill_slots(p, i);
}

__global__ __launch_bounds__(256) void kv4_slots_kernel(Kv4Pages p) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < p.n) fill_slots(p, i);
}

// Slots that the first launch's one workgroup fills by itself.
constexpr int64_t kFewSlots = 4096;

// ---------------------------------------------------------------------------
// accept: the drafted tokens that were confirmed
// ---------------------------------------------------------------------------
constexpr int kTree = 64;  // new tokens of a sequence that are looked at

// A wave a sequence, a lane for each of its new tokens.
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
// ones.  All rows are read before any is written.
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
  if (!few) hipLaunchKernelGGL(kv4_slots_kernel, dim3((unsigned)((p.n + 255) / 256)), dim3(256), 0, st, p);
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
