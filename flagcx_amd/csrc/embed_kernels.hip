// embed_kernels.hip - rows of a table by token id, and the table's gradient.
//
// Lookup: out[t] = scale * table[ids[t] - first], zeros where the shard has no such row.  A
// gather of whole rows: memory bounds it, and every row is read and written in pieces of
// 16 bytes a lane.
//
// Gradient: G[v] = scale * sum of grad[t] over the tokens of row v.  A scatter with atomics
// would move fp32 read-modify-writes for every element and sum in an order that changes
// from run to run, so the tokens are sorted by row first (a stable radix sort of 32-bit
// keys: 8 us in one launch, 26 to 35 in the four of some ten thousand tokens, 11 to 35 % of a
// gradient) and the sums become a stream over grad: a wavefront takes a
// chunk of consecutive sorted tokens and one slice of the columns, keeps the running sum
// in registers and writes a row when its last token is behind it.  A row whose tokens lie
// in several chunks leaves one fp32 partial sum in each, and a last kernel adds those in
// order: the work of one chunk is the same however often an id occurs.
//
// Compiled once per pair of types: -DFLAGCX_TABLE=<enum> -DFLAGCX_OUT=<enum>; the pair of
// fp32 and fp32 also holds what does not depend on types.
#include "launch.h"
#include "residual.h"
#include "residual_device.h"

namespace flagcx_amd {

// Row of the shard that token t names; `vocab` if the shard has none.
static __device__ __forceinline__ uint64_t rowOf(const void *ids, bool wide, uint64_t t, int64_t first, uint64_t vocab) {
  const int64_t id = wide ? ((const int64_t *)ids)[t] : (int64_t)((const int32_t *)ids)[t];
  const uint64_t row = (uint64_t)id - (uint64_t)first;
  return id >= first && row < vocab ? row : vocab;
}

namespace { // per unit: the same names stand for other types in the next one

#if FLAGCX_TABLE == 6
typedef h16 Tab;
#elif FLAGCX_TABLE == 7
typedef float Tab;
#else
typedef b16 Tab;
#endif
#if FLAGCX_OUT == 6
typedef h16 Out;
#elif FLAGCX_OUT == 7
typedef float Out;
#else
typedef b16 Out;
#endif
constexpr int kVec = 16 / (int)(sizeof(Tab) > sizeof(Out) ? sizeof(Tab) : sizeof(Out)); // 16 bytes of the wider type

// ------------------------------------------------------------------ lookup

constexpr unsigned kMaxGrid = 1u << 20;

// A wavefront takes one slice of the columns, R runs a lane, of T tokens, all in flight
// together.  Workgroups that follow one another take the slices in turn and land on the XCDs in
// turn, so an XCD mostly reads the same columns, and rows that many tokens name pass through
// fewer of the eight L2s.  A batch of 65536 tokens over an fp32 table of 131072 x 4096, ids
// falling off as words do, bf16 out: whole rows to a workgroup 175 us with 730 MB read behind
// L2; slices of one run and eight tokens 181 us with 517 MB (pieces of 512 bytes write badly);
// four runs and two tokens 168 us, 6.3 TB/s behind L2.
constexpr uint32_t kLookupWaves = 4;
template <int V, int R, int T>
__global__ void __launch_bounds__(64 * kLookupWaves) embeddingKernel(EmbedCall p, uint32_t slices) {
  constexpr uint32_t kSlice = 64 * V * R;
  const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint64_t at = (uint64_t)(blockIdx.x % slices) * kSlice;
  const uint32_t n = p.dim - at < kSlice ? (uint32_t)(p.dim - at) : kSlice;
  const uint64_t step = (uint64_t)(gridDim.x / slices) * kLookupWaves * T;
  for (uint64_t t0 = ((uint64_t)(blockIdx.x / slices) * kLookupWaves + wave) * T; t0 < p.tokens; t0 += step) {
    const uint64_t mine = lane < T && t0 + lane < p.tokens ? rowOf(p.ids, p.wideIds != 0, t0 + lane, p.first, p.vocab) : p.vocab;
    Run<Tab, V> x[T][R];
    bool here[T];
#pragma unroll
    for (int t = 0; t < T; t++) {
      const uint64_t row = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(mine >> 32), t) << 32 |
                           (uint32_t)__builtin_amdgcn_readlane((int)mine, t);
      here[t] = row < p.vocab; // else zeros are read
      const Row in((const Tab *)p.table + (here[t] ? row * p.tableStride + at : 0), here[t] ? n * (uint32_t)sizeof(Tab) : 0);
#pragma unroll
      for (int r = 0; r < R; r++) x[t][r].load(in, r * 64 * V, lane * V);
    }
#pragma unroll
    for (int t = 0; t < T; t++) {
      const bool live = t0 + t < p.tokens;
      const float scale = here[t] ? p.scale : 0.0f; // zeros stay +0, whatever the scale
      const Row out((Out *)p.out + (live ? (t0 + t) * p.outStride + at : 0), live ? n * (uint32_t)sizeof(Out) : 0);
#pragma unroll
      for (int r = 0; r < R; r++) {
        Run<Out, V> y;
#pragma unroll
        for (int i = 0; i < V; i++) y.set(i, scale * x[t][r].at(i));
        y.template store<(V > 1 ? kAuxStream : kAuxPlain)>(out, r * 64 * V, lane * V);
      }
    }
  }
}

template <int V, int R, int T>
int lookupWith(const EmbedCall &c, hipStream_t stream) {
  const uint64_t slices = (c.dim + 64 * V * R - 1) / (64 * V * R);
  const uint64_t groups = (c.tokens + kLookupWaves * T - 1) / (kLookupWaves * T);
  const uint64_t most = kMaxGrid / slices > 0 ? kMaxGrid / slices : 1;
  const dim3 grid((unsigned)((groups < most ? groups : most) * slices)), block(64 * kLookupWaves);
  embeddingKernel<V, R, T><<<grid, block, 0, stream>>>(c, (uint32_t)slices);
  return (int)hipGetLastError();
}

template <int V>
int lookupFor(const EmbedCall &c, hipStream_t stream) {
  // enough wavefronts to fill the chip with several runs each
  const bool many = c.tokens * ((c.dim + 64 * V - 1) / (64 * V)) >= 32768;
  // single elements: twice the runs (32768 of 50000 x 2049 bf16: 54 us against 61)
  return many ? lookupWith<V, V == 1 ? 8 : 4, 2>(c, stream) : lookupWith<V, 1, 1>(c, stream);
}

} // namespace

// -------------------------------------------------------- gradient: layout

// Workspace: keys and tokens of the sorted order (twice: a pass reads one and writes the
// other), a pass's digit counts, a flag for each row that a token names, and two partial
// rows per chunk.
struct GradPlan {
  uint32_t tokens, vocab;
  uint32_t passes, bits;  // digits of the keys 0 .. vocab
  uint32_t blocks, per;   // workgroups of a sorting pass and tokens each
  uint32_t chunk, chunks; // sorted tokens a wavefront sums
  uint32_t dimPad;        // floats between partial rows
  uint64_t bytes;
  uint64_t keyAt[2], tokAt[2], countAt, flagAt, partAt;
};
GradPlan gradPlan(uint64_t tokens, uint64_t vocab, uint64_t dim);
constexpr uint32_t kTinyTokens = 256; // at most so many tokens need no workspace: gradTinyKernel

// The rows of the table that no token names become zeros.  Which those are is told by the
// rows' flags, by the sorted keys or by the ids themselves, whichever there is by then.
struct ClearParams {
  char *table;
  uint64_t rowBytes, strideBytes;
  uint32_t elem;        // bytes
  uint32_t vocab, tokens;
  uint32_t rows;        // a workgroup looks after so many: see clearGroup
  const uint8_t *flags; // or NULL
  const uint32_t *key;  // or NULL
  const void *ids;
  int64_t first;
  int32_t wideIds;
};
constexpr uint32_t kClearRows = 64;
// Groups of 64 rows, smaller ones of a small table, so that every CU gets several.
static inline uint32_t clearGroup(uint64_t vocab) {
  uint32_t rows = kClearRows;
  while (rows > 16 && vocab / rows < 2048) rows /= 2;
  return rows;
}
static inline uint64_t clearGroups(const ClearParams &p) { return ((uint64_t)p.vocab + p.rows - 1) / p.rows; }

// Groups count from the table's end: where ids are numbered by how often they occur, that is
// where most of the rows to clear are, and what is cleared first is cleared next to the sort.
static __device__ __forceinline__ void clearRows(const ClearParams &p, uint64_t group) {
  __shared__ uint32_t named[kClearRows / 32];
  const uint64_t base = ((p.vocab + p.rows - 1) / p.rows - 1 - group) * p.rows;
  if (p.flags) {
    if (threadIdx.x < 64) {
      const uint64_t row = base + threadIdx.x, set = __ballot(row < p.vocab && p.flags[row < p.vocab ? row : 0] != 0); // 64 rows' flags, more than may be asked for
      if (threadIdx.x < 2) named[threadIdx.x] = (uint32_t)(set >> (32 * threadIdx.x));
    }
  } else {
    if (threadIdx.x < 2) named[threadIdx.x] = 0;
    __syncthreads();
#pragma unroll 8
    for (uint32_t i = threadIdx.x; i < p.tokens; i += blockDim.x) {
      const uint64_t row = (p.key ? (uint64_t)p.key[i] : rowOf(p.ids, p.wideIds != 0, i, p.first, p.vocab)) - base;
      if (row < p.rows) atomicOr(&named[row >> 5], 1u << (row & 31u));
    }
  }
  __syncthreads();
  const uint64_t skip = (uint64_t)named[1] << 32 | named[0];
  const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  for (uint32_t r = wave; r < p.rows && base + r < p.vocab; r += waves) {
    if ((skip >> r) & 1u) continue;
    char *row = p.table + (base + r) * p.strideBytes;
    // whole 16-byte vectors, and the elements before the first and after the last
    const uint64_t head = (-(uintptr_t)row & 15u) < p.rowBytes ? -(uintptr_t)row & 15u : p.rowBytes, body = (p.rowBytes - head) & ~15ull;
    constexpr uint32_t kStep = 4096;
    for (uint64_t at = 0; at < body; at += kStep) {
      const Row out(row + head + at, body - at < kStep ? (uint32_t)(body - at) : kStep);
      const Run<float, 4> zero = {{0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
      for (int u = 0; u < 4; u++) zero.store<kAuxStream>(out, u * 256, lane * 4);
    }
    if (body == p.rowBytes) continue;
    const Row first(row, (uint32_t)head), last(row + head + body, (uint32_t)(p.rowBytes - head - body));
    if (p.elem == 4) {
      const Run<float, 1> zero = {{0.0f}};
      zero.store(first, 0, lane);
      zero.store(last, 0, lane);
    } else {
      const Run<h16, 1> zero = {{(h16)0.0f}};
      zero.store(first, 0, lane);
      zero.store(last, 0, lane);
    }
  }
}

// Sorts c's tokens by row.  Where `clear` is given, launches of the sort also clear rows, as many as
// fill the time that a launch takes anyway; returns in *cleared how many groups of rows that were.
int launchSort(const EmbedGradCall &c, const GradPlan &g, const ClearParams *clear, uint64_t *cleared, hipStream_t stream);

#if FLAGCX_TABLE == 7 && FLAGCX_OUT == 7
// ---------------------------------------------------------- gradient: sort

constexpr uint32_t kSortThreads = 512, kSortWaves = kSortThreads / 64;
constexpr uint32_t kSortTile = 2048; // tokens of a workgroup while there are few
constexpr uint32_t kMaxBits = 11, kMaxBins = 1u << kMaxBits;
constexpr uint32_t kMaxBlocks = 256;
constexpr uint64_t kClearBytes = 32ull << 20; // rows that a launch of the sort clears next to it

GradPlan gradPlan(uint64_t tokens, uint64_t vocab, uint64_t dim) {
  GradPlan g{};
  g.tokens = (uint32_t)tokens;
  g.vocab = (uint32_t)vocab;
  uint32_t bits = 1;
  while (bits < 32 && (vocab >> bits) != 0) bits++;
  g.passes = (bits + kMaxBits - 1) / kMaxBits;
  g.bits = (bits + g.passes - 1) / g.passes;
  uint64_t blocks = (tokens + kSortTile - 1) / kSortTile;
  if (blocks < 1) blocks = 1;
  if (blocks > kMaxBlocks) blocks = kMaxBlocks;
  g.per = (uint32_t)(((tokens + blocks - 1) / blocks + kSortThreads - 1) / kSortThreads * kSortThreads);
  if (g.per < kSortThreads) g.per = kSortThreads;
  g.blocks = (uint32_t)((tokens + g.per - 1) / g.per);
  if (g.blocks < 1) g.blocks = 1;
  // enough wavefronts to fill the chip before chunks grow
  const uint64_t slices = (dim + 511) / 512;
  g.chunk = 8;
  while (g.chunk < 32 && tokens * slices / g.chunk > 4096) g.chunk *= 2;
  g.chunks = (uint32_t)((tokens + g.chunk - 1) / g.chunk);
  g.dimPad = (uint32_t)((dim + 3) & ~3ull);
  uint64_t at = 0;
  auto take = [&at](uint64_t bytes) {
    const uint64_t here = at;
    at += (bytes + 255) & ~255ull;
    return here;
  };
  // What is taken is the most that any call with no more tokens, rows and columns needs, so that a
  // workspace of the largest serves them all; digits, workgroups and chunks have steps at which a larger
  // call needs less.  Digits of at most min(bits, kMaxBits) bits; one workgroup a tile at most.  Chunks
  // of fewer than 32 tokens, at least 8, are there only while tokens * slices / chunk <= 4096 (a whole
  // division), so their number times slices is below 4097 + slices.
  const uint64_t tiles = (tokens + kSortTile - 1) / kSortTile;
  const uint64_t large = (tokens + 31) / 32 * g.dimPad, small = (tokens + 7) / 8 * g.dimPad, few = 512 * (4097 + slices);
  const uint64_t most = small < few ? small : few;
  for (int i = 0; i < 2; i++) g.keyAt[i] = take(tokens * 4), g.tokAt[i] = take(tokens * 4);
  g.countAt = take((tiles < kMaxBlocks ? tiles : kMaxBlocks) * (4u << (bits < kMaxBits ? bits : kMaxBits)));
  g.flagAt = take(vocab);
  g.partAt = take((large > most ? large : most) * 2 * 4);
  g.bytes = at;
  return g;
}

uint64_t embedGradWorkspace(uint64_t tokens, uint64_t vocab, uint64_t dim) {
  return tokens <= kTinyTokens ? 0 : gradPlan(tokens, vocab, dim).bytes;
}

struct SortParams {
  const void *ids;
  int64_t first;
  int32_t wideIds;
  uint32_t tokens, vocab, per, blocks, bits;
  uint32_t *counts; // [block][digit]
  uint32_t *key[2], *tok[2];
  uint8_t *flags;   // or NULL: nobody asks which rows are named
  uint32_t pass, passEnd;
  ClearParams clear; // workgroups from number `blocks` on clear groups of rows from clearFrom on
  uint64_t clearFrom;
};

__device__ __forceinline__ uint32_t sortKey(const SortParams &p, uint32_t pass, uint32_t i) {
  return pass ? p.key[(pass + 1) & 1][i] : (uint32_t)rowOf(p.ids, p.wideIds != 0, i, p.first, p.vocab);
}

// Digit counts of one pass; the first also clears the rows' flags.
__global__ void __launch_bounds__(kSortThreads) sortCountKernel(SortParams p) {
  __shared__ uint32_t hist[kMaxBins];
  if (blockIdx.x >= p.blocks) return clearRows(p.clear, p.clearFrom + (blockIdx.x - p.blocks));
  const uint32_t bins = 1u << p.bits;
  for (uint32_t d = threadIdx.x; d < bins; d += kSortThreads) hist[d] = 0;
  if (p.pass == 0 && p.flags)
    for (uint64_t v = ((uint64_t)blockIdx.x * kSortThreads + threadIdx.x) * 16; v < p.vocab; v += (uint64_t)p.blocks * kSortThreads * 16)
      *(raw4 *)(p.flags + v) = raw4{0, 0, 0, 0}; // the flags' room is rounded up to 256 bytes
  __syncthreads();
  const uint32_t from = blockIdx.x * p.per, to = p.tokens - from < p.per ? p.tokens : from + p.per;
#pragma unroll 4
  for (uint32_t i = from + threadIdx.x; i < to; i += kSortThreads)
    atomicAdd(&hist[(sortKey(p, p.pass, i) >> (p.pass * p.bits)) & (bins - 1)], 1u);
  __syncthreads();
  for (uint32_t d = threadIdx.x; d < bins; d += kSortThreads) p.counts[blockIdx.x * bins + d] = hist[d];
}

// Stable passes, one per launch, or all of them where one workgroup holds the tokens.  A
// workgroup's place for a digit: the digits before it, the same digit in the workgroups
// before it, then its own wavefronts in order, each of which takes its tokens 64 at a time
// and ranks equal digits by lane.
__global__ void __launch_bounds__(kSortThreads) sortPassKernel(SortParams p) {
  __shared__ uint32_t place[kSortWaves][kMaxBins];
  __shared__ uint32_t waveTotal[kSortWaves];
  if (blockIdx.x >= p.blocks) return clearRows(p.clear, p.clearFrom + (blockIdx.x - p.blocks));
  constexpr uint32_t kMaxRun = kMaxBins / kSortThreads;
  constexpr uint32_t kAhead = 4; // rounds of 64 tokens whose keys are loaded together
  const uint32_t bins = 1u << p.bits;
  const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t from = blockIdx.x * p.per, to = p.tokens - from < p.per ? p.tokens : from + p.per;
  const uint32_t mine = p.per / kSortWaves; // tokens of a wavefront
  const uint32_t begin = from + wave * mine < to ? from + wave * mine : to, end = begin + mine < to ? begin + mine : to;
  for (uint32_t pass = p.pass; pass < p.passEnd; pass++) {
    const uint32_t shift = pass * p.bits;
    // the wavefront's first tokens, all of them while there are few, are read once
    uint32_t key[kAhead], token[kAhead];
    auto fetch = [&](uint32_t base) {
#pragma unroll
      for (uint32_t a = 0; a < kAhead; a++) {
        const uint32_t i = base + a * 64 + lane;
        key[a] = i < end ? sortKey(p, pass, i) : 0;
        token[a] = i < end ? (pass ? p.tok[(pass + 1) & 1][i] : i) : 0;
      }
    };
    fetch(begin);
    for (uint32_t w = 0; w < kSortWaves; w++)
      for (uint32_t d = threadIdx.x; d < bins; d += kSortThreads) place[w][d] = 0;
    // this thread's run of digits: how many before this workgroup, how many in all
    const uint32_t run = bins > kSortThreads ? bins / kSortThreads : 1, d0 = threadIdx.x * run;
    uint32_t before[kMaxRun], total[kMaxRun], sum = 0;
#pragma unroll
    for (uint32_t r = 0; r < kMaxRun; r++) {
      before[r] = total[r] = 0;
      if (p.blocks > 1 && r < run && d0 + r < bins) {
        const uint32_t *c = p.counts + d0 + r;
#pragma unroll 16
        for (uint32_t b = 0; b < p.blocks; b++) {
          const uint32_t n = c[(uint64_t)b * bins];
          if (b < blockIdx.x) before[r] += n;
          total[r] += n;
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (uint32_t a = 0; a < kAhead; a++)
      if (begin + a * 64 + lane < end) atomicAdd(&place[wave][(key[a] >> shift) & (bins - 1)], 1u);
#pragma unroll 4
    for (uint32_t i = begin + kAhead * 64 + lane; i < end; i += 64) atomicAdd(&place[wave][(sortKey(p, pass, i) >> shift) & (bins - 1)], 1u);
    __syncthreads();
#pragma unroll
    for (uint32_t r = 0; r < kMaxRun; r++)
      if (r < run && d0 + r < bins) {
        if (p.blocks == 1)
          for (uint32_t w = 0; w < kSortWaves; w++) total[r] += place[w][d0 + r];
        sum += total[r];
      }
    uint32_t scan = sum; // inclusive over the wavefront's lanes
    for (uint32_t s = 1; s < 64; s *= 2) {
      const uint32_t o = __shfl_up(scan, s);
      if (lane >= s) scan += o;
    }
    if (lane == 63) waveTotal[wave] = scan;
    __syncthreads();
    uint32_t at = scan - sum;
    for (uint32_t w = 0; w < wave; w++) at += waveTotal[w];
#pragma unroll
    for (uint32_t r = 0; r < kMaxRun; r++)
      if (r < run && d0 + r < bins) {
        uint32_t here = at + before[r];
        for (uint32_t w = 0; w < kSortWaves; w++) {
          const uint32_t n = place[w][d0 + r];
          place[w][d0 + r] = here;
          here += n;
        }
        at += total[r];
      }
    __syncthreads();
    volatile uint32_t *next = place[wave]; // this wavefront's alone from here on
    for (uint32_t base = begin; base < end; base += 64 * kAhead) {
      if (base != begin) fetch(base);
#pragma unroll
      for (uint32_t a = 0; a < kAhead; a++) {
        const bool live = base + a * 64 + lane < end;
        const uint32_t digit = (key[a] >> shift) & (bins - 1);
        uint64_t same = __ballot(live); // lanes with this lane's digit
        for (uint32_t b = 0; b < p.bits; b++) {
          const uint64_t set = __ballot((digit >> b) & 1u);
          same &= (digit >> b) & 1u ? set : ~set;
        }
        const uint32_t rank = (uint32_t)__popcll(same & ((1ull << lane) - 1ull));
        uint32_t out = 0;
        if (live) out = next[digit];
        __builtin_amdgcn_wave_barrier();
        if (live && rank == 0) next[digit] = out + (uint32_t)__popcll(same);
        __builtin_amdgcn_wave_barrier();
        if (live) {
          p.key[pass & 1][out + rank] = key[a];
          p.tok[pass & 1][out + rank] = token[a];
          if (pass == 0 && p.flags && key[a] < p.vocab) p.flags[key[a]] = 1; // whoever else writes, writes the same
        }
      }
    }
    __syncthreads(); // the next pass reads what this workgroup wrote
  }
}

int launchSort(const EmbedGradCall &c, const GradPlan &g, const ClearParams *clear, uint64_t *cleared, hipStream_t stream) {
  char *ws = (char *)c.workspace;
  SortParams p{};
  p.ids = c.ids;
  p.first = c.first;
  p.wideIds = c.wideIds;
  p.tokens = g.tokens;
  p.vocab = g.vocab;
  p.per = g.per;
  p.blocks = g.blocks;
  p.bits = g.bits;
  p.counts = (uint32_t *)(ws + g.countAt);
  for (int i = 0; i < 2; i++) {
    p.key[i] = (uint32_t *)(ws + g.keyAt[i]);
    p.tok[i] = (uint32_t *)(ws + g.tokAt[i]);
  }
  uint64_t share = 0, groups = 0;
  if (clear) {
    p.clear = *clear;
    p.flags = (uint8_t *)(ws + g.flagAt);
    groups = clearGroups(*clear);
    share = kClearBytes / (clear->rowBytes * clear->rows) + 1;
  }
  auto launch = [&](void (*kernel)(SortParams), bool flagged) {
    // without flags yet, a workgroup that clears reads all ids: only where they are few
    uint64_t n = 0;
    if (clear && (flagged || g.blocks == 1)) n = groups - *cleared < share ? groups - *cleared : share;
    p.clear.flags = flagged ? p.flags : nullptr;
    p.clearFrom = clear ? *cleared : 0;
    kernel<<<dim3(g.blocks + (unsigned)n), dim3(kSortThreads), 0, stream>>>(p);
    if (clear) *cleared += n;
    return (int)hipGetLastError();
  };
  if (g.blocks == 1) { // a few microseconds in one launch
    p.flags = nullptr;
    p.passEnd = g.passes;
    return launch(sortPassKernel, false);
  }
  for (uint32_t q = 0; q < g.passes; q++) {
    p.pass = q;
    p.passEnd = q + 1;
    int e = launch(sortCountKernel, q > 0);
    if (!e) e = launch(sortPassKernel, q > 0);
    if (e) return e;
  }
  return (int)hipSuccess;
}
#endif

// ---------------------------------------------------------- gradient: sums

namespace {

struct SumParams {
  const Out *grad;
  uint64_t gradStride;
  Tab *table;
  uint64_t tableStride;
  uint64_t dim;
  uint32_t slices;     // workgroups that share a chunk
  uint32_t base;       // first workgroup of this launch
  uint32_t sumBlocks;  // workgroups that sum chunks (join long rows), the others clear rows (join short ones)
  uint32_t waves;      // wavefronts of a workgroup that have columns
  uint32_t tokens, vocab, chunk, chunks, dimPad;
  float scale;
  const uint32_t *key, *tok;
  ClearParams clear;
  uint64_t clearFrom;  // first group of rows that is left to clear
  float *part; // [chunk][2][dimPad]: a row that began before the chunk, a row that ends after it
};

constexpr uint32_t kSumThreads = 256;
// runs a lane of a slice, and rows of grad that are loaded together: 8 KB of them a wavefront, or 4 rows next to old rows.
// Of single elements four runs: 16384 tokens added to 16384 x 4095 fp32 take 118 us so, 159 with one.
template <int V, bool ACC> constexpr int kSumRuns = V == 1 ? 4 : ACC ? 2 : 1;
template <int V, bool ACC> constexpr int kSumRows = V > 1 && ACC ? 4 : 8;
// old rows are read once, so is what comes of them; rows that are only written stay for whoever reads them next
// (accumulated shard of 16384 x 4096, 65536 tokens: 200 us against 208 with plain accesses; dense 284 against 289)
template <int V, bool ACC> constexpr int kSumStore = V > 1 && ACC ? kAuxStream : kAuxPlain;

template <int V, int R, int B, bool ACC>
__device__ __forceinline__ void sumChunk(const SumParams &p, uint32_t block) {
  constexpr uint32_t kSlice = 64 * V * R;
  const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (wave >= p.waves) return;
  const uint32_t c = block / p.slices, slice = (block % p.slices) * p.waves + wave;
  const uint64_t at = (uint64_t)slice * kSlice;
  if (at >= p.dim) return;
  const uint32_t n = p.dim - at < kSlice ? (uint32_t)(p.dim - at) : kSlice;
  const uint32_t from = c * p.chunk, count = p.tokens - from < p.chunk ? p.tokens - from : p.chunk;
  const uint32_t none = p.vocab; // the key of tokens that the shard has no row for, the last in order
  const uint32_t myKey = lane < count ? p.key[from + lane] : none;
  const uint32_t myTok = lane < count ? p.tok[from + lane] : 0;
  const uint32_t before = from ? p.key[from - 1] : ~0u, after = from + count < p.tokens ? p.key[from + count] : ~0u;
  const uint32_t firstKey = __builtin_amdgcn_readlane(myKey, 0);
  const bool began = before != firstKey; // the first row's first token is in this chunk
  float sum[R][V];
  auto restart = [&]() {
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
      for (int e = 0; e < V; e++) sum[r][e] = -0.0f; // -0 + x is x, bit for bit
  };
  restart();

  struct Batch {
    Run<Out, V> x[B][R];
    Run<Tab, V> old[ACC ? B : 1][R]; // of the rows that end here
  };
  auto keyAt = [&](uint32_t i) { return (uint32_t)__builtin_amdgcn_readlane(myKey, i); };
  auto nextKey = [&](uint32_t i) { return i + 1 < count ? keyAt(i + 1) : after; };
  auto load = [&](Batch &b, uint32_t i0) {
#pragma unroll
    for (int j = 0; j < B; j++) {
      const uint32_t i = i0 + j;
      const uint32_t k = i < count ? keyAt(i) : none, t = __builtin_amdgcn_readlane(myTok, i & 63u);
      const Row in(p.grad + (uint64_t)t * p.gradStride + at, k != none ? n * (uint32_t)sizeof(Out) : 0);
#pragma unroll
      for (int r = 0; r < R; r++) b.x[j][r].template load<kAuxStream>(in, r * 64 * V, lane * V);
      if constexpr (ACC) {
        const bool whole = k != none && k != nextKey(i) && (began || k != firstKey);
        const Row old(p.table + (whole ? (uint64_t)k * p.tableStride + at : 0), whole ? n * (uint32_t)sizeof(Tab) : 0);
#pragma unroll
        for (int r = 0; r < R; r++) b.old[j][r].template load<kAuxStream>(old, r * 64 * V, lane * V);
      }
    }
  };
  auto add = [&](Batch &b, uint32_t i0) {
#pragma unroll
    for (int j = 0; j < B; j++) {
      const uint32_t i = i0 + j;
      const uint32_t k = i < count ? keyAt(i) : none;
      if (k == none) return;
#pragma unroll
      for (int r = 0; r < R; r++)
#pragma unroll
        for (int e = 0; e < V; e++) sum[r][e] += b.x[j][r].at(e);
      const bool ends = k != nextKey(i);
      if (!ends && i + 1 < count) continue;
      const bool whole = ends && (began || k != firstKey);
      if (whole) {
        const Row out(p.table + (uint64_t)k * p.tableStride + at, n * (uint32_t)sizeof(Tab));
#pragma unroll
        for (int r = 0; r < R; r++) {
          Run<Tab, V> y;
#pragma unroll
          for (int e = 0; e < V; e++)
            y.set(e, ACC ? __builtin_fmaf(p.scale, sum[r][e], b.old[ACC ? j : 0][r].at(e)) : p.scale * sum[r][e]);
          y.template store<kSumStore<V, ACC>>(out, r * 64 * V, lane * V);
        }
      } else { // a row that began before the chunk goes to the first place, one that goes on to the second
        const uint32_t second = k == firstKey && !began ? 0 : 1;
        const Row out(p.part + ((uint64_t)c * 2 + second) * p.dimPad + at, n * 4u);
#pragma unroll
        for (int r = 0; r < R; r++) {
          Run<float, V> y;
#pragma unroll
          for (int e = 0; e < V; e++) y.v[e] = sum[r][e];
          y.store(out, r * 64 * V, lane * V);
        }
      }
      restart();
    }
  };
  Batch b0, b1; // one is added while the other arrives
  load(b0, 0);
  for (uint32_t i = 0; i < count; i += 2 * B) {
    if (i + B < count) load(b1, i + B);
    add(b0, i);
    if (i + 2 * B < count) load(b0, i + 2 * B);
    if (i + B < count) add(b1, i + B);
  }
}

// Chunks go out in the order of the table's rows: what is read and written at one time lies together
// (from the last row to the first: dense 291 us against 282, accumulated shard 209 against 199; first
// and last rows in turn: 296 and 202).
template <int V, bool ACC>
__global__ void __launch_bounds__(kSumThreads) gradSumKernel(SumParams p) {
  const uint32_t block = p.base + blockIdx.x;
  if (block < p.sumBlocks) sumChunk<V, kSumRuns<V, ACC>, kSumRows<V, ACC>, ACC>(p, block);
  else if constexpr (!ACC) clearRows(p.clear, p.clearFrom + (block - p.sumBlocks));
}

// Adds the partial sums of a row that spans chunks, in fp32 and in an order that follows from
// the keys.  A wavefront looks at one chunk in which such a row may begin, for 512 columns, and
// takes rows of up to kShort chunks.  A row of more, say a padding token's, is taken for 64
// columns by the workgroup that stands for the first multiple of kShort among its chunks, 16
// lanes to a partial row, so 16 of them at a time.
constexpr uint32_t kJoinWaves = 4;
constexpr uint32_t kShort = 64;
constexpr uint32_t kShortColumns = 512, kLongColumns = 64;

// the last chunk that begins with row `cur`, which goes on behind chunk c; `ahead` is the first key of chunk c + 1 + lane
__device__ __forceinline__ uint32_t lastChunkOf(const SumParams &p, uint32_t c, uint32_t cur, uint32_t ahead) {
  const uint64_t same = __ballot(c + 1 + (threadIdx.x & 63u) < p.chunks && ahead == cur);
  if (same != ~0ull) return c + (uint32_t)__builtin_ctzll(~same);
  uint32_t lo = c + 64, hi = p.chunks - 1;
  while (lo < hi) {
    const uint32_t mid = lo + (hi - lo + 1) / 2;
    if (p.key[mid * p.chunk] == cur) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// Four elements of a part of a row: one access where the table's rows are aligned, else four.
template <bool VEC>
struct Four {
  Run<Tab, VEC ? 4 : 1> v[VEC ? 1 : 4];
  __device__ __forceinline__ void load(const Row &row, uint32_t at) {
#pragma unroll
    for (int k = 0; k < (VEC ? 1 : 4); k++) v[k].load(row, k, at);
  }
  __device__ __forceinline__ void store(const Row &row, uint32_t at) const {
#pragma unroll
    for (int k = 0; k < (VEC ? 1 : 4); k++) v[k].store(row, k, at);
  }
  __device__ __forceinline__ float at(int k) const { return VEC ? v[0].at(VEC ? k : 0) : v[VEC ? 0 : k].at(0); }
  __device__ __forceinline__ void set(int k, float x) { v[VEC ? 0 : k].set(VEC ? k : 0, x); }
};

// sum[w] += partial rows i, i + step, ... of the chunks c .. last, elements at + 256 w .. + 3
template <int W>
__device__ __forceinline__ void addPartials(float4v (&sum)[W], const SumParams &p, uint32_t c, uint32_t last, uint32_t i, uint32_t step,
                                            uint64_t at) {
  constexpr uint32_t kAhead = 8; // partial rows in flight
  for (; i <= last; i += kAhead * step) {
    float4v x[kAhead][W];
#pragma unroll
    for (uint32_t a = 0; a < kAhead; a++) {
      const uint32_t j = i + a * step;
#pragma unroll
      for (int w = 0; w < W; w++) {
        x[a][w] = float4v{-0.0f, -0.0f, -0.0f, -0.0f}; // changes no sum
        if (j <= last && at + 256 * w < p.dimPad)
          x[a][w] = *(const float4v *)(p.part + ((uint64_t)j * 2 + (j == c ? 1 : 0)) * p.dimPad + at + 256 * w);
      }
    }
#pragma unroll
    for (uint32_t a = 0; a < kAhead; a++)
#pragma unroll
      for (int w = 0; w < W; w++) sum[w] += x[a][w];
  }
}

template <bool VEC, bool ACC>
__global__ void __launch_bounds__(64 * kJoinWaves) gradJoinKernel(SumParams p) {
  __shared__ float part[kJoinWaves][4][16][4];
  const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t block = p.base + blockIdx.x;
  if (block >= p.sumBlocks) {
    constexpr int W = kShortColumns / 256;
    const uint32_t unit = (block - p.sumBlocks) * kJoinWaves + wave, c = unit / p.slices;
    if (c + 1 >= p.chunks) return;
    const uint32_t edge = (c + 1) * p.chunk, look = c + 1 + lane;
    const uint32_t cur = p.key[edge - 1], next = p.key[edge], before = c ? p.key[c * p.chunk - 1] : ~0u;
    const uint32_t ahead = p.key[look < p.chunks ? look * p.chunk : 0];
    if (cur == p.vocab || next != cur || before == cur) return; // no row begins here and goes on
    const uint32_t last = lastChunkOf(p, c, cur, ahead);
    if (last - c > kShort) return;
    const uint64_t from = (uint64_t)(unit % p.slices) * kShortColumns;
    const uint32_t n = p.dim - from < kShortColumns ? (uint32_t)(p.dim - from) : kShortColumns;
    const Row out(p.table + (uint64_t)cur * p.tableStride + from, n * (uint32_t)sizeof(Tab));
    Four<VEC> y[W];
    if constexpr (ACC) {
#pragma unroll
      for (int w = 0; w < W; w++) y[w].load(out, w * 256 + lane * 4);
    }
    float4v sum[W];
#pragma unroll
    for (int w = 0; w < W; w++) sum[w] = float4v{-0.0f, -0.0f, -0.0f, -0.0f};
    addPartials<W>(sum, p, c, last, c, 1, from + lane * 4);
#pragma unroll
    for (int w = 0; w < W; w++) {
#pragma unroll
      for (int k = 0; k < 4; k++) y[w].set(k, ACC ? __builtin_fmaf(p.scale, sum[w][k], y[w].at(k)) : p.scale * sum[w][k]);
      y[w].store(out, w * 256 + lane * 4);
    }
    return;
  }
  const uint32_t slices = (uint32_t)((p.dim + kLongColumns - 1) / kLongColumns);
  const uint32_t mark = (block / slices + 1) * kShort; // a chunk that begins with the row
  const uint32_t cur = p.key[mark * p.chunk];
  if (cur == p.vocab || p.key[mark * p.chunk - 1] != cur) return;
  if (mark != kShort && p.key[(mark - kShort) * p.chunk] == cur && p.key[(mark - kShort) * p.chunk - 1] == cur)
    return; // an earlier mark's
  // the first of the kShort chunks before the mark that begins with the row; the row begins there or in the one before
  const uint64_t same = __ballot(p.key[(mark - kShort + lane) * p.chunk] == cur);
  const uint32_t begins = same ? mark - kShort + (uint32_t)__builtin_ctzll(same) : mark;
  const uint32_t c = begins == 0 ? 0 : p.key[begins * p.chunk - 1] == cur ? begins - 1 : begins;
  const uint32_t look = c + 1 + lane;
  const uint32_t last = lastChunkOf(p, c, cur, p.key[look < p.chunks ? look * p.chunk : 0]);
  if (last - c <= kShort) return;
  const uint64_t from = (uint64_t)(block % slices) * kLongColumns;
  const uint32_t quarter = lane >> 4, at = (lane & 15u) * 4;
  float4v sum[1] = {{-0.0f, -0.0f, -0.0f, -0.0f}};
  addPartials<1>(sum, p, c, last, c + wave * 4 + quarter, kJoinWaves * 4, from + at);
#pragma unroll
  for (int k = 0; k < 4; k++) part[wave][quarter][lane & 15u][k] = sum[0][k];
  __syncthreads();
  if (wave || quarter) return;
  for (uint32_t w = 0; w < kJoinWaves; w++)
    for (uint32_t q = 0; q < 4; q++)
      if (w || q) {
#pragma unroll
        for (int k = 0; k < 4; k++) sum[0][k] += part[w][q][lane][k];
      }
  const Row out(p.table + (uint64_t)cur * p.tableStride + from,
                (p.dim - from < kLongColumns ? (uint32_t)(p.dim - from) : kLongColumns) * (uint32_t)sizeof(Tab));
  Four<VEC> y;
  if constexpr (ACC) y.load(out, at);
#pragma unroll
  for (int k = 0; k < 4; k++) y.set(k, ACC ? __builtin_fmaf(p.scale, sum[0][k], y.at(k)) : p.scale * sum[0][k]);
  y.store(out, at);
}

// A batch of at most kTinyTokens tokens in one launch and without a workspace: the workgroup of a
// slice of columns ranks the tokens itself, its wavefronts sum kTinyChunk sorted tokens each, and
// partial sums meet in LDS.  Other workgroups clear rows.  128 / 256 tokens added to an fp32 shard of
// 16384 x 4096 take 13 / 16 us a call so, 257 with the launches above 20; with 512 tokens, the ranks
// grow with their square, it would be 31 against 20.
constexpr uint32_t kTinyWaves = 16, kTinyChunk = kTinyTokens / kTinyWaves;
static_assert(kTinyTokens * 4 == 64 * kTinyWaves && kTinyChunk < 64, "four lanes a token; a chunk's keys are lanes");
template <int V, bool ACC>
__global__ void __launch_bounds__(64 * kTinyWaves) gradTinyKernel(SumParams p) {
  __shared__ __attribute__((aligned(16))) uint32_t key[kTinyTokens];
  __shared__ uint32_t sortedKey[kTinyTokens], sortedTok[kTinyTokens];
  __shared__ float part[kTinyWaves][2][64][V];
  const uint32_t block = p.base + blockIdx.x;
  if (block >= p.sumBlocks) {
    if constexpr (!ACC) clearRows(p.clear, block - p.sumBlocks);
    return;
  }
  const uint32_t t = threadIdx.x, lane = t & 63u, wave = __builtin_amdgcn_readfirstlane(t >> 6), none = p.vocab;
  if (t < kTinyTokens) key[t] = t < p.tokens ? (uint32_t)rowOf(p.clear.ids, p.clear.wideIds != 0, t, p.clear.first, p.vocab) : none;
  __syncthreads();
  { // four lanes count the tokens before one, four keys at a time; keys of no token are behind all others
    const uint32_t me = t >> 2, mine = key[me];
    uint32_t before = 0;
#pragma unroll
    for (uint32_t i = 0; i < kTinyTokens / 16; i++) {
      const uint32_t j = (i * 4 + (t & 3u)) * 4;
      const raw4 other = *(const raw4 *)&key[j];
#pragma unroll
      for (uint32_t q = 0; q < 4; q++) before += other[q] < mine || (other[q] == mine && j + q < me) ? 1u : 0u;
    }
    before += __builtin_amdgcn_update_dpp(0, before, 0xB1, 0xf, 0xf, true); // the neighbour's
    before += __builtin_amdgcn_update_dpp(0, before, 0x4E, 0xf, 0xf, true); // the other pair's
    if ((t & 3u) == 0 && me < p.tokens) {
      sortedKey[before] = mine;
      sortedTok[before] = me;
    }
  }
  __syncthreads();
  const uint32_t from = wave * kTinyChunk;
  const uint32_t count = from >= p.tokens ? 0 : p.tokens - from < kTinyChunk ? p.tokens - from : kTinyChunk;
  const uint64_t at = (uint64_t)block * 64 * V;
  const uint32_t n = p.dim - at < 64 * V ? (uint32_t)(p.dim - at) : 64 * V;
  const uint32_t myKey = lane < count ? sortedKey[from + lane] : none, myTok = lane < count ? sortedTok[from + lane] : 0;
  const uint32_t beforeKey = __builtin_amdgcn_readfirstlane(count && from ? sortedKey[from - 1] : ~0u);
  const uint32_t after = __builtin_amdgcn_readfirstlane(from + count < p.tokens && count ? sortedKey[from + count] : ~0u);
  const uint32_t firstKey = __builtin_amdgcn_readlane(myKey, 0), lastKey = __builtin_amdgcn_readlane(myKey, count ? count - 1 : 0);
  const bool began = beforeKey != firstKey;
  // a row that begins in this chunk and goes on in the next is this wavefront's to finish
  const bool join = count && lastKey != none && after == lastKey && (lastKey != firstKey || began);
  float sum[V];
#pragma unroll
  for (int e = 0; e < V; e++) sum[e] = -0.0f;
  auto write = [&](uint32_t k) {
    const Row out(p.table + (uint64_t)k * p.tableStride + at, n * (uint32_t)sizeof(Tab));
    Run<Tab, V> y;
    if constexpr (ACC) y.load(out, 0, lane * V);
#pragma unroll
    for (int e = 0; e < V; e++) y.set(e, ACC ? __builtin_fmaf(p.scale, sum[e], y.at(e)) : p.scale * sum[e]);
    y.store(out, 0, lane * V);
  };
  if (firstKey != none) {
    Run<Out, V> x[kTinyChunk];
    auto keyAt = [&](uint32_t i) { return (uint32_t)__builtin_amdgcn_readlane(myKey, i); }; // none from `count` on
#pragma unroll
    for (uint32_t i = 0; i < kTinyChunk; i++) {
      const uint32_t token = __builtin_amdgcn_readlane(myTok, i);
      x[i].template load<kAuxStream>(Row(p.grad + (uint64_t)token * p.gradStride + at, keyAt(i) != none ? n * (uint32_t)sizeof(Out) : 0), 0, lane * V);
    }
#pragma unroll
    for (uint32_t i = 0; i < kTinyChunk; i++) {
      const uint32_t k = keyAt(i), next = i + 1 < count ? keyAt(i + 1) : after;
      if (k == none) continue;
#pragma unroll
      for (int e = 0; e < V; e++) sum[e] += x[i].at(e);
      if (k == next && i + 1 < count) continue;
      if (k != next && (began || k != firstKey)) {
        write(k);
      } else {
        const uint32_t second = k == firstKey && !began ? 0 : 1;
#pragma unroll
        for (int e = 0; e < V; e++) part[wave][second][lane][e] = sum[e];
      }
#pragma unroll
      for (int e = 0; e < V; e++) sum[e] = -0.0f;
    }
  }
  __syncthreads();
  if (!join) return;
#pragma unroll
  for (int e = 0; e < V; e++) sum[e] = part[wave][1][lane][e];
  for (uint32_t w = wave + 1; w < kTinyWaves && w * kTinyChunk < p.tokens && sortedKey[w * kTinyChunk] == lastKey; w++)
#pragma unroll
    for (int e = 0; e < V; e++) sum[e] += part[w][0][lane][e];
  write(lastKey);
}

// `sums` workgroups of the first kind and `others` of the second, in launches of at most kMaxGrid.
template <typename K>
int inPieces(K kernel, SumParams p, uint64_t sums, uint64_t others, uint32_t threads, hipStream_t stream) {
  if (sums + others > 0xffffffffull) return (int)hipErrorInvalidValue;
  p.sumBlocks = (uint32_t)sums;
  for (uint64_t base = 0; base < sums + others; base += kMaxGrid) {
    p.base = (uint32_t)base;
    const uint64_t left = sums + others - base;
    kernel<<<dim3((unsigned)(left < kMaxGrid ? left : kMaxGrid)), dim3(threads), 0, stream>>>(p);
    const int e = (int)hipGetLastError();
    if (e) return e;
  }
  return (int)hipSuccess;
}

template <int V, bool ACC>
int gradientFor(const EmbedGradCall &c, hipStream_t stream) {
  const GradPlan g = gradPlan(c.tokens, c.vocab, c.dim);
  char *ws = (char *)c.workspace;
  const uint32_t sorted = (g.passes - 1) & 1;
  SumParams p{};
  if constexpr (!ACC) {
    p.clear.table = (char *)c.table;
    p.clear.rowBytes = c.dim * sizeof(Tab);
    p.clear.strideBytes = c.tableStride * sizeof(Tab);
    p.clear.elem = (uint32_t)sizeof(Tab);
    p.clear.vocab = g.vocab;
    p.clear.rows = clearGroup(c.vocab);
    p.clear.tokens = g.tokens;
    p.clear.ids = c.ids;
    p.clear.first = c.first;
    p.clear.wideIds = c.wideIds;
  }
  if (c.tokens <= kTinyTokens) {
    p.grad = (const Out *)c.grad;
    p.gradStride = c.gradStride;
    p.table = (Tab *)c.table;
    p.tableStride = c.tableStride;
    p.dim = c.dim;
    p.tokens = g.tokens;
    p.vocab = g.vocab;
    p.scale = c.scale;
    p.clear.ids = c.ids;
    p.clear.first = c.first;
    p.clear.wideIds = c.wideIds;
    return inPieces(gradTinyKernel<V, ACC>, p, c.tokens ? (c.dim + 64 * V - 1) / (64 * V) : 0,
                    ACC ? 0 : clearGroups(p.clear), 64 * kTinyWaves, stream);
  }
  {
    const int e = launchSort(c, g, ACC ? nullptr : &p.clear, &p.clearFrom, stream);
    if (e) return e;
  }
  p.grad = (const Out *)c.grad;
  p.gradStride = c.gradStride;
  p.table = (Tab *)c.table;
  p.tableStride = c.tableStride;
  p.dim = c.dim;
  p.tokens = g.tokens;
  p.vocab = g.vocab;
  p.chunk = g.chunk;
  p.chunks = g.chunks;
  p.dimPad = g.dimPad;
  p.scale = c.scale;
  p.key = (const uint32_t *)(ws + g.keyAt[sorted]);
  p.tok = (const uint32_t *)(ws + g.tokAt[sorted]);
  if (g.blocks > 1) p.clear.flags = (const uint8_t *)(ws + g.flagAt);
  else p.clear.key = p.key;
  p.part = (float *)(ws + g.partAt);
  const uint64_t waves = (c.dim + 64 * V * kSumRuns<V, ACC> - 1) / (64 * V * kSumRuns<V, ACC>);
  p.waves = waves < kSumThreads / 64 ? (uint32_t)waves : kSumThreads / 64;
  p.slices = (uint32_t)((waves + p.waves - 1) / p.waves);
  const uint64_t groups = ACC ? 0 : clearGroups(p.clear) - p.clearFrom, sums = (uint64_t)g.chunks * p.slices;
  int e = inPieces(gradSumKernel<V, ACC>, p, sums, groups, kSumThreads, stream);
  if (e || g.chunks < 2) return e;
  p.slices = (uint32_t)((c.dim + kShortColumns - 1) / kShortColumns);
  const uint64_t units = (uint64_t)(g.chunks - 1) * p.slices;
  return inPieces(gradJoinKernel<(V > 1), ACC>, p, (uint64_t)((g.chunks - 1) / kShort) * ((c.dim + kLongColumns - 1) / kLongColumns),
                  (units + kJoinWaves - 1) / kJoinWaves, 64 * kJoinWaves, stream);
}

} // namespace

#define FLAGCX_NAME2(a, x, y) a##_##x##_##y
#define FLAGCX_NAME(a, x, y) FLAGCX_NAME2(a, x, y)
int FLAGCX_NAME(launchEmbedding, FLAGCX_TABLE, FLAGCX_OUT)(const EmbedCall &c, hipStream_t stream) {
  return c.vec ? lookupFor<kVec>(c, stream) : lookupFor<1>(c, stream);
}
int FLAGCX_NAME(launchEmbeddingGrad, FLAGCX_TABLE, FLAGCX_OUT)(const EmbedGradCall &c, hipStream_t stream) {
  if (c.accumulate) return c.vec ? gradientFor<kVec, true>(c, stream) : gradientFor<1, true>(c, stream);
  return c.vec ? gradientFor<kVec, false>(c, stream) : gradientFor<1, false>(c, stream);
}

} // namespace flagcx_amd
