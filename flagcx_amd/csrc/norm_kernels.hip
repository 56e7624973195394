// norm_kernels.hip - the end of a tensor-parallel block and its gradient.
//
//   s = sum_j x_j                           u = s r1 W1,  r1 = (mean(s^2) + eps)^-1/2   (or u = s)
//   h = residual + scale g u                y = h r2 W2,  r2 = (mean(h^2) + eps)^-1/2
// and, from dy and dh, with d the whole gradient of h:
//   d  = dh + r2 (dy W2 - n2 mean(dy W2 n2)),  n2 = h r2      dW2 = sum_rows dy n2
//   dg = sum scale d u (over the rows that share g)           c   = scale g d
//   ds = r1 (c W1 - n1 mean(c W1 n1)),  n1 = s r1             dW1 = sum_rows c n1
//
// Both are streams: a few operations an element against 10 to 40 bytes, so memory bounds
// them and the layout serves one thing, that every byte of a row moves once.  A team of
// wavefronts holds its row in registers, E elements a lane, between the two sums that the
// norms need; the sums go through the vector unit inside a wavefront and through 64 bytes
// of LDS between them.  All state is fp32.
//
// Compiled once per pair of types: -DFLAGCX_ACT=<enum> -DFLAGCX_RES=<enum>.
#include "launch.h"
#include "residual.h"
#include "residual_device.h"

namespace flagcx_amd {
namespace { // per unit: the same names stand for other types in the next one

#if FLAGCX_ACT == 6
typedef h16 Act;
#elif FLAGCX_ACT == 7
typedef float Act;
#elif FLAGCX_ACT == 9
typedef b16 Act;
#endif
#if FLAGCX_RES == 7
typedef float Res;
#else
typedef Act Res;
#endif

constexpr int kVec = 16 / (int)sizeof(Res); // elements of a run: 16 bytes of the wider type

// Single elements are stored plainly: L2 gathers them to lines.
template <int V>
constexpr int kRowStore = V > 1 ? kAuxStream : kAuxPlain;

// Sums of M values over the team's wavefronts, the same bits in every lane.  `parity`
// alternates between two sets of slots: a wavefront that writes a set has passed the
// barrier of the sum in between, which every wavefront reaches after reading that set.
// After the barrier lane i takes the sum of wavefront i mod 16 (zero beyond the last, see
// clearSlots), one read and a sum over 16 lanes instead of a read for each wavefront.
constexpr int kMaxWaves = 16;
typedef float Slots[2][3][kMaxWaves];
__device__ __forceinline__ void clearSlots(Slots &slots) { // seen by all after the first sum's barrier
  const uint32_t i = threadIdx.x & 63u, waves = blockDim.x >> 6;
  if (threadIdx.x < 64 && threadIdx.y == 0 && (i & 15u) >= waves && i < 48) slots[0][i >> 4][i & 15u] = slots[1][i >> 4][i & 15u] = 0.0f;
}
template <int M>
__device__ __forceinline__ void teamSum(float (&x)[M], Slots &slots, uint32_t &parity) {
#pragma unroll
  for (int m = 0; m < M; m++) x[m] = waveSum(x[m]);
  if (blockDim.x <= 64) return; // the team is one wavefront
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  float(*s)[kMaxWaves] = slots[parity & 1u];
  parity++;
  if ((threadIdx.x & 63u) == 0) {
#pragma unroll
    for (int m = 0; m < M; m++) s[m][wave] = x[m];
  }
  __syncthreads();
#pragma unroll
  for (int m = 0; m < M; m++) x[m] = rowSum(s[m][threadIdx.x & 15u]);
}

// With 16 elements a lane the scheduler would start the loads of all of them at once and run
// out of registers: eight at a time.
template <int E>
__device__ __forceinline__ void pace() {
  if constexpr (E > 8)
    __builtin_amdgcn_sched_barrier(0);
}

// v_rsq_f32, off by at most one unit in the last place; x is at least eps, a normal number
__device__ __forceinline__ float inverseRoot(float x) { return __builtin_amdgcn_rsqf(x); }

// The row of gates that belongs to a row, without a division of 64 bits where 32 will do.
__device__ __forceinline__ uint64_t groupOf(uint64_t row, uint64_t rows) {
  return ((row | rows) >> 32) == 0 ? (uint64_t)((uint32_t)row / (uint32_t)rows) : row / rows;
}

// acc += x_{j0} + ... + x_{j0 + KB - 1}, in that order; all loads are issued before the first use
template <int KB, int V, int N>
__device__ __forceinline__ void foldInputs(float (&acc)[N][V], const NormForward &p, int j0, uint64_t row, uint32_t t,
                                           uint32_t team) {
  Run<Act, V> x[KB][N];
  afresh(t, team);
  const uint32_t bytes = p.c.dim * (uint32_t)sizeof(Act);
#pragma unroll
  for (int j = 0; j < KB; j++) {
    const Row in((const Act *)p.src[j0 + j] + row * p.srcStride, bytes);
#pragma unroll
    for (int n = 0; n < N; n++) x[j][n].template load<kAuxStream>(in, n * team * V, t * V);
  }
#pragma unroll
  for (int j = 0; j < KB; j++)
#pragma unroll
    for (int n = 0; n < N; n++)
#pragma unroll
      for (int i = 0; i < V; i++) acc[n][i] = x[j][n].at(i) + acc[n][i];
}

// blockDim = (team, teams of this workgroup); several teams only where a team is one wavefront.
template <int V, int E>
__global__ void __launch_bounds__(1024) normForwardKernel(NormForward p) {
  constexpr int N = E / V;
  // inputs whose loads are in flight together: at most eight and 32 registers of them
  constexpr int kWords = V == 1 ? E : E * (int)sizeof(Act) / 4;
  constexpr int KB = 32 / kWords < 8 ? 32 / kWords : 8;
  static_assert(KB == 8 || KB == 4 || KB == 2, "what KB leaves is 4, 2 and 1 once each");
  __shared__ Slots slots;
  clearSlots(slots);
  const uint32_t dim = p.c.dim;
  uint32_t team = blockDim.x;
  const float perDim = 1.0f / (float)dim;
  const bool f32w = p.c.weightF32 != 0;
  uint32_t parity = 0;
  const uint64_t stride = (uint64_t)gridDim.x * blockDim.y;
  for (uint64_t row = (uint64_t)blockIdx.x * blockDim.y + __builtin_amdgcn_readfirstlane(threadIdx.y); row < p.c.rows;
       row += stride) {
    uint32_t t = threadIdx.x;
    afresh(t, team);
    Run<Res, V> res[N];
    if (p.res) {
      const Row in((const Res *)p.res + row * p.resStride, dim * (uint32_t)sizeof(Res));
#pragma unroll
      for (int n = 0; n < N; n++) res[n].template load<kAuxStream>(in, n * team * V, t * V);
    }
    float a[N][V];
#pragma unroll
    for (int n = 0; n < N; n++)
#pragma unroll
      for (int i = 0; i < V; i++) a[n][i] = -0.0f; // -0 + x is x, bit for bit
    int j = 0;
    for (; j + KB <= p.k; j += KB) foldInputs<KB, V, N>(a, p, j, row, t, team);
    if constexpr (KB > 4)
      if (p.k - j >= 4) foldInputs<4, V, N>(a, p, j, row, t, team), j += 4;
    if constexpr (KB > 2)
      if (p.k - j >= 2) foldInputs<2, V, N>(a, p, j, row, t, team), j += 2;
    if constexpr (KB > 1)
      if (p.k - j >= 1) foldInputs<1, V, N>(a, p, j, row, t, team), j += 1;
    pace<E>();
    afresh(t, team);
    if (p.sumOut) {
      const Row out((Act *)p.sumOut + row * p.sumStride, dim * (uint32_t)sizeof(Act));
#pragma unroll
      for (int n = 0; n < N; n++) {
        Run<Act, V> o;
#pragma unroll
        for (int i = 0; i < V; i++) o.set(i, a[n][i]);
        o.template store<kRowStore<V>>(out, n * team * V, t * V);
      }
    }
    if (p.c.post) {
      float w[N][V], q[1] = {0.0f};
      if (p.c.w1) {
        loadWeights<Act, V, N>(w, p.c.w1, f32w, dim, 0, team * V, t * V);
      }
#pragma unroll
      for (int n = 0; n < N; n++)
#pragma unroll
        for (int i = 0; i < V; i++) q[0] = __builtin_fmaf(a[n][i], a[n][i], q[0]);
      teamSum(q, slots, parity);
      const float r1 = inverseRoot(__builtin_fmaf(q[0], perDim, p.c.eps));
#pragma unroll
      for (int n = 0; n < N; n++)
#pragma unroll
        for (int i = 0; i < V; i++) a[n][i] *= p.c.w1 ? r1 * (w[n][i] + p.c.offset) : r1;
    }
    // h = residual + scale g u
    afresh(t, team);
    const uint64_t group = p.c.gate && p.c.gateRows ? groupOf(row, p.c.gateRows) : 0;
    const Row gates(p.c.gate ? (const Act *)p.c.gate + group * p.c.gateStride : nullptr, p.c.gate ? dim * (uint32_t)sizeof(Act) : 0);
    const Row out((Res *)p.resOut + row * p.resOutStride, dim * (uint32_t)sizeof(Res));
    float q[1] = {0.0f};
#pragma unroll
    for (int n = 0; n < N; n++) {
      if (p.c.gate) {
        Run<Act, V> g;
        g.load(gates, n * team * V, t * V);
#pragma unroll
        for (int i = 0; i < V; i++) a[n][i] *= g.at(i);
      }
      Run<Res, V> o;
#pragma unroll
      for (int i = 0; i < V; i++) {
        a[n][i] = __builtin_fmaf(p.c.scale, a[n][i], p.res ? res[n].at(i) : 0.0f);
        o.set(i, a[n][i]);
        q[0] = __builtin_fmaf(a[n][i], a[n][i], q[0]);
      }
      o.template store<kRowStore<V>>(out, n * team * V, t * V);
      pace<E>();
    }
    if (p.c.pre) {
      float w[N][V];
      if (p.c.w2) {
        loadWeights<Act, V, N>(w, p.c.w2, f32w, dim, 0, team * V, t * V);
      }
      teamSum(q, slots, parity);
      afresh(t, team);
      const float r2 = inverseRoot(__builtin_fmaf(q[0], perDim, p.c.eps));
      const Row y((Act *)p.normOut + row * p.normStride, dim * (uint32_t)sizeof(Act));
#pragma unroll
      for (int n = 0; n < N; n++) {
        Run<Act, V> o;
#pragma unroll
        for (int i = 0; i < V; i++) o.set(i, a[n][i] * r2 * (p.c.w2 ? w[n][i] + p.c.offset : 1.0f));
        o.template store<kRowStore<V>>(y, n * team * V, t * V);
      }
    }
  }
}

// Rows that one wavefront holds with four elements a lane (20624 x 90 fp32: forward 17 -> 14 us, gradient 28 -> 23)
template <int V> constexpr int kFew = V <= 4 ? V : 4; // elements of a run then

constexpr unsigned kMaxGrid = 1u << 20; // workgroups; beyond that they take several rows each

template <int V>
int forwardFor(const NormForward &f, hipStream_t stream) {
  const TeamShape s = forwardShape(f.c.dim, f.c.rows);
  const unsigned teams = s.lanes == 64 ? 4 : 1;
  const uint64_t groups = (f.c.rows + teams - 1) / teams;
  const dim3 grid((unsigned)(groups < kMaxGrid ? groups : kMaxGrid)), block(s.lanes, teams);
  if (f.c.dim <= kNormNarrow) normForwardKernel<kFew<V>, 4><<<grid, block, 0, stream>>>(f);
  else if (s.elements == 8) normForwardKernel<V, 8><<<grid, block, 0, stream>>>(f);
  else normForwardKernel<V, 16><<<grid, block, 0, stream>>>(f);
  return (int)hipGetLastError();
}

// ---------------------------------------------------------------- backward

// One team walks every parts-th row of its part and carries the column sums of its part, A in registers,
// those of the weights in LDS (an update costs a few hundred cycles a row of some ten thousand).
// Gates enter through the rows that share them: with A = sum of d n1 over such rows,
//   dg = scale A W1   and   dW1 gets scale g A,
// so a row costs one sum for both, and f = scale g W1 is made once per group of gates.  Where
// every row has gates of its own, A takes g d n1 (dW1) and dg goes out with the row.
//
// A row's registers take the loads of a later row as soon as they are free: a CU holds 16
// wavefronts of this kernel, one or two teams, and would else wait out the latency of every row.
// With 8 elements a lane there is room for two rows (one where elements are loaded one by one,
// two bytes to a register), and for f; with 16 (dim above 8192) for none next to the column
// sums: all inputs but s are read again where they are used again, from L2, and so are weights.
template <int E>
constexpr uint32_t kHeld = (E <= 8 ? 3 : 2) * E; // floats of LDS a lane
template <int V, int E>
__global__ void __launch_bounds__(1024) normBackwardKernel(NormBackward p) {
  constexpr int N = E / V;
  constexpr bool kHold = E <= 8;              // a row's inputs stay in registers until they are used, and so does f
  constexpr uint32_t kRows = V > 1 ? 2 : 1; // of so many rows
  // pieces that are loaded together: inputs and weights where they are not held, gates of every row, what the sums need at
  // a group's end.  As many as the registers take: single elements would wait out the memory's latency one by one.
  constexpr int kLoads = V == 1 ? (kHold ? N : sizeof(Act) == sizeof(Res) ? 4 : 2) : 1, kPieces = kHold ? N : 1;
  __shared__ Slots slots;
  clearSlots(slots);
  extern __shared__ __attribute__((aligned(16))) float held[]; // a lane's own columns: dW1 of finished groups, dW2, with kHold W2
  const uint32_t dim = p.c.dim;
  const uint32_t team = blockDim.x;
  const uint32_t me = blockIdx.x * blockDim.y + __builtin_amdgcn_readfirstlane(threadIdx.y);
  // element j of a lane's columns; the lanes' runs of four lie side by side, which no bank minds
  const uint32_t all = blockDim.x * blockDim.y, slot = threadIdx.y * blockDim.x + threadIdx.x;
  auto column = [&](uint32_t j) -> float & { return held[((j / 4) * all + slot) * 4 + j % 4]; };
  auto w1Held = [&](int n, int i) -> float & { return column(n * V + i); };
  auto w2Held = [&](int n, int i) -> float & { return column(E + n * V + i); };
  auto w2Kept = [&](int n, int i) -> float & { return column(2 * E + n * V + i); };
  const float perDim = 1.0f / (float)dim;
  const bool f32w = p.c.weightF32 != 0;
  const uint32_t actBytes = dim * (uint32_t)sizeof(Act), resBytes = dim * (uint32_t)sizeof(Res);
  const bool perRow = p.c.gate && p.c.gateRows == 1;
  // the team's rows: every parts-th one of a run from number me % parts on, then the same of the run `abreast` further on
  struct Place {
    uint64_t row, end, run; // there is such a row if it lies before its run's end
  };
  auto placeIn = [&](uint64_t run) {
    const uint64_t start = run * p.t.groupRows, end = start + p.t.groupRows;
    return Place{start + me % p.t.parts, end < p.c.rows ? end : p.c.rows, run};
  };
  auto following = [&](Place at) {
    at.row += p.t.parts;
    return at.row >= at.end && at.run + p.t.abreast < p.t.groups ? placeIn(at.run + p.t.abreast) : at;
  };
  auto isRow = [](const Place &at) { return at.row < at.end; };
  Place ahead = placeIn(me / p.t.parts); // the row whose inputs are asked for next
  if (me >= p.t.teams) ahead.end = 0;    // a team beyond the last, in the last workgroup
  const bool any = isRow(ahead);
  const bool needSum = p.c.post || p.dgate;

  struct Inputs {
    Run<Res, V> h[N], dh[N];
    Run<Act, V> dy[N], s[N];
  };
  // nothing is read behind the last row
  auto loadStreams = [&](Inputs &x, const Place &at) {
    const bool is = isRow(at);
    const uint64_t row = is ? at.row : 0;
    uint32_t t = threadIdx.x, lanes = team;
    afresh(t, lanes);
    const Row h((const Res *)p.h + row * p.hStride, p.c.pre && is ? resBytes : 0);
    const Row dy((const Act *)p.dy + row * p.dyStride, p.dy && is ? actBytes : 0);
    const Row dh((const Res *)p.dh + row * p.dhStride, p.dh && is ? resBytes : 0);
#pragma unroll
    for (int n = 0; n < N; n++) {
      x.h[n].template load<kAuxStream>(h, n * lanes * V, t * V);
      x.dy[n].template load<kAuxStream>(dy, n * lanes * V, t * V);
      x.dh[n].template load<kAuxStream>(dh, n * lanes * V, t * V);
    }
  };
  auto loadSum = [&](Inputs &x, const Place &at) {
    const bool is = isRow(at);
    const uint64_t row = is ? at.row : 0;
    uint32_t t = threadIdx.x, lanes = team;
    afresh(t, lanes);
    const Row s((const Act *)p.sum + row * p.sumStride, needSum && is ? actBytes : 0);
#pragma unroll
    for (int n = 0; n < N; n++) x.s[n].template load<kAuxStream>(s, n * lanes * V, t * V);
  };
  // M pieces from number n on, all in flight together: a weight with its offset, a row of gates,
  // and f for the gates of a run
  auto weightsOf = [&](auto &w, const void *from, int n, uint32_t t, uint32_t lanes) {
    constexpr int M = sizeof(w) / sizeof(w[0]);
    if (from) loadWeights<Act, V, M>(w, from, f32w, dim, n * lanes * V, lanes * V, t * V);
#pragma unroll
    for (int m = 0; m < M; m++)
#pragma unroll
      for (int i = 0; i < V; i++) w[m][i] = from ? w[m][i] + p.c.offset : 1.0f;
  };
  auto gatesOf = [&](auto &g, uint64_t index, int n, uint32_t t, uint32_t lanes) {
    constexpr int M = sizeof(g) / sizeof(g[0]);
    Run<Act, V> x[M];
    if (p.c.gate) {
      const Row in((const Act *)p.c.gate + index * p.c.gateStride, actBytes);
#pragma unroll
      for (int m = 0; m < M; m++) x[m].load(in, (n + m) * lanes * V, t * V);
    }
#pragma unroll
    for (int m = 0; m < M; m++)
#pragma unroll
      for (int i = 0; i < V; i++) g[m][i] = p.c.gate ? x[m].at(i) : 1.0f;
  };
  auto factorOf = [&](auto &f, uint64_t run, int n, uint32_t t, uint32_t lanes) {
    constexpr int M = sizeof(f) / sizeof(f[0]);
    weightsOf(f, p.c.w1, n, t, lanes);
    if (!perRow) {
      float g[M][V];
      gatesOf(g, run, n, t, lanes);
#pragma unroll
      for (int m = 0; m < M; m++)
#pragma unroll
        for (int i = 0; i < V; i++) f[m][i] *= p.c.scale * g[m][i];
    }
  };
  Inputs x0, x1; // x1 only with two rows
  Place p0 = ahead, p1{};
  if constexpr (kHold) {
    loadStreams(x0, ahead);
    loadSum(x0, ahead);
    if constexpr (kRows == 2) {
      p1 = following(p0);
      loadStreams(x1, p1);
      loadSum(x1, p1);
    }
  }
  ahead = following(kRows == 2 && kHold ? p1 : p0);
  float A[N][V];
  float f[kHold ? N : 1][V];
  {
    const uint32_t t = threadIdx.x, lanes = team;
    float w[kHold ? N : 1][V];
    if constexpr (kHold) {
      weightsOf(w, p.c.w2, 0, t, lanes);
      if (any) factorOf(f, p0.run, 0, t, lanes);
    }
#pragma unroll
    for (int n = 0; n < N; n++)
#pragma unroll
      for (int i = 0; i < V; i++) {
        A[n][i] = 0.0f;
        w1Held(n, i) = 0.0f;
        w2Held(n, i) = 0.0f;
        if constexpr (kHold) w2Kept(n, i) = w[n][i];
      }
  }
  uint32_t parity = 0;
  // one row, whose inputs x has or awaits; takes those of a later row where it is done with them
  auto doRow = [&](Inputs &x, Place &at) {
    const uint64_t row = at.row;
    uint32_t t = threadIdx.x, lanes = team;
    afresh(t, lanes);
    const Row hIn((const Res *)p.h + row * p.hStride, p.c.pre ? resBytes : 0);
    const Row dyIn((const Act *)p.dy + row * p.dyStride, p.dy ? actBytes : 0);
    const Row dhIn((const Res *)p.dh + row * p.dhStride, p.dh ? resBytes : 0);
    const Row sIn((const Act *)p.sum + row * p.sumStride, needSum ? actBytes : 0);
    float d[N][V]; // the whole gradient of h, then c W1
    float q[3] = {0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int n0 = 0; n0 < N; n0 += kLoads) {
      float w[kLoads][V];
      if constexpr (!kHold) {
#pragma unroll
        for (int n = n0; n < n0 + kLoads; n++) {
          x.h[n].load(hIn, n * lanes * V, t * V);
          x.dy[n].load(dyIn, n * lanes * V, t * V);
          x.s[n].template load<kAuxStream>(sIn, n * lanes * V, t * V);
        }
        weightsOf(w, p.c.w2, n0, t, lanes);
      }
#pragma unroll
      for (int n = n0; n < n0 + kLoads; n++)
#pragma unroll
        for (int i = 0; i < V; i++) {
          q[0] = __builtin_fmaf(x.h[n].at(i), x.h[n].at(i), q[0]);
          q[1] = __builtin_fmaf(x.dy[n].at(i) * (kHold ? w2Kept(n, i) : w[n - n0][i]), x.h[n].at(i), q[1]);
          q[2] = __builtin_fmaf(x.s[n].at(i), x.s[n].at(i), q[2]);
        }
      pace<E>();
    }
    teamSum(q, slots, parity);
    if constexpr (!kHold) __asm__ volatile("" ::: "memory"); // what follows reads anew
    afresh(t, lanes);
    pace<E>();
    const float r2 = p.c.pre ? inverseRoot(__builtin_fmaf(q[0], perDim, p.c.eps)) : 0.0f;
    const float m2 = q[1] * r2 * perDim; // mean(dy W2 n2)
    const float r1 = p.c.post ? inverseRoot(__builtin_fmaf(q[2], perDim, p.c.eps)) : 1.0f;
    const Row dresOut((Res *)p.dres + row * p.dresStride, p.dres ? resBytes : 0);
    const Row gateOut((Act *)p.dgate + row * p.dgateStride, p.dgate && perRow ? actBytes : 0);
    float e[1] = {0.0f};
#pragma unroll
    for (int n0 = 0; n0 < N; n0 += kLoads) {
      float w[kLoads][V], fn[kLoads][V], g[kLoads][V];
      if constexpr (!kHold) {
#pragma unroll
        for (int n = n0; n < n0 + kLoads; n++) {
          x.h[n].template load<kAuxStream>(hIn, n * lanes * V, t * V);
          x.dy[n].template load<kAuxStream>(dyIn, n * lanes * V, t * V);
          x.dh[n].template load<kAuxStream>(dhIn, n * lanes * V, t * V);
        }
        weightsOf(w, p.c.w2, n0, t, lanes);
      }
      if constexpr (kLoads > 1) {
        if constexpr (!kHold) factorOf(fn, at.run, n0, t, lanes);
        if (perRow) gatesOf(g, row, n0, t, lanes);
      }
#pragma unroll
      for (int n = n0; n < n0 + kLoads; n++) {
        Run<Res, V> o;
#pragma unroll
        for (int i = 0; i < V; i++) {
          const float n2 = x.h[n].at(i) * r2;
          w2Held(n, i) = __builtin_fmaf(x.dy[n].at(i), n2, w2Held(n, i));
          d[n][i] = __builtin_fmaf(r2, __builtin_fmaf(-n2, m2, x.dy[n].at(i) * (kHold ? w2Kept(n, i) : w[n - n0][i])), x.dh[n].at(i));
          o.set(i, d[n][i]);
        }
        if (p.dres) o.template store<kRowStore<V>>(dresOut, n * lanes * V, t * V);
        if constexpr (kLoads == 1 && !kHold) factorOf(fn, at.run, n, t, lanes); // registers are free by now
        float c1[V]; // the factor between d and c W1
#pragma unroll
        for (int i = 0; i < V; i++) c1[i] = kHold ? f[kHold ? n : 0][i] : fn[n - n0][i];
        if (perRow) {
          if constexpr (kLoads == 1) gatesOf(g, row, n, t, lanes);
          Run<Act, V> dg;
#pragma unroll
          for (int i = 0; i < V; i++) {
            const float u = d[n][i] * (x.s[n].at(i) * r1);
            A[n][i] = __builtin_fmaf(g[n - n0][i], u, A[n][i]);
            dg.set(i, p.c.scale * u * c1[i]);
            c1[i] *= p.c.scale * g[n - n0][i];
          }
          if (p.dgate) dg.template store<kRowStore<V>>(gateOut, n * lanes * V, t * V);
        } else {
#pragma unroll
          for (int i = 0; i < V; i++) A[n][i] = __builtin_fmaf(d[n][i], x.s[n].at(i) * r1, A[n][i]);
        }
#pragma unroll
        for (int i = 0; i < V; i++) {
          d[n][i] *= c1[i];
          e[0] = __builtin_fmaf(d[n][i], x.s[n].at(i) * r1, e[0]);
        }
      }
      pace<E>();
    }
    if constexpr (kHold) loadStreams(x, ahead);
    if (p.ds) {
      float m1 = 0.0f;
      if (p.c.post) {
        teamSum(e, slots, parity);
        m1 = e[0] * perDim;
      }
      afresh(t, lanes);
      const Row out((Act *)p.ds + row * p.dsStride, actBytes);
#pragma unroll
      for (int n = 0; n < N; n++) {
        Run<Act, V> o;
#pragma unroll
        for (int i = 0; i < V; i++)
          o.set(i, p.c.post ? r1 * __builtin_fmaf(-(x.s[n].at(i) * r1), m1, d[n][i]) : d[n][i]);
        o.template store<kRowStore<V>>(out, n * lanes * V, t * V);
        pace<E>();
      }
    }
    if constexpr (kHold) loadSum(x, ahead);
    if (!perRow && row + p.t.parts >= at.end) { // the last row that this team has of these gates
      const bool whole = p.t.parts == 1;
      afresh(t, lanes);
      const Row gates((Act *)p.dgate + at.run * p.dgateStride, p.dgate && whole ? actBytes : 0);
      const Row part(p.partial + (2ull * p.t.teams + at.run * p.t.parts + me % p.t.parts) * dim, p.dgate && !whole ? dim * 4u : 0);
#pragma unroll
      for (int n0 = 0; n0 < N; n0 += kPieces) {
        float w[kPieces][V], g[kPieces][V];
        weightsOf(w, p.c.w1, n0, t, lanes);
        gatesOf(g, at.run, n0, t, lanes);
#pragma unroll
        for (int m = 0; m < kPieces; m++) {
          const int n = n0 + m;
          if (p.dgate) {
            Run<Act, V> o;
            Run<float, V> o32;
#pragma unroll
            for (int i = 0; i < V; i++) {
              o32.v[i] = p.c.scale * A[n][i] * w[m][i];
              o.set(i, o32.v[i]);
            }
            if (whole) o.template store<kRowStore<V>>(gates, n * lanes * V, t * V);
            else o32.store(part, n * lanes * V, t * V);
          }
#pragma unroll
          for (int i = 0; i < V; i++) {
            w1Held(n, i) += p.c.scale * g[m][i] * A[n][i];
            A[n][i] = 0.0f;
          }
        }
        pace<E>();
      }
      if constexpr (kHold)
        if (at.run + p.t.abreast < p.t.groups) factorOf(f, at.run + p.t.abreast, 0, t, lanes);
    }
    at = ahead;
    ahead = following(ahead);
  };
  while (isRow(p0)) {
    doRow(x0, p0);
    if constexpr (kHold && kRows == 2) {
      if (!isRow(p1)) break;
      doRow(x1, p1);
    }
  }
  // this workgroup's column sums: of its one team, or of its teams of one wavefront, joined in order
  const uint32_t t = threadIdx.x, lanes = team;
  const uint64_t slab = (uint64_t)p.t.teams * dim;
  const Row out1(p.partial + (uint64_t)blockIdx.x * dim, p.dw1 ? dim * 4u : 0);
  const Row out2(p.partial + slab + (uint64_t)blockIdx.x * dim, p.dw2 ? dim * 4u : 0);
  if (perRow) {
#pragma unroll
    for (int n = 0; n < N; n++)
#pragma unroll
      for (int i = 0; i < V; i++) w1Held(n, i) = p.c.scale * A[n][i];
  }
  if (!kHold || blockDim.y == 1) {
#pragma unroll
    for (int n = 0; n < N; n++) {
      Run<float, V> o1, o2;
#pragma unroll
      for (int i = 0; i < V; i++) {
        o1.v[i] = w1Held(n, i);
        o2.v[i] = w2Held(n, i);
      }
      o1.store(out1, n * lanes * V, t * V);
      o2.store(out2, n * lanes * V, t * V);
    }
  } else {
    __syncthreads();
    for (uint32_t u = __builtin_amdgcn_readfirstlane(threadIdx.y); u < 2 * N; u += blockDim.y) { // a run of dW1 or of dW2
      Run<float, V> o;
#pragma unroll
      for (int i = 0; i < V; i++) {
        const uint32_t j = (u < N ? u * V : E + (u - N) * V) + i;
        o.v[i] = 0.0f;
        for (uint32_t y = 0; y < blockDim.y; y++) o.v[i] += held[((j / 4) * all + y * blockDim.x + t) * 4 + j % 4];
      }
      o.store(u < N ? out1 : out2, (u < N ? u : u - N) * lanes * V, t * V);
    }
  }
}

// Joins the workgroups' column sums (the teams' for gates): blockIdx.x takes COLS columns,
// blockIdx.y one sum (dW1, dW2, then one per group of gates).  Sixteen wavefronts take 64 / COLS
// of them at a time and are joined in order.  Narrow rows, which have the most, fill few
// workgroups of 64 columns.  Groups of few parts, of which there may be many, are a wavefront's
// each (7742 x 192 in groups of 6 rows: 44 -> 19 us, 16384 x 6144 in groups of 55: 421 -> 378).
struct JoinParams {
  const float *partial;
  uint64_t slab;
  uint32_t dim, rows, parts, groups; // partial rows of a weight's gradient, of a run's gates at most; runs
  uint64_t groupRows, batch; // rows of a run, of all
  void *out[3];
  uint64_t gateStride;
  int32_t weightF32;
  uint32_t which[2]; // slabs that blockIdx.y = 0, 1 stand for; blockIdx.y >= weights is group blockIdx.y - weights
  uint32_t weights;
};
constexpr int kJoinWaves = 16;
constexpr uint32_t kNarrowJoin = 1024, kFewParts = 16;
template <int COLS>
__global__ void __launch_bounds__(64 * kJoinWaves) normJoinKernel(JoinParams p) {
  static_assert(COLS == 64 || COLS == 16, "a wavefront's lanes are one or four teams");
  __shared__ float part[kJoinWaves][COLS];
  constexpr uint32_t kTeams = 64 / COLS;
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const uint32_t col = blockIdx.x * COLS + lane % COLS;
  const bool isGate = blockIdx.y >= p.weights;
  const bool few = isGate && p.parts <= kFewParts; // then every wavefront has a group of its own
  const uint32_t which = isGate ? 2u : p.which[blockIdx.y];
  const uint32_t group = !isGate ? 0 : few ? (blockIdx.y - p.weights) * kJoinWaves + wave : blockIdx.y - p.weights;
  if (few && group >= p.groups) return;
  const uint64_t left = p.batch - group * p.groupRows;
  const uint32_t n = !isGate ? p.rows : left < p.parts ? (uint32_t)left : p.parts;
  const float *in = p.partial + which * p.slab + ((uint64_t)group * p.parts) * p.dim + col;
  float s = 0.0f;
  if (col < p.dim) {
    if (few) {
#pragma unroll
      for (uint32_t i = 0; i < kFewParts / kTeams; i++) {
        const uint32_t j = i * kTeams + lane / COLS;
        s += j < n ? in[(uint64_t)j * p.dim] : -0.0f; // changes no sum
      }
    } else {
#pragma unroll 8
      for (uint32_t i = wave * kTeams + lane / COLS; i < n; i += kJoinWaves * kTeams) s += in[(uint64_t)i * p.dim];
    }
  }
  if constexpr (COLS == 16) {
    s += __shfl_xor(s, 16);
    s += __shfl_xor(s, 32);
  }
  if (!few) {
    if (lane < COLS) part[wave][lane] = s;
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int w = 1; w < kJoinWaves; w++) s += part[w][lane % COLS];
  }
  if (lane >= COLS || col >= p.dim) return;
  if (isGate) ((Act *)p.out[2])[group * p.gateStride + col] = (Act)s;
  else if (p.weightF32) ((float *)p.out[which])[col] = s;
  else ((Act *)p.out[which])[col] = (Act)s;
}

template <int V>
int backwardFor(const NormBackward &b, hipStream_t stream) {
  const TeamShape s = backwardShape(b.c.dim);
  const unsigned per = s.lanes == 64 && b.t.teams > 1024 ? 4 : 1; // few teams are spread over the CUs
  const dim3 grid((b.t.teams + per - 1) / per), block(s.lanes, per);
  int e = (int)hipSuccess;
  if (b.t.teams) { // else there are no rows, and the sums below are zeros
    const unsigned lds = s.lanes * per * 4u;
    if (b.c.dim <= kNormNarrow) normBackwardKernel<kFew<V>, 4><<<grid, block, kHeld<4> * lds, stream>>>(b);
    else if (s.elements == 8) normBackwardKernel<V, 8><<<grid, block, kHeld<8> * lds, stream>>>(b);
    else normBackwardKernel<V, 16><<<grid, block, kHeld<16> * lds, stream>>>(b);
    e = (int)hipGetLastError();
  }
  if (e) return e;
  JoinParams j{};
  j.partial = b.partial;
  j.slab = (uint64_t)b.t.teams * b.c.dim;
  j.dim = b.c.dim;
  j.rows = grid.x;
  j.parts = b.t.parts;
  j.groups = (uint32_t)b.t.groups; // where there are gates' sums to join
  j.groupRows = b.t.groupRows;
  j.batch = b.c.rows;
  j.out[0] = b.dw1;
  j.out[1] = b.dw2;
  j.out[2] = b.dgate;
  j.gateStride = b.dgateStride;
  j.weightF32 = b.c.weightF32;
  if (b.dw1) j.which[j.weights++] = 0;
  if (b.dw2) j.which[j.weights++] = 1;
  unsigned sums = j.weights;
  if (b.dgate && b.c.gateRows != 1 && b.t.parts > 1) sums += b.t.parts > kFewParts ? j.groups : (j.groups + kJoinWaves - 1) / kJoinWaves;
  if (b.dgate && !b.t.teams && !b.c.gateRows) sums++, j.groups = 1;
  if (sums) {
    // by dim alone: a gradient has the same bits whichever others are asked for
    if (b.c.dim <= kNarrowJoin) normJoinKernel<16><<<dim3((b.c.dim + 15) / 16, sums), dim3(64 * kJoinWaves), 0, stream>>>(j);
    else normJoinKernel<64><<<dim3((b.c.dim + 63) / 64, sums), dim3(64 * kJoinWaves), 0, stream>>>(j);
    e = (int)hipGetLastError();
  }
  return e;
}

} // namespace

#define FLAGCX_NAME2(a, x, y) a##_##x##_##y
#define FLAGCX_NAME(a, x, y) FLAGCX_NAME2(a, x, y)
int FLAGCX_NAME(launchNormForward, FLAGCX_ACT, FLAGCX_RES)(const NormForward &f, hipStream_t stream) {
  return f.c.vec ? forwardFor<kVec>(f, stream) : forwardFor<1>(f, stream);
}
int FLAGCX_NAME(launchNormBackward, FLAGCX_ACT, FLAGCX_RES)(const NormBackward &b, hipStream_t stream) {
  return b.c.vec ? backwardFor<kVec>(b, stream) : backwardFor<1>(b, stream);
}

} // namespace flagcx_amd
