// host_residual.cpp - the C ABI of the residual stream's operators (include/flagcx_amd.h):
// checks on the host what the kernels and their grids assume, picks the launcher of the
// types, launches.  Allocates nothing, keeps nothing between calls.
#include "../../include/flagcx_amd.h"
#include "launch.h"
#include "residual.h"

#include <cstdarg>
#include <cstdio>
#include <cstring>

namespace flagcx_amd {

#define FLAGCX_DECL_NORM(a, r)                                     \
  int launchNormForward_##a##_##r(const NormForward &, hipStream_t); \
  int launchNormBackward_##a##_##r(const NormBackward &, hipStream_t);
FLAGCX_DECL_NORM(6, 6) FLAGCX_DECL_NORM(6, 7) FLAGCX_DECL_NORM(7, 7) FLAGCX_DECL_NORM(9, 9) FLAGCX_DECL_NORM(9, 7)
#undef FLAGCX_DECL_NORM
#define FLAGCX_DECL_EMBED(t, o)                                 \
  int launchEmbedding_##t##_##o(const EmbedCall &, hipStream_t); \
  int launchEmbeddingGrad_##t##_##o(const EmbedGradCall &, hipStream_t);
FLAGCX_DECL_EMBED(6, 6) FLAGCX_DECL_EMBED(6, 7) FLAGCX_DECL_EMBED(7, 6) FLAGCX_DECL_EMBED(7, 7) FLAGCX_DECL_EMBED(7, 9)
FLAGCX_DECL_EMBED(9, 7) FLAGCX_DECL_EMBED(9, 9)
#undef FLAGCX_DECL_EMBED

int launchNormForward(const NormForward &f, int act, int res, hipStream_t stream) {
  switch (act * 16 + res) {
    case 0x66: return launchNormForward_6_6(f, stream);
    case 0x67: return launchNormForward_6_7(f, stream);
    case 0x77: return launchNormForward_7_7(f, stream);
    case 0x99: return launchNormForward_9_9(f, stream);
    case 0x97: return launchNormForward_9_7(f, stream);
    default: return (int)hipErrorInvalidValue;
  }
}
int launchNormBackward(const NormBackward &b, int act, int res, hipStream_t stream) {
  switch (act * 16 + res) {
    case 0x66: return launchNormBackward_6_6(b, stream);
    case 0x67: return launchNormBackward_6_7(b, stream);
    case 0x77: return launchNormBackward_7_7(b, stream);
    case 0x99: return launchNormBackward_9_9(b, stream);
    case 0x97: return launchNormBackward_9_7(b, stream);
    default: return (int)hipErrorInvalidValue;
  }
}
int launchEmbedding(const EmbedCall &c, int table, int out, hipStream_t stream) {
  switch (table * 16 + out) {
    case 0x66: return launchEmbedding_6_6(c, stream);
    case 0x67: return launchEmbedding_6_7(c, stream);
    case 0x76: return launchEmbedding_7_6(c, stream);
    case 0x77: return launchEmbedding_7_7(c, stream);
    case 0x79: return launchEmbedding_7_9(c, stream);
    case 0x97: return launchEmbedding_9_7(c, stream);
    case 0x99: return launchEmbedding_9_9(c, stream);
    default: return (int)hipErrorInvalidValue;
  }
}
int launchEmbeddingGrad(const EmbedGradCall &c, int out, int table, hipStream_t stream) {
  switch (table * 16 + out) {
    case 0x66: return launchEmbeddingGrad_6_6(c, stream);
    case 0x67: return launchEmbeddingGrad_6_7(c, stream);
    case 0x76: return launchEmbeddingGrad_7_6(c, stream);
    case 0x77: return launchEmbeddingGrad_7_7(c, stream);
    case 0x79: return launchEmbeddingGrad_7_9(c, stream);
    case 0x97: return launchEmbeddingGrad_9_7(c, stream);
    case 0x99: return launchEmbeddingGrad_9_9(c, stream);
    default: return (int)hipErrorInvalidValue;
  }
}

// As many teams as the 256 CUs hold at once, 16 wavefronts each.
static uint64_t mostTeams(uint32_t dim) { return 256 * (16 / (backwardShape(dim).lanes / 64)); }
constexpr uint64_t kRowEach = 256;     // up to so many rows a team takes one, of more at least two
constexpr uint64_t kMostPartsTimes = 8; // parts of all groups of gates, in mostTeams

NormTeams normTeams(uint64_t rows, uint32_t dim, uint64_t gateRows) {
  NormTeams t{};
  if (!rows) return t;
  const bool shared = gateRows > 1 && gateRows < rows;
  t.groupRows = shared ? gateRows : rows;
  t.groups = (rows + t.groupRows - 1) / t.groupRows;
  // of more rows than CUs a team takes two at least, so that its column sums (up to three rows of
  // fp32) stay small next to the rows themselves.  Up to there the latency of one row is the time
  // (128 x 4096: 10 us against 11.5).
  const uint64_t most = mostTeams(dim), least = rows > kRowEach ? 2 : 1;
  const uint64_t limit = (rows + least - 1) / least < most ? (rows + least - 1) / least : most;
  // The split whose longest team is done first, in rows: one more for the end of a run, a 24th for each
  // doubling of the places that are read at a time.  16384 x 6144 bf16/fp32 on 256 teams: 8 groups in
  // turns of two 325 us, abreast 342; 3 groups abreast, as 86 teams each, are two rounds and 495, in
  // turns 326.
  uint64_t best = ~0ull;
  for (uint64_t c = 1;; c *= 2) {
    if (c > t.groups) c = t.groups;
    if (c > limit) c = limit;
    const bool last = c == t.groups || c == limit;
    uint64_t parts = limit / c;
    if (parts > (t.groupRows + least - 1) / least) parts = (t.groupRows + least - 1) / least;
    const uint64_t each = (t.groupRows + parts - 1) / parts, turns = (t.groups + c - 1) / c;
    parts = (t.groupRows + each - 1) / each;
    uint64_t doublings = 0;
    while ((c >> doublings) > 1) doublings++;
    const uint64_t cost = turns * (each + (shared ? 1 : 0)) * (24 + doublings);
    // partial sums of gates stay few next to the rows
    if (cost < best && (last || parts == 1 || t.groups * parts <= kMostPartsTimes * most)) {
      best = cost;
      t.parts = (uint32_t)parts;
      t.abreast = (uint32_t)((t.groups + turns - 1) / turns);
    }
    if (last) break;
  }
  t.teams = t.parts * t.abreast;
  return t;
}

namespace {

flagcxResult_t fail(flagcxResult_t code, const char *fmt, ...) {
  char text[256];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(text, sizeof(text), fmt, ap);
  va_end(ap);
  setLastError(text);
  return code;
}

// Enum arguments come from C callers and may hold any int: read their bits.
template <typename E>
int bitsOf(const E &e) {
  static_assert(sizeof(E) == sizeof(int), "flagcx enums are int sized");
  int v;
  memcpy(&v, &e, sizeof(v));
  return v;
}

hipStream_t hipStreamOf(flagcxStream_t s) { return s ? *reinterpret_cast<hipStream_t *>(s) : nullptr; }

// A NULL stream blocks until the work has finished.
flagcxResult_t finish(flagcxStream_t s, int err, const char *who) {
  if (err == (int)hipSuccess && !s) err = (int)hipStreamSynchronize(nullptr);
  if (err == (int)hipSuccess) return flagcxSuccess;
  return fail(flagcxUnhandledDeviceError, "%s: %s", who, hipGetErrorString((hipError_t)err));
}

uint64_t floatSize(int dt) { return dt == flagcxFloat16 || dt == flagcxBfloat16 ? 2 : dt == flagcxFloat32 ? 4 : 0; }

// One argument of a call that lies in device memory.
struct Span {
  const char *name;
  const void *p;
  uint64_t rows, rowBytes, stride; // stride in bytes
  uint64_t bytes;                  // from the first byte to the last
  uint32_t elem;
  bool output, rowwise; // rowwise: element i of the row is read before element i is written
};

// Collects the arguments of a call, checks each, and then each output against all others.
struct Args {
  const char *who;
  Span s[16];
  int n = 0;
  bool vec = true; // every row starts on 16 bytes
  flagcxResult_t bad = flagcxSuccess;

  explicit Args(const char *w) : who(w) {}

  // A matrix of `rows` rows; strideElems 0 stands for dim.  Returns the stride in elements.
  uint64_t add(const char *name, const void *p, uint64_t rows, uint64_t dim, uint64_t strideElems, uint32_t elem, bool output,
               bool rowwise, bool vector = true) {
    const uint64_t stride = strideElems ? strideElems : dim;
    if (bad != flagcxSuccess || !p || !rows || !dim) return stride;
    if ((uintptr_t)p % elem) return bad = fail(flagcxInvalidArgument, "%s: %s not aligned to %u", who, name, elem), stride;
    if (rows > 1 && stride < dim) return bad = fail(flagcxInvalidArgument, "%s: stride of %s below dim", who, name), stride;
    const unsigned __int128 bytes = ((unsigned __int128)(rows - 1) * stride + dim) * elem;
    if (bytes > (unsigned __int128)(UINT64_MAX - (uintptr_t)p))
      return bad = fail(flagcxInvalidArgument, "%s: size of %s overflows", who, name), stride;
    s[n++] = Span{name, p, rows, dim * elem, stride * elem, (uint64_t)bytes, elem, output, rowwise};
    if (vector && ((uintptr_t)p % 16 || (rows > 1 && stride * elem % 16))) vec = false;
    return stride;
  }

  static bool overlap(const Span &a, const Span &b) {
    const uintptr_t x = (uintptr_t)a.p, y = (uintptr_t)b.p;
    if (x >= y + b.bytes || y >= x + a.bytes) return false;
    if (a.rows > 1 && b.rows > 1 && a.stride == b.stride) { // side by side in rows of one stride
      const Span &lo = x <= y ? a : b, &hi = x <= y ? b : a;
      const uint64_t off = ((uintptr_t)hi.p - (uintptr_t)lo.p) % a.stride;
      if (off >= lo.rowBytes && off + hi.rowBytes <= a.stride) return false;
    }
    return true;
  }

  flagcxResult_t check() {
    if (bad != flagcxSuccess) return bad;
    for (int i = 0; i < n; i++) {
      if (!s[i].output) continue;
      for (int j = 0; j < n; j++) {
        if (i == j || (s[j].output && j < i)) continue;
        const Span &o = s[i], &x = s[j];
        const bool inPlace = !x.output && o.rowwise && x.rowwise && o.p == x.p && o.elem == x.elem &&
                             (o.rows == 1 || o.stride == x.stride);
        if (!inPlace && overlap(o, x)) return fail(flagcxInvalidArgument, "%s: %s overlaps %s", who, o.name, x.name);
      }
    }
    return flagcxSuccess;
  }
};

// What the forward and the backward call share.  Fills c but for the strides' checks.
flagcxResult_t prepareEnd(const char *who, const flagcxLocalBlockEnd *end, NormCall &c, int &act, int &res, int &weight) {
  if (!end) return fail(flagcxInvalidArgument, "%s: end is NULL", who);
  act = bitsOf(end->datatype);
  res = bitsOf(end->residualtype);
  weight = bitsOf(end->weighttype);
  if (!floatSize(act)) return fail(flagcxInvalidArgument, "%s: unsupported data type %d", who, act);
  if (res != act && res != flagcxFloat32) return fail(flagcxInvalidArgument, "%s: unsupported residualtype %d", who, res);
  if (weight != act && weight != flagcxFloat32) return fail(flagcxInvalidArgument, "%s: unsupported weighttype %d", who, weight);
  if (end->norms & ~(FLAGCX_LOCAL_NORM_POST | FLAGCX_LOCAL_NORM_PRE))
    return fail(flagcxInvalidArgument, "%s: norms %d", who, end->norms);
  if (end->dim < 1 || end->dim > FLAGCX_LOCAL_NORM_MAX_DIM)
    return fail(flagcxInvalidArgument, "%s: dim %zu outside [1, %d]", who, end->dim, FLAGCX_LOCAL_NORM_MAX_DIM);
  if (!(end->eps >= 1.17549435e-38f) || end->eps > 3.0e38f) // rejects NaN, zero, subnormals and infinity
    return fail(flagcxInvalidArgument, "%s: eps is not a normal number above zero", who);
  if (end->rows >> 40) return fail(flagcxInvalidArgument, "%s: rows %zu", who, end->rows);
  c = NormCall{};
  c.rows = end->rows;
  c.dim = (uint32_t)end->dim;
  c.post = (end->norms & FLAGCX_LOCAL_NORM_POST) != 0;
  c.pre = (end->norms & FLAGCX_LOCAL_NORM_PRE) != 0;
  c.weightF32 = weight == flagcxFloat32;
  c.scale = end->scale;
  c.eps = end->eps;
  c.offset = end->weightoffset;
  if (c.post) c.w1 = end->postweight;
  if (c.pre) c.w2 = end->preweight;
  c.gate = end->gate;
  c.gateRows = end->gaterows > 1 && end->gaterows >= end->rows && end->rows ? 0 : end->gaterows; // one group is all rows
  return flagcxSuccess;
}

uint64_t gateRowsOf(const NormCall &c) { return c.gateRows ? (c.rows + c.gateRows - 1) / c.gateRows : 1; }

void addEnd(Args &a, NormCall &c, const flagcxLocalBlockEnd *end, uint32_t as, uint32_t ws) {
  a.add("postweight", c.w1, 1, c.dim, 0, ws, false, false);
  a.add("preweight", c.w2, 1, c.dim, 0, ws, false, false);
  c.gateStride = a.add("gate", c.gate, gateRowsOf(c), c.dim, end->gatestride, as, false, false);
}

// Room for the partial rows of the sums: two a team, and one for each part of a group of gates where
// groups have several.  normTeams' split has fewer of them for 257 rows (129 teams) than for 256, and
// for some longer batches of groups than for shorter ones; what is asked for is the most that any
// batch up to this one needs, so that a workspace of the longest batch serves them all.  A group has
// at most as many parts as rows, all groups together kMostPartsTimes * mostTeams.  In whole sets of
// three rows.
flagcxResult_t backwardBytes(const char *who, const flagcxLocalBlockEnd *end, uint64_t *bytes) {
  NormCall c;
  int act, res, weight;
  flagcxResult_t r = prepareEnd(who, end, c, act, res, weight);
  if (r != flagcxSuccess) return r;
  const uint64_t most = mostTeams(c.dim), alone = c.rows < kRowEach ? c.rows : kRowEach, twos = (c.rows + 1) / 2;
  uint64_t teams = twos < most ? twos : most;
  if (teams < alone) teams = alone;
  uint64_t gates = 0;
  if (c.gate && c.gateRows == 0) gates = teams; // the parts of one group
  else if (c.gate && c.gateRows > 1) gates = c.rows < kMostPartsTimes * most ? c.rows : kMostPartsTimes * most;
  *bytes = (2 * teams + gates + 2) / 3 * 3 * c.dim * 4;
  return flagcxSuccess;
}

} // namespace
} // namespace flagcx_amd

using namespace flagcx_amd;

#pragma GCC visibility push(default)
extern "C" {

flagcxResult_t flagcxLocalReduceNorm(const flagcxLocalBlockEnd *end, const void *const *sendbuffs, int nranks,
                                     size_t sendstride, const void *residual, size_t residualstride,
                                     void *residualout, size_t residualoutstride, void *normout, size_t normstride,
                                     void *sumout, size_t sumstride, flagcxStream_t stream) {
  const char *who = "flagcxLocalReduceNorm";
  NormForward f{};
  int act, res, weight;
  flagcxResult_t r = prepareEnd(who, end, f.c, act, res, weight);
  if (r != flagcxSuccess) return r;
  if (!sendbuffs) return fail(flagcxInvalidArgument, "%s: sendbuffs is NULL", who);
  if (nranks < 1 || nranks > FLAGCX_LOCAL_MAX_RANKS)
    return fail(flagcxInvalidArgument, "%s: nranks %d outside [1, %d]", who, nranks, FLAGCX_LOCAL_MAX_RANKS);
  if (f.c.rows == 0) return flagcxSuccess;
  if (!residualout) return fail(flagcxInvalidArgument, "%s: residualout is NULL", who);
  if ((normout != nullptr) != (f.c.pre != 0))
    return fail(flagcxInvalidArgument, "%s: normout goes with FLAGCX_LOCAL_NORM_PRE", who);
  const uint32_t as = (uint32_t)floatSize(act), rs = (uint32_t)floatSize(res), ws = (uint32_t)floatSize(weight);
  const uint64_t rows = f.c.rows, dim = f.c.dim;
  Args a(who);
  f.resOut = residualout;
  f.resOutStride = a.add("residualout", residualout, rows, dim, residualoutstride, rs, true, true);
  f.normOut = normout;
  f.normStride = a.add("normout", normout, rows, dim, normstride, as, true, true);
  f.sumOut = sumout;
  f.sumStride = a.add("sumout", sumout, rows, dim, sumstride, as, true, true);
  f.res = residual;
  f.resStride = a.add("residual", residual, rows, dim, residualstride, rs, false, true);
  addEnd(a, f.c, end, as, ws);
  const int fixed = a.n;
  bool vec = true;
  for (int j = 0; j < nranks; j++) { // one after another: the list may be longer than Args holds
    if (!sendbuffs[j]) return fail(flagcxInvalidArgument, "%s: sendbuffs[%d] is NULL", who, j);
    f.src[j] = sendbuffs[j];
    a.n = fixed;
    f.srcStride = a.add("a sendbuff", sendbuffs[j], rows, dim, sendstride, as, false, true);
    if ((r = a.check()) != flagcxSuccess) return r;
    vec = vec && a.vec;
  }
  f.k = nranks;
  f.c.vec = vec && dim * as % 16 == 0;
  return finish(stream, launchNormForward(f, act, res, hipStreamOf(stream)), who);
}

flagcxResult_t flagcxLocalReduceNormBackwardWorkspace(const flagcxLocalBlockEnd *end, size_t *bytes) {
  const char *who = "flagcxLocalReduceNormBackwardWorkspace";
  if (!bytes) return fail(flagcxInvalidArgument, "%s: bytes is NULL", who);
  uint64_t b = 0;
  flagcxResult_t r = backwardBytes(who, end, &b);
  if (r == flagcxSuccess) *bytes = (size_t)b;
  return r;
}

flagcxResult_t flagcxLocalReduceNormBackward(const flagcxLocalBlockEnd *end, const void *sum, size_t sumstride,
                                             const void *residualout, size_t residualoutstride,
                                             const void *normgrad, size_t normgradstride,
                                             const void *residualoutgrad, size_t residualoutgradstride,
                                             void *sendgrad, size_t sendgradstride,
                                             void *residualgrad, size_t residualgradstride,
                                             void *postweightgrad, void *preweightgrad,
                                             void *gategrad, size_t gategradstride,
                                             void *workspace, size_t workspacebytes, flagcxStream_t stream) {
  const char *who = "flagcxLocalReduceNormBackward";
  NormBackward b{};
  int act, res, weight;
  flagcxResult_t r = prepareEnd(who, end, b.c, act, res, weight);
  if (r != flagcxSuccess) return r;
  if (postweightgrad && !b.c.w1) return fail(flagcxInvalidArgument, "%s: postweightgrad without a postweight", who);
  if (preweightgrad && !b.c.w2) return fail(flagcxInvalidArgument, "%s: preweightgrad without a preweight", who);
  if (gategrad && !b.c.gate) return fail(flagcxInvalidArgument, "%s: gategrad without a gate", who);
  if (normgrad && !b.c.pre) return fail(flagcxInvalidArgument, "%s: normgrad goes with FLAGCX_LOCAL_NORM_PRE", who);
  const uint64_t rows = b.c.rows, dim = b.c.dim;
  if (rows) {
    if (!normgrad && !residualoutgrad) return fail(flagcxInvalidArgument, "%s: normgrad and residualoutgrad are NULL", who);
    if (b.c.pre && !residualout) return fail(flagcxInvalidArgument, "%s: residualout is NULL", who);
    if (!sum && (b.c.post || gategrad)) return fail(flagcxInvalidArgument, "%s: sum is NULL", who);
  }
  uint64_t need = 0;
  r = backwardBytes(who, end, &need);
  if (r != flagcxSuccess) return r;
  if (need && !workspace) return fail(flagcxInvalidArgument, "%s: workspace is NULL", who);
  if ((uintptr_t)workspace % 16) return fail(flagcxInvalidArgument, "%s: workspace not aligned to 16", who);
  if (workspacebytes < need)
    return fail(flagcxInvalidArgument, "%s: workspace of %zu bytes, %llu are needed", who, workspacebytes, (unsigned long long)need);
  const uint32_t as = (uint32_t)floatSize(act), rs = (uint32_t)floatSize(res), ws = (uint32_t)floatSize(weight);
  Args a(who);
  b.sum = b.c.post || gategrad ? sum : nullptr;
  b.sumStride = a.add("sum", b.sum, rows, dim, sumstride, as, false, true);
  b.h = b.c.pre ? residualout : nullptr;
  b.hStride = a.add("residualout", b.h, rows, dim, residualoutstride, rs, false, true);
  b.dy = normgrad;
  b.dyStride = a.add("normgrad", normgrad, rows, dim, normgradstride, as, false, true);
  b.dh = residualoutgrad;
  b.dhStride = a.add("residualoutgrad", residualoutgrad, rows, dim, residualoutgradstride, rs, false, true);
  b.ds = sendgrad;
  b.dsStride = a.add("sendgrad", sendgrad, rows, dim, sendgradstride, as, true, true);
  b.dres = residualgrad;
  b.dresStride = a.add("residualgrad", residualgrad, rows, dim, residualgradstride, rs, true, true);
  b.dw1 = postweightgrad;
  a.add("postweightgrad", postweightgrad, 1, dim, 0, ws, true, false, false);
  b.dw2 = preweightgrad;
  a.add("preweightgrad", preweightgrad, 1, dim, 0, ws, true, false, false);
  b.dgate = gategrad;
  b.dgateStride = a.add("gategrad", gategrad, gateRowsOf(b.c), dim, gategradstride, as, true, false);
  addEnd(a, b.c, end, as, ws);
  if (need) a.add("workspace", workspace, 1, need, 0, 1, true, false, false);
  if ((r = a.check()) != flagcxSuccess) return r;
  b.c.vec = a.vec && dim * as % 16 == 0;
  b.partial = (float *)workspace;
  b.t = normTeams(rows, b.c.dim, b.c.gate ? b.c.gateRows : 0);
  return finish(stream, launchNormBackward(b, act, res, hipStreamOf(stream)), who);
}

flagcxResult_t flagcxLocalEmbedding(const void *table, flagcxDataType_t tabletype, size_t vocab, size_t dim,
                                    size_t tablestride, const void *ids, flagcxDataType_t idtype, size_t tokens,
                                    int64_t first, float scale, void *out, flagcxDataType_t outtype,
                                    size_t outstride, flagcxStream_t stream) {
  const char *who = "flagcxLocalEmbedding";
  const int tt = bitsOf(tabletype), ot = bitsOf(outtype), it = bitsOf(idtype);
  const uint32_t ts = (uint32_t)floatSize(tt), os = (uint32_t)floatSize(ot);
  if (!ts) return fail(flagcxInvalidArgument, "%s: unsupported tabletype %d", who, tt);
  if (!os || (ot != tt && ot != flagcxFloat32 && tt != flagcxFloat32))
    return fail(flagcxInvalidArgument, "%s: unsupported outtype %d", who, ot);
  if (it != flagcxInt32 && it != flagcxInt64) return fail(flagcxInvalidArgument, "%s: unsupported idtype %d", who, it);
  if (tokens == 0 || dim == 0) return flagcxSuccess;
  if (!out || !ids || (!table && vocab)) return fail(flagcxInvalidArgument, "%s: NULL argument", who);
  if (dim >> 31 || tokens >> 40) return fail(flagcxInvalidArgument, "%s: dim %zu or tokens %zu too large", who, dim, tokens);
  EmbedCall c{};
  Args a(who);
  c.table = table;
  c.vocab = vocab;
  c.tableStride = a.add("table", table, vocab, dim, tablestride, ts, false, false);
  c.ids = ids;
  c.wideIds = it == flagcxInt64;
  a.add("ids", ids, 1, tokens, 0, c.wideIds ? 8 : 4, false, false, false);
  c.out = out;
  c.outStride = a.add("out", out, tokens, dim, outstride, os, true, false);
  const flagcxResult_t r = a.check();
  if (r != flagcxSuccess) return r;
  c.dim = dim;
  c.tokens = tokens;
  c.first = first;
  c.scale = scale;
  c.vec = a.vec && dim * (ts < os ? ts : os) % 16 == 0;
  return finish(stream, launchEmbedding(c, tt, ot, hipStreamOf(stream)), who);
}

flagcxResult_t flagcxLocalEmbeddingGradWorkspace(size_t tokens, size_t vocab, size_t dim, size_t *bytes) {
  const char *who = "flagcxLocalEmbeddingGradWorkspace";
  if (!bytes) return fail(flagcxInvalidArgument, "%s: bytes is NULL", who);
  if (tokens >> 31 || vocab >> 31 || dim >> 31)
    return fail(flagcxInvalidArgument, "%s: tokens %zu, vocab %zu or dim %zu too large", who, tokens, vocab, dim);
  *bytes = tokens && vocab && dim ? (size_t)embedGradWorkspace(tokens, vocab, dim) : 0;
  return flagcxSuccess;
}

flagcxResult_t flagcxLocalEmbeddingGrad(const void *outgrad, flagcxDataType_t outtype, size_t outstride,
                                        const void *ids, flagcxDataType_t idtype, size_t tokens, int64_t first,
                                        float scale, void *tablegrad, flagcxDataType_t tabletype, size_t vocab,
                                        size_t dim, size_t tablestride, int accumulate,
                                        void *workspace, size_t workspacebytes, flagcxStream_t stream) {
  const char *who = "flagcxLocalEmbeddingGrad";
  const int tt = bitsOf(tabletype), ot = bitsOf(outtype), it = bitsOf(idtype);
  const uint32_t ts = (uint32_t)floatSize(tt), os = (uint32_t)floatSize(ot);
  if (!ts) return fail(flagcxInvalidArgument, "%s: unsupported tabletype %d", who, tt);
  if (!os || (ot != tt && ot != flagcxFloat32 && tt != flagcxFloat32))
    return fail(flagcxInvalidArgument, "%s: unsupported outtype %d", who, ot);
  if (it != flagcxInt32 && it != flagcxInt64) return fail(flagcxInvalidArgument, "%s: unsupported idtype %d", who, it);
  size_t need = 0;
  flagcxResult_t r = flagcxLocalEmbeddingGradWorkspace(tokens, vocab, dim, &need);
  if (r != flagcxSuccess) return r;
  if (vocab == 0 || dim == 0 || (tokens == 0 && accumulate)) return flagcxSuccess;
  if (!tablegrad || (tokens && (!outgrad || !ids))) return fail(flagcxInvalidArgument, "%s: NULL argument", who);
  if (need && !workspace) return fail(flagcxInvalidArgument, "%s: workspace is NULL", who);
  if ((uintptr_t)workspace % 16) return fail(flagcxInvalidArgument, "%s: workspace not aligned to 16", who);
  if (workspacebytes < need) return fail(flagcxInvalidArgument, "%s: workspace of %zu bytes, %zu are needed", who, workspacebytes, need);
  EmbedGradCall c{};
  Args a(who);
  c.grad = outgrad;
  c.gradStride = a.add("outgrad", outgrad, tokens, dim, outstride, os, false, false);
  c.ids = ids;
  c.wideIds = it == flagcxInt64;
  a.add("ids", ids, tokens ? 1 : 0, tokens, 0, c.wideIds ? 8 : 4, false, false, false);
  c.table = tablegrad;
  c.tableStride = a.add("tablegrad", tablegrad, vocab, dim, tablestride, ts, true, false);
  if (need) a.add("workspace", workspace, 1, need, 0, 1, true, false, false);
  if ((r = a.check()) != flagcxSuccess) return r;
  c.dim = dim;
  c.tokens = tokens;
  c.vocab = vocab;
  c.first = first;
  c.scale = scale;
  c.accumulate = accumulate != 0;
  c.workspace = workspace;
  c.vec = a.vec && dim * (ts < os ? ts : os) % 16 == 0;
  return finish(stream, launchEmbeddingGrad(c, ot, tt, hipStreamOf(stream)), who);
}

} // extern "C"
#pragma GCC visibility pop
