// Launchers of the language-model operators (rmsnorm.hip, ffn.hip, xent.hip,
// clip.hip): checks of arguments, choice of kernel and geometry, workspaces.  The
// entry points are documented in include/hc_amd_runtime.h.
#include "hc_amd_runtime.h"
#include "internal.h"
#include "kernels/op_args.h"

#include <algorithm>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <functional>
#include <utility>
#include <vector>

using namespace hcamd;

namespace {

constexpr size_t kMaxDim = 0x7fffff00; // sizes are held in 32 bits, tiles may run past an edge

inline size_t ceilDiv(size_t a, size_t b) { return (a + b - 1) / b; }
inline size_t alignUp(size_t a, size_t b) { return ceilDiv(a, b) * b; }
inline size_t elemBytes(int type) { return type == HCAMD_F32 ? 4 : type == HCAMD_I8 ? 1 : 2; }
inline const char *typeName(int type) {
  return type == HCAMD_F32 ? "f32" : type == HCAMD_F16 ? "f16" : type == HCAMD_BF16 ? "bf16" : "i8";
}
inline bool half16(int type) { return type == HCAMD_F16 || type == HCAMD_BF16; }

// rows that do not all begin at a multiple of 4 bytes
bool oddRows(const void *p, size_t ld, size_t bytes) {
  return reinterpret_cast<uintptr_t>(p) % 4 != 0 || ld * bytes % 4 != 0;
}

// One operand of a call: what the checks look at.
struct Arg {
  const char *name;
  const void *p;
  size_t ld, rows, cols, bytes; // bytes: of an element
};

struct Call {
  OlQueue q;
  const char *who;

  int fail(const char *fmt, ...) const __attribute__((format(printf, 2, 3))) {
    char text[200];
    va_list ap;
    va_start(ap, fmt);
    std::vsnprintf(text, sizeof(text), fmt, ap);
    va_end(ap);
    hcamdInternalReport(q, "%s: %s", who, text);
    return 1;
  }
  int check(const Arg &a) const {
    if (!a.p)
      return fail("%s is null", a.name);
    if (reinterpret_cast<uintptr_t>(a.p) % a.bytes)
      return fail("%s is not aligned to its elements", a.name);
    if (a.rows > 1 && a.ld < a.cols)
      return fail("%s: leading dimension smaller than a row", a.name);
    if (a.ld > ((size_t)1 << 40) || (a.rows > 1 && a.ld > ((size_t)1 << 46) / a.rows))
      return fail("%s: leading dimension out of range", a.name);
    return 0;
  }
  int checkAll(std::initializer_list<Arg> all) const {
    for (const Arg &a : all)
      if (check(a))
        return 1;
    return 0;
  }
  // outputs that begin where another one or an input does
  int apart(std::initializer_list<const void *> outputs, std::initializer_list<const void *> inputs) const {
    for (auto o = outputs.begin(); o != outputs.end(); ++o) {
      if (!*o)
        continue;
      for (auto p = outputs.begin(); p != o; ++p)
        if (*p == *o)
          return fail("two outputs are one buffer");
      for (const void *i : inputs)
        if (i == *o)
          return fail("an output is an input's buffer");
    }
    return 0;
  }
  // an output that may be this input, row for row
  int inPlace(const void *out, size_t ldo, const void *in, size_t ldi, size_t rows) const {
    return out && out == in && ldo != ldi && rows > 1 ? fail("in place with another leading dimension") : 0;
  }
  int work(const void *work, size_t have, size_t need) const {
    if (need == 0)
      return 0;
    if (!work || have < need)
      return fail("workspace of %zu bytes, %zu needed", work ? have : 0, need);
    if (reinterpret_cast<uintptr_t>(work) % 256)
      return fail("the workspace is not aligned to 256 bytes");
    return 0;
  }
  template <class T>
  int launch(const char *module, const char *kernel, T &args, size_t x, size_t y = 1, size_t z = 1,
             size_t threads = 256) const {
    if (x > 0x7fffff || y > 65535 || z > 65535)
      return fail("%zu x %zu x %zu workgroups", x, y, z);
    void *ptrs[] = {&args};
    return hcamdInternalLaunch(q, module, kernel, x, y, z, threads, ptrs);
  }
};

// ---- tiled products -----------------------------------------------------------
// Tile and splits of a product, from its shape alone (a workspace is sized before any
// pointer is seen): the cheapest by a model of the card's 256 compute units (with fewer of
// them the choice is less good, the results are the same).  Its unit is
// what a 256 x 256 tile takes for one k tile, 1.65 us at the 1.3 PFLOP/s those kernels
// reach; measured beside it: two 128 x 128 tiles on a unit 0.64, one alone 0.4, half a
// 256 x 256 tile 0.55; a tile's beginning and end cost about three k tiles; fp32 partial
// sums move at 4 TB/s and their folding is one more launch (5 us).
constexpr size_t kUnits = 256;
struct Product {
  int tile; // 256 or 128
  int splits;
  double groups, steps, fold, cost; // of the model: workgroups, k tiles of each, folding, all
};
size_t padCols(size_t n) { return alignUp(n, 8); }
// units of time of `groups` workgroups that each hold one tile's share of k
double roundsOf(int tile, size_t groups) {
  if (tile == 128) {
    const size_t rem = groups % (2 * kUnits);
    return 0.64 * (groups / (2 * kUnits)) + (rem == 0 ? 0.0 : rem <= kUnits ? 0.4 : 0.64);
  }
  const size_t rem = groups % kUnits;
  return (double)(groups / kUnits) + (rem == 0 ? 0.0 : rem <= kUnits / 2 ? 0.55 : 1.0);
}
// `products` of one shape in one launch; maxSplits 1: the k of a tile stays with one
// workgroup; only: this tile size (0: either)
Product productOf(size_t m, size_t n, size_t k, int segments, size_t products, size_t maxSplits, int only = 0) {
  const int v = hcamdInternalVariant("mma");
  const size_t kTiles = ceilDiv(k, (size_t)64) * segments;
  Product best{128, 1, 0, 0, 0, 1e300};
  for (int tile : {128, 256}) {
    if ((tile == 256 && (m < 256 || n < 256 || v == 2)) || (tile == 128 && v == 3 && m >= 256 && n >= 256) ||
        (only && tile != only))
      continue;
    const size_t tiles = ceilDiv(m, tile) * ceilDiv(n, tile) * products;
    for (size_t s = 1; s <= maxSplits && (s == 1 || kTiles / s >= 4); s *= 2) {
      const double bytes = s > 1 ? (double)s * m * padCols(n) * 4 * products : 0.0;
      if (bytes > (double)((size_t)128 << 20) * products)
        break;
      // (split tiles are not halved)
      const double rounds = s > 1 && tile == 256 ? (double)ceilDiv(tiles * s, kUnits) : roundsOf(tile, tiles * s);
      const double steps = (double)ceilDiv(kTiles, s) + 3.0, fold = s > 1 ? (2 * bytes / 8e12 * 1e6 + 5.0) / 1.65 : 0.0;
      if (rounds * steps + fold < best.cost)
        best = {tile, (int)s, (double)(tiles * s), steps, fold, rounds * steps + fold};
    }
  }
  return best;
}
// dx and dW: with 128 x 128 tiles they go in one launch, which saves 2.4 units and lets either
// fill the places that the other leaves, for as long as the card holds most of them at once
// (us apart / together: loss 300 x 1000 x 5000 bf16 backward, 704 workgroups 45 / 38; 300 x
// 1000 x 20000, 1640 of them 100 / 91; block 1000 x 2224 x 5000, 2016 of them 155 / 168).
void pairOf(Product &dx, Product &dw, const Product &dx128, const Product &dw128) {
  const double work = dx128.groups * dx128.steps + dw128.groups * dw128.steps;
  const double together = std::max(0.64 / (2 * kUnits) * work, 0.64 * std::max(dx128.steps, dw128.steps)) +
                          dx128.fold + dw128.fold;
  if (hcamdInternalVariant("mma") == 0 && dx128.groups + dw128.groups <= 3.5 * 2 * kUnits &&
      together < dx.cost + dw.cost + 2.4)
    dx = dx128, dw = dw128;
}
constexpr size_t kMaxSplits = 64;
size_t partialBytes(const Product &p, size_t m, size_t n) {
  return p.splits > 1 ? alignUp((size_t)p.splits * m * padCols(n) * 4, 256) : 0;
}

// Whether the pipelined kernels can fetch an operand: 16-byte pieces, offsets inside a
// tile (of up to 256 rows, in 32 bits) below 2^31: asked for every operand, the library's own
// too, whose rows are as long as the block is wide or a piece of the vocabulary.  `along` is
// its extent in the direction that runs through memory (k for a k-fast operand, its rows
// for a k-slow one); the library's own buffers are padded there.
bool fetchable(const void *p, size_t ld, size_t along, size_t bytes, bool padded) {
  const size_t piece = 16 / bytes;
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % piece == 0 && (padded || along % piece == 0) &&
         ld * bytes < ((size_t)1 << 23);
}
// The kernel of a product: "general", "half" (the same with 64 rows), "t128" or "t256".  The
// variant family "mma" (0: by size) asks for one of them where the operands allow it: 1
// general, 2 t128, 3 t256, 4 one pass over the weights up to 128 tokens, 5 half (forward).
struct Kernel {
  const char *suffix;
  size_t threads;
  int tile;
  int rows; // of a tile
};
// (fewM: a k-fast A may have fewer rows than the tile)
Kernel kernelOf(int tile, size_t m, size_t n, bool fetch, bool fewM) {
  if (!fetch || hcamdInternalVariant("mma") == 1 || (m < 128 && !fewM) || n < 128)
    return {"general", 256, 128, 128};
  if (tile == 256 && m >= 256 && n >= 256)
    return {"t256", 512, 256, 256};
  return {"t128", 256, 128, 128};
}
// A product with weights, whose tiles take as many columns as there are: while 64 x 128 tiles
// fill the card no more than once they take less time than 128 x 128 ones on half of it (48
// tokens, 2 x 11264 x 4096 bf16: 30 us against 43 us; 500 x 1001 x 1001 fp16 13 against 19;
// where they need a second round 333 x 1001 x 2731 21 against 18.4).
Kernel forwardKernel(size_t m, size_t n, size_t k, bool fetch) {
  Kernel kernel = kernelOf(productOf(m, n, k, 1, 1, 1).tile, m, n, fetch, true);
  const int v = hcamdInternalVariant("mma");
  if ((v == 0 && kernel.tile == 128 && ceilDiv(m, 64) * ceilDiv(n, 128) <= kUnits) || v == 5)
    kernel = {"half", 256, 128, 64};
  return kernel;
}
// The workgroups of `tiles` tiles: a last round of 256 x 256 tiles that fills at most half
// the card is worked in halves, from `halfFrom` on.
size_t groupsOf(const Kernel &k, size_t tiles, int splits, int &halfFrom) {
  const size_t rem = tiles % kUnits;
  const bool halves = k.tile == 256 && splits == 1 && rem != 0 && rem <= kUnits / 2;
  halfFrom = halves ? (int)(tiles - rem) : 0x7fffffff;
  return halves ? tiles + rem : tiles;
}

// Few tokens: the products with the weights as one pass over them.  Up to 32 tokens always:
// the tiles feed that pass from too few workgroups (one token, 2 x 11264 x 4096 bf16: 35 us
// against 65 us).  Up to 128 where it is estimated to take less time: its workgroups read
// every token's row again, altogether 8.4 TB/s (a workgroup at most 36 KB a us, odd rows
// 1.6 times as long), the tiles take 0.42 us for each k tile while 64 x 128 ones fit the
// card, 0.66 us while 128 x 128 ones do, more from odd rows.  (In tiles / so: 64 x 1000 x 2000
// bf16 11 / 5.9 us; 100 x 1001 x 2001 13 / 12; 64 x 2232 x 5000 19 / 22; 64 x 4096 x 11264 31 / 69;
// loss 64 x 1001 x 1500 17 / 12, 64 x 1000 x 20000 22 / 24.)  Null: in tiles.
// rows: of the weights, 32 to a workgroup; k: elements of a row; tileGroups: workgroups in
// 128 x 128 tiles.
constexpr size_t kFewTokens = 32, kMostFewTokens = 128;
const char *fewOf(size_t tokens, size_t rows, size_t k, size_t bytes, size_t tileGroups, bool odd) {
  const int v = hcamdInternalVariant("mma");
  if (tokens > kMostFewTokens || (v >= 1 && v <= 3) || v == 5)
    return nullptr;
  if (tokens > kFewTokens && v != 4) {
    const double groups = (double)ceilDiv(rows, 32), share = (tokens <= 64 ? 96.0 : 160.0) * k * bytes;
    const double few = 3.5 * std::max(1.0, groups / (2 * kUnits)) +
                       (odd ? 1.6 : 1.0) * std::max(groups * share / 8.4e6, share / 3.6e4);
    const double kTiles = (double)ceilDiv(k * bytes, 128);
    const double tiles = ceilDiv(tokens, 64) * tileGroups <= kUnits
                             ? 4.0 + (odd ? 0.55 : 0.42) * kTiles
                             : (odd ? 1.5 : 1.0) * 1.65 * roundsOf(128, tileGroups) * (kTiles + 3.0);
    if (few >= tiles)
      return nullptr;
  }
  return tokens <= 16   ? (odd ? "s16odd" : "s16")
         : tokens <= 32 ? (odd ? "s32odd" : "s32")
         : tokens <= 64 ? (odd ? "s64odd" : "s64")
                        : (odd ? "s128odd" : "s128");
}
constexpr size_t kFewOutputs = 16; // of the gated block to a workgroup
size_t fewColumns(size_t tokens) { return tokens <= kFewTokens ? 64 : 32; } // of the loss to a workgroup

// Products over rows whose length is not a multiple of 16 bytes.  The general kernel reads
// them as they lie; with enough tokens a copy in rows that the pipelined kernels can fetch
// costs less than those kernels gain.  A backward pass reads its copies twice.  (us, as
// they lie / copied: block 500 x 2231 x 5001 bf16 forward 55 / 63, backward 121 / 111;
// 700 x 1001 x 2731 forward 29 / 32; 1000 x 2231 x 5001 83 / 75 and 202 / 169; 333 x 4085 x
// 11001 backward 300 / 309; loss 500 x 1025 x 50021 111 / 106 and 382 / 310, 300 x 1001 x
// 20001 backward 111 / 112.)
// Rows shorter than a piece are always copied: the general kernel reads whole pieces.
enum Pass { kForward, kBackward };
bool laidOut(Pass pass, size_t tokens, size_t d, size_t bytes) {
  return d * bytes < 16 || (tokens >= (pass == kForward ? 768 : 384) && d * bytes % 16 != 0);
}
size_t layBytes(size_t rows, size_t d, size_t bytes) { return alignUp(rows * alignUp(d * bytes, 16), 256); }
// The copies of a call, one launch for up to three of them.
struct Lays {
  LayJobs jobs{};
  size_t count = 0, most = 0;
  // p and ld become those of the copy at `to`
  void add(const void *&p, size_t &ld, void *to, size_t rows, size_t d, size_t bytes) {
    const size_t own = alignUp(d * bytes, 16) / bytes;
    jobs.job[count++] = {p, to, ld, own, (uint32_t)rows, (uint32_t)d};
    most = std::max(most, rows);
    p = to, ld = own;
  }
  int launch(const Call &c, size_t bytes) {
    const size_t n = count, groups = std::min<size_t>(ceilDiv(most, (size_t)4), 4096);
    count = most = 0;
    return n == 0 ? 0 : c.launch("ffn", bytes == 1 ? "hcamd_lay_out_1" : "hcamd_lay_out_2", jobs, groups, n);
  }
};

// The folds of a call, one launch for up to three of them.
struct Folds {
  FoldJobs jobs{};
  size_t count = 0, most = 0;
  void add(const FoldArgs &f) {
    jobs.job[count++] = f;
    most = std::max(most, (size_t)f.rows * ceilDiv(f.cols, 4));
  }
  int launch(const Call &c, int type) {
    if (count == 0)
      return 0;
    char name[64];
    std::snprintf(name, sizeof(name), "hcamd_fold_%s", typeName(type));
    const size_t n = count, groups = std::min<size_t>(ceilDiv(most, (size_t)256), 4096);
    count = most = 0;
    return c.launch("ffn", name, jobs, groups, n);
  }
};

// The products of a backward pass.  With 128 x 128 tiles both go in one launch.
struct Products {
  ProductsArgs args{};
  Kernel nn{}, tn{};
  size_t gn = 0, gt = 0; // workgroups of one split of each
  int launch(const Call &c, int type) {
    char name[64];
    const size_t sn = args.nn.mma.splits, st = args.tn.p[0].mma.splits;
    const bool resident = gn * sn + gt * st <= 2 * kUnits; // all at once: one launch beats the faster kernel
    if (gn && gt && nn.tile == 128 && tn.tile == 128 && resident && std::strcmp(nn.suffix, tn.suffix))
      nn.suffix = tn.suffix = "general";
    const bool together = gn && gt && nn.tile == 128 && tn.tile == 128 && !std::strcmp(nn.suffix, tn.suffix);
    for (int k = together ? 1 : 0; k < 2; ++k) {
      const Kernel &kernel = k ? tn : nn;
      if (!(k ? gt : gn))
        continue;
      if (kernel.tile == 256) {
        std::snprintf(name, sizeof(name), "hcamd_product_%s_%s_t256", k ? "tn" : "nn", typeName(type));
        if (k ? c.launch("ffn", name, args.tn, gt, st, 1, 512) : c.launch("ffn", name, args.nn, gn, sn, 1, 512))
          return 1;
        continue;
      }
      const size_t n = together || !k ? gn : 0, t = together || k ? gt : 0;
      if (n > 0x7fffff || t > 0x7fffff)
        return c.fail("%zu workgroups", std::max(n, t));
      args.nn_groups = (int)n, args.tn_groups = (int)t;
      std::snprintf(name, sizeof(name), "hcamd_products_%s_%s", typeName(type), kernel.suffix);
      if (c.launch("ffn", name, args, n * sn + t * st))
        return 1;
    }
    return 0;
  }
};

bool dimsOk(const Call &c, size_t a, size_t b, size_t d) {
  if (a > kMaxDim || b > kMaxDim || d > kMaxDim) {
    c.fail("a dimension exceeds 2^31 - 256");
    return false;
  }
  return true;
}

} // namespace

namespace {
// The kernel of a row length: as many lanes a row and 16-byte pieces a lane as hold it.  A
// wave to a row needs no barrier; longer rows take more lanes.  16-bit rows, whose values take
// twice their size in registers, do better with more lanes than with more pieces to a lane
// (4096 x 8192 bf16 with 1024 lanes: 45 us forward against 51 us, 50 against 58 us in 8 bits; the
// backward pass 58 us with 512 lanes, 62 us with 1024), fp32 rows do not.  From 257 to 512
// pieces too (8192 x 4096: 43 against 46 us, 4 rows 3.6 against 4.3), but many 8-bit rows do not
// (8192 x 3001 49 against 43 us; 512 x 3001 6.3 against 7.3), and from 65 to 128 pieces only
// up to 1024 rows forward (512 x 1000 3.6 against 4.5 us, 2000 x 1000 5.9 against 5.5).
// Rows beyond 1024 lanes x 2 pieces (fp32: x 4) are read twice by the general kernel.
enum RowPass { kRowForward, kRowTo8Bits, kRowBackward };
struct RowKernel {
  const char *suffix;
  size_t lanes, threads;
  bool general;
};
RowKernel rowKernel(int type, size_t rows, size_t cols, RowPass pass) {
  struct Entry {
    size_t pieces;
    RowKernel kernel;
  };
  static const Entry shortRows[] = {{64, {"r64v1", 64, 256, false}},
                                    {128, {"r64v2", 64, 256, false}},
                                    {256, {"r256v1", 256, 256, false}},
                                    {512, {"r256v2", 256, 256, false}}};
  static const Entry forward16[] = {{1024, {"r1024v1", 1024, 1024, false}}, {2048, {"r1024v2", 1024, 1024, false}}};
  static const Entry back16[] = {{1024, {"r512v2", 512, 512, false}}, {2048, {"r1024v2", 1024, 1024, false}}};
  static const Entry rows32[] = {{1024, {"r256v4", 256, 256, false}},
                                 {2048, {"r512v4", 512, 512, false}},
                                 {4096, {"r1024v4", 1024, 1024, false}}};
  const size_t need = ceilDiv(cols, 16 / elemBytes(type));
  if (hcamdInternalVariant("rmsnorm") == 1)
    return {"general", 256, 256, true};
  const bool half = type != HCAMD_F32;
  if (half && pass != kRowBackward && rows <= 4 * kUnits && need > 64 && need <= 128)
    return shortRows[2].kernel;
  if (half && need > 256 && need <= 512 && (pass != kRowTo8Bits || rows <= 2 * kUnits))
    return {"r512v1", 512, 512, false};
  for (const Entry &e : shortRows)
    if (need <= e.pieces)
      return e.kernel;
  if (type == HCAMD_F32) {
    for (const Entry &e : rows32)
      if (need <= e.pieces)
        return e.kernel;
  } else {
    for (const Entry &e : pass == kRowBackward ? back16 : forward16)
      if (need <= e.pieces)
        return e.kernel;
  }
  return {"general", 256, 256, true};
}
// workgroups walk the rows: as many as fill the card
size_t rowGroups(OlQueue q, const RowKernel &k, size_t rows) {
  if (k.general)
    return std::min<size_t>(rows, 0x7fffff);
  return std::min(ceilDiv(rows, k.threads / k.lanes), (size_t)hcamdInternalComputeUnits(q) * 2048 / k.threads);
}
} // namespace

extern "C" {

// ===========================================================================
// add + RMS norm
// ===========================================================================
int hcamdLaunchAddRmsNorm(OlQueue q, int elemType, const void *x, size_t ldx, const void *residual, size_t ldr,
                          const void *weight, int weightType, float eps, void *summed, size_t lds, void *out,
                          int outType, size_t ldo, float *scale, float *rstd, size_t rows, size_t cols) noexcept {
  const Call c{q, "hcamdLaunchAddRmsNorm"};
  if (!q)
    return 1;
  if (elemType != HCAMD_F32 && !half16(elemType))
    return c.fail("element type %d (fp32, fp16, bf16)", elemType);
  if (outType != elemType && outType != HCAMD_I8)
    return c.fail("output type %d (the element type, or int8)", outType);
  if (weight && weightType != HCAMD_F32 && weightType != elemType)
    return c.fail("weight type %d (fp32, or the element type)", weightType);
  if (!(eps >= 0.0f))
    return c.fail("eps must not be negative");
  if (!dimsOk(c, rows, cols, 0))
    return 1;
  if (rows == 0)
    return 0;
  if (cols == 0)
    return c.fail("rows without elements");
  const size_t e = elemBytes(elemType);
  if (c.checkAll({{"x", x, ldx, rows, cols, e}, {"out", out, ldo, rows, cols, elemBytes(outType)}}) ||
      (residual && c.check({"residual", residual, ldr, rows, cols, e})) ||
      (weight && c.check({"weight", weight, cols, 1, cols, elemBytes(weightType)})) ||
      (summed && c.check({"summed", summed, lds, rows, cols, e})) ||
      (rstd && c.check({"rstd", rstd, rows, 1, rows, 4})))
    return 1;
  if (outType == HCAMD_I8 ? c.check({"scale", scale, rows, 1, rows, 4}) : scale != nullptr)
    return outType == HCAMD_I8 ? 1 : c.fail("a scale needs an int8 output");
  if (c.apart({out, summed, scale, rstd}, {weight}) || c.apart({scale, rstd}, {x, residual}) ||
      (outType != elemType && c.apart({out}, {x, residual})) || c.inPlace(out, ldo, x, ldx, rows) ||
      c.inPlace(out, ldo, residual, ldr, rows) || c.inPlace(summed, lds, x, ldx, rows) ||
      c.inPlace(summed, lds, residual, ldr, rows))
    return 1;
  NormArgs a{};
  a.x = x, a.residual = residual, a.weight = weight, a.summed = summed, a.out = out, a.scale = scale, a.rstd = rstd;
  a.ldx = ldx, a.ldr = ldr, a.lds = lds, a.ldo = ldo;
  a.rows = (uint32_t)rows, a.cols = (uint32_t)cols, a.eps = eps;
  a.weight_f32 = !weight || weightType == HCAMD_F32;
  const RowKernel k = rowKernel(elemType, rows, cols, outType == HCAMD_I8 ? kRowTo8Bits : kRowForward);
  char name[64];
  std::snprintf(name, sizeof(name), "hcamd_rmsnorm_%s%s_%s", typeName(elemType), outType == HCAMD_I8 ? "_i8" : "",
                k.suffix);
  return c.launch("rmsnorm", name, a, rowGroups(q, k, rows), 1, 1, k.threads);
}

namespace {
// lines of partial sums of the weight's gradient: enough workgroups to fill the card
size_t normBands(size_t rows) { return std::min<size_t>(rows, 512); }
} // namespace

size_t hcamdAddRmsNormBackwardWorkspace(size_t rows, size_t cols) noexcept {
  if (rows == 0 || rows > kMaxDim || cols > kMaxDim)
    return 0;
  return normBands(rows) * cols * 4;
}

int hcamdLaunchAddRmsNormBackward(OlQueue q, int elemType, const void *gradOut, size_t ldg, const void *summed,
                                  size_t lds, const void *weight, int weightType, const float *rstd,
                                  const void *gradSummed, size_t ldgs, void *gradIn, size_t ldgi, void *gradWeight,
                                  size_t rows, size_t cols, void *work, size_t workBytes) noexcept {
  const Call c{q, "hcamdLaunchAddRmsNormBackward"};
  if (!q)
    return 1;
  if (elemType != HCAMD_F32 && !half16(elemType))
    return c.fail("element type %d (fp32, fp16, bf16)", elemType);
  if (weightType != HCAMD_F32 && weightType != elemType)
    return c.fail("weight type %d (fp32, or the element type)", weightType);
  if (!dimsOk(c, rows, cols, 0))
    return 1;
  if (cols == 0)
    return rows == 0 ? 0 : c.fail("rows without elements");
  const size_t e = elemBytes(elemType), we = elemBytes(weightType);
  if (gradWeight && c.check({"grad_weight", gradWeight, cols, 1, cols, we}))
    return 1;
  if (rows && (c.checkAll({{"grad_out", gradOut, ldg, rows, cols, e},
                           {"summed", summed, lds, rows, cols, e},
                           {"rstd", rstd, rows, 1, rows, 4},
                           {"grad_in", gradIn, ldgi, rows, cols, e}}) ||
               (gradSummed && c.check({"grad_summed", gradSummed, ldgs, rows, cols, e})) ||
               (weight && c.check({"weight", weight, cols, 1, cols, we}))))
    return 1;
  NormBackArgs a{};
  a.grad_out = gradOut, a.summed = summed, a.weight = weight, a.grad_summed = gradSummed, a.rstd = rstd;
  a.grad_in = gradIn, a.grad_weight = gradWeight, a.partial = static_cast<float *>(work);
  a.ldg = ldg, a.ldh = lds, a.ldgs = ldgs, a.ldgi = ldgi;
  a.rows = (uint32_t)rows, a.cols = (uint32_t)cols, a.weight_f32 = weightType == HCAMD_F32;
  const RowKernel k = rowKernel(elemType, rows, cols, kRowBackward);
  const size_t lines = normBands(rows);
  char name[64];
  if (gradWeight && c.work(work, workBytes, hcamdAddRmsNormBackwardWorkspace(rows, cols)))
    return 1;
  if (rows && (c.apart({gradIn, gradWeight}, {summed, weight, rstd}) || c.apart({gradWeight}, {gradOut, gradSummed}) ||
               c.inPlace(gradIn, ldgi, gradOut, ldg, rows) || c.inPlace(gradIn, ldgi, gradSummed, ldgs, rows)))
    return 1;
  if (k.general) {
    // the weight's gradient first: grad_in may be grad_out
    a.band = (uint32_t)ceilDiv(rows, std::max<size_t>(lines, 1));
    a.bands = rows ? (uint32_t)ceilDiv(rows, a.band) : 0;
    std::snprintf(name, sizeof(name), "hcamd_rmsnorm_back_weight_%s_general", typeName(elemType));
    if (gradWeight && rows && c.launch("rmsnorm", name, a, ceilDiv(cols, 256), a.bands))
      return 1;
    std::snprintf(name, sizeof(name), "hcamd_rmsnorm_back_%s_general", typeName(elemType));
    if (rows && c.launch("rmsnorm", name, a, std::min<size_t>(rows, 0x7fffff)))
      return 1;
  } else if (rows) {
    a.bands = (uint32_t)std::min(ceilDiv(rows, k.threads / k.lanes), lines);
    std::snprintf(name, sizeof(name), "hcamd_rmsnorm_back_%s_%s", typeName(elemType), k.suffix);
    if (c.launch("rmsnorm", name, a, a.bands, 1, 1, k.threads))
      return 1;
  }
  if (!gradWeight)
    return 0;
  std::snprintf(name, sizeof(name), "hcamd_rmsnorm_fold_%s", typeName(weightType));
  return c.launch("rmsnorm", name, a, ceilDiv(cols, 64), 1, 1, 1024);
}

// ===========================================================================
// gated feed-forward block
// ===========================================================================
size_t hcamdGatedFfnWorkspace(int elemType, size_t tokens, size_t d, size_t f) noexcept {
  if (d == 0 || f == 0 || tokens > kMaxDim || d > kMaxDim || f > kMaxDim)
    return 0;
  const size_t e = elemBytes(elemType);
  return laidOut(kForward, tokens, d, e) ? layBytes(tokens, d, e) + 2 * layBytes(f, d, e) : 0;
}

int hcamdLaunchGatedFfn(OlQueue q, int elemType, const void *x, size_t ldx, const float *xScale, const void *wGate,
                        size_t ldwg, const float *gateScale, const void *wUp, size_t ldwu, const float *upScale,
                        int activation, void *out, int outType, size_t ldo, void *gate, size_t ldgate, void *up,
                        size_t ldup, size_t tokens, size_t d, size_t f, void *work, size_t workBytes) noexcept {
  const Call c{q, "hcamdLaunchGatedFfn"};
  if (!q)
    return 1;
  const bool i8 = elemType == HCAMD_I8;
  if (!i8 && !half16(elemType))
    return c.fail("element type %d (fp16, bf16, int8)", elemType);
  if (i8 ? !half16(outType) : outType != elemType)
    return c.fail("output type %d (the element type; fp16 or bf16 for int8)", outType);
  if (activation != HCAMD_SILU && activation != HCAMD_GELU)
    return c.fail("activation %d", activation);
  if (!dimsOk(c, tokens, d, f))
    return 1;
  if (tokens == 0 || f == 0)
    return 0;
  if (d == 0)
    return c.fail("the inner dimension must be at least 1");
  if (i8 && d >= 131072) // 2^17 products of 2^14 would be 2^31
    return c.fail("an inner dimension of %zu (int8 sums are exact below 131072)", d);
  const size_t e = elemBytes(elemType), oe = elemBytes(outType);
  if (c.checkAll({{"x", x, ldx, tokens, d, e}, {"w_gate", wGate, ldwg, f, d, e}, {"w_up", wUp, ldwu, f, d, e},
                  {"out", out, ldo, tokens, f, oe}}))
    return 1;
  if (i8) {
    if (gate || up)
      return c.fail("the pre-activations of an int8 product are not kept");
    if (c.checkAll({{"x_scale", xScale, tokens, 1, tokens, 4}, {"gate_scale", gateScale, f, 1, f, 4},
                    {"up_scale", upScale, f, 1, f, 4}}))
      return 1;
  } else {
    if (xScale || gateScale || upScale)
      return c.fail("scales belong to int8 operands");
    if ((gate && c.check({"gate", gate, ldgate, tokens, f, oe})) || (up && c.check({"up", up, ldup, tokens, f, oe})))
      return 1;
  }
  if (c.work(work, workBytes, hcamdGatedFfnWorkspace(elemType, tokens, d, f)) ||
      c.apart({out, gate, up}, {x, wGate, wUp, xScale, gateScale, upScale}))
    return 1;
  const bool lay = laidOut(kForward, tokens, d, e);
  if (lay) {
    char *w = static_cast<char *>(work);
    Lays l;
    l.add(x, ldx, w, tokens, d, e);
    l.add(wGate, ldwg, w + layBytes(tokens, d, e), f, d, e);
    l.add(wUp, ldwu, w + layBytes(tokens, d, e) + layBytes(f, d, e), f, d, e);
    if (l.launch(c, e))
      return 1;
  }
  GatedArgs a{};
  a.mma.a[0] = x, a.mma.lda[0] = ldx;
  a.mma.b[0] = wGate, a.mma.ldb[0] = ldwg, a.mma.b[1] = wUp, a.mma.ldb[1] = ldwu;
  a.mma.M = (int)tokens, a.mma.N = (int)f, a.mma.K = (int)d, a.mma.segments = 1, a.mma.splits = 1;
  a.x_scale = xScale, a.gate_scale = gateScale, a.up_scale = upScale;
  a.out = out, a.gate = gate, a.up = up, a.ldo = ldo, a.ldgate = ldgate, a.ldup = ldup;
  a.activation = activation, a.out_f16 = outType == HCAMD_F16;
  char name[64];
  if (const char *few = fewOf(tokens, 2 * f, d, e, ceilDiv(f, 64), oddRows(x, ldx, e) || oddRows(wGate, ldwg, e) || oddRows(wUp, ldwu, e))) {
    std::snprintf(name, sizeof(name), "hcamd_gated_%s_%s", typeName(elemType), few);
    return c.launch("ffn", name, a, ceilDiv(f, kFewOutputs), 1, 1, 512);
  }
  // (a tile of outputs takes twice its columns of the two weight matrices)
  const Kernel k = forwardKernel(tokens, 2 * f, i8 ? d / 2 : d,
                                 fetchable(x, ldx, d, e, lay) && fetchable(wGate, ldwg, d, e, lay) &&
                                     fetchable(wUp, ldwu, d, e, lay));
  std::snprintf(name, sizeof(name), "hcamd_gated_%s_%s", typeName(elemType), k.suffix);
  const size_t groups = groupsOf(k, ceilDiv(tokens, k.rows) * ceilDiv(f, k.tile / 2), 1, a.mma.half_from);
  return c.launch("ffn", name, a, groups, 1, 1, k.threads);
}

namespace {
// the workspace of the backward pass: fp16's scaling (what undoes it, the maxima it comes from), dg,
// du, then the partial sums of dx, then of the two weight gradients, then the copies of x, Wg
// and Wu
constexpr size_t kMosts = 1024, kFfnBackHead = 256 + kMosts * 4;
struct FfnBack {
  size_t ldd, dg, dx, dw, lay, bytes;
  Product px, pw;
};
FfnBack ffnBack(size_t tokens, size_t d, size_t f) {
  FfnBack b;
  b.ldd = padCols(f);
  b.dg = alignUp(tokens * b.ldd * 2, 256);
  b.px = productOf(tokens, d, f, 2, 1, kMaxSplits);
  b.pw = productOf(f, d, tokens, 1, 2, kMaxSplits);
  pairOf(b.px, b.pw, productOf(tokens, d, f, 2, 1, kMaxSplits, 128), productOf(f, d, tokens, 1, 2, kMaxSplits, 128));
  b.dx = partialBytes(b.px, tokens, d);
  b.dw = partialBytes(b.pw, f, d);
  b.lay = 2 * b.dg + b.dx + 2 * b.dw;
  b.bytes = kFfnBackHead + b.lay +
            (laidOut(kBackward, tokens, d, 2) ? layBytes(tokens, d, 2) + 2 * layBytes(f, d, 2) : 0);
  return b;
}
} // namespace

size_t hcamdGatedFfnBackwardWorkspace(size_t tokens, size_t d, size_t f) noexcept {
  if (tokens == 0 || d == 0 || f == 0 || tokens > kMaxDim || d > kMaxDim || f > kMaxDim)
    return 0;
  return ffnBack(tokens, d, f).bytes;
}

int hcamdLaunchGatedFfnBackward(OlQueue q, int elemType, const void *gradOut, size_t ldg, const void *x, size_t ldx,
                                const void *wGate, size_t ldwg, const void *wUp, size_t ldwu, const void *gate,
                                size_t ldgate, const void *up, size_t ldup, int activation, void *gradX, size_t ldgx,
                                void *gradWGate, size_t ldgwg, void *gradWUp, size_t ldgwu, size_t tokens, size_t d,
                                size_t f, void *work, size_t workBytes) noexcept {
  const Call c{q, "hcamdLaunchGatedFfnBackward"};
  if (!q)
    return 1;
  if (!half16(elemType))
    return c.fail("element type %d (fp16, bf16)", elemType);
  if (activation != HCAMD_SILU && activation != HCAMD_GELU)
    return c.fail("activation %d", activation);
  if (!dimsOk(c, tokens, d, f))
    return 1;
  if (d == 0 || f == 0)
    return c.fail("an empty dimension (%zu, %zu)", d, f);
  if (tokens == 0)
    gradX = nullptr; // no rows; the weights' gradients are zeros
  if (tokens && c.checkAll({{"grad_out", gradOut, ldg, tokens, f, 2}, {"gate", gate, ldgate, tokens, f, 2},
                            {"up", up, ldup, tokens, f, 2}}))
    return 1;
  if (gradX && c.checkAll({{"w_gate", wGate, ldwg, f, d, 2}, {"w_up", wUp, ldwu, f, d, 2},
                           {"grad_x", gradX, ldgx, tokens, d, 2}}))
    return 1;
  if (tokens && (gradWGate || gradWUp) && c.check({"x", x, ldx, tokens, d, 2}))
    return 1;
  if ((gradWGate && c.check({"grad_w_gate", gradWGate, ldgwg, f, d, 2})) ||
      (gradWUp && c.check({"grad_w_up", gradWUp, ldgwu, f, d, 2})))
    return 1;
  const FfnBack b = ffnBack(tokens, d, f);
  if ((tokens && c.work(work, workBytes, b.bytes)) ||
      c.apart({gradX, gradWGate, gradWUp}, {gradOut, x, wGate, wUp, gate, up}))
    return 1;
  if (!gradX && !gradWGate && !gradWUp)
    return 0;
  char *w = static_cast<char *>(work) + kFfnBackHead;
  char name[64];
  GatedBackArgs e{};
  e.undo = static_cast<float *>(work), e.most = e.undo + 64;
  const float *undo = tokens && elemType == HCAMD_F16 ? e.undo : nullptr;
  e.grad_out = gradOut, e.gate = gate, e.up = up, e.dgate = w, e.dup = w + b.dg;
  e.ldg = ldg, e.ldgate = ldgate, e.ldup = ldup, e.ldd = b.ldd;
  e.rows = (uint32_t)tokens, e.cols = (uint32_t)f, e.activation = activation;
  const size_t eights = ceilDiv(tokens * ceilDiv(f, 8), 256);
  e.mosts = (uint32_t)std::min(eights, kMosts);
  if (undo && c.launch("ffn", "hcamd_gated_back_most_f16", e, e.mosts))
    return 1;
  std::snprintf(name, sizeof(name), "hcamd_gated_back_%s", typeName(elemType));
  if (tokens && c.launch("ffn", name, e, std::min<size_t>(eights, 8192)))
    return 1;
  const bool lay = tokens && laidOut(kBackward, tokens, d, 2);
  if (lay) {
    char *to = w + b.lay;
    Lays l;
    if (gradWGate || gradWUp)
      l.add(x, ldx, to, tokens, d, 2);
    if (gradX) {
      l.add(wGate, ldwg, to + layBytes(tokens, d, 2), f, d, 2);
      l.add(wUp, ldwu, to + layBytes(tokens, d, 2) + layBytes(f, d, 2), f, d, 2);
    }
    if (l.launch(c, 2))
      return 1;
  }
  Folds folds;
  Products products;
  if (gradX) {
    StoreArgs &s = products.args.nn;
    s.mma.a[0] = e.dgate, s.mma.a[1] = e.dup, s.mma.lda[0] = s.mma.lda[1] = b.ldd;
    s.mma.b[0] = wGate, s.mma.b[1] = wUp, s.mma.ldb[0] = ldwg, s.mma.ldb[1] = ldwu;
    s.mma.M = (int)tokens, s.mma.N = (int)d, s.mma.K = (int)f, s.mma.segments = 2, s.mma.splits = b.px.splits;
    s.out = gradX, s.ldo = ldgx, s.ldp = padCols(d), s.undo = undo;
    s.partial = b.dx ? reinterpret_cast<float *>(w + 2 * b.dg) : nullptr;
    products.nn = kernelOf(b.px.tile, tokens, d,
                           fetchable(w, b.ldd, f, 2, true) && fetchable(wGate, ldwg, d, 2, lay) &&
                               fetchable(wUp, ldwu, d, 2, lay),
                           true);
    products.gn = groupsOf(products.nn, ceilDiv(tokens, products.nn.tile) * ceilDiv(d, products.nn.tile),
                                            b.px.splits, s.mma.half_from);
    if (s.partial)
      folds.add({s.partial, gradX, s.ldp, ldgx, (uint32_t)tokens, (uint32_t)d, (uint32_t)b.px.splits, undo});
  }
  if (gradWGate || gradWUp) {
    PairStoreArgs &s = products.args.tn;
    size_t n = 0;
    for (int k = 0; k < 2; ++k) {
      void *to = k ? gradWUp : gradWGate;
      if (!to)
        continue;
      StoreArgs &t = s.p[n];
      t.mma.a[0] = k ? e.dup : e.dgate, t.mma.lda[0] = b.ldd;
      t.mma.b[0] = x, t.mma.ldb[0] = ldx;
      t.mma.M = (int)f, t.mma.N = (int)d, t.mma.K = (int)tokens, t.mma.segments = 1, t.mma.splits = b.pw.splits;
      t.out = to, t.ldo = k ? ldgwu : ldgwg, t.ldp = padCols(d), t.undo = undo;
      t.partial = b.dw ? reinterpret_cast<float *>(w + 2 * b.dg + b.dx + n * b.dw) : nullptr;
      ++n;
    }
    products.tn = kernelOf(b.pw.tile, f, d, fetchable(w, b.ldd, f, 2, true) && fetchable(x, ldx, d, 2, lay), false);
    s.tiles = (int)(ceilDiv(f, products.tn.tile) * ceilDiv(d, products.tn.tile));
    products.gt = groupsOf(products.tn, s.tiles * n, b.pw.splits, s.p[0].mma.half_from);
    for (size_t k = 0; b.dw && k < n; ++k)
      folds.add({s.p[k].partial, s.p[k].out, s.p[k].ldp, s.p[k].ldo, (uint32_t)f, (uint32_t)d, (uint32_t)b.pw.splits,
                 undo});
  }
  if (products.launch(c, elemType))
    return 1;
  return folds.launch(c, elemType);
}

// ===========================================================================
// linear cross entropy
// ===========================================================================
namespace {
// columns of the narrowest statistics tile
size_t statsCols(size_t tokens) { return tokens <= kMostFewTokens ? fewColumns(tokens) : 128; }
int xentCommon(const Call &c, int elemType, const void *x, size_t ldx, const void *weight, size_t ldw,
               const void *targets, int targetType, size_t tokens, size_t d, size_t vocab) {
  if (!half16(elemType))
    return c.fail("element type %d (fp16, bf16)", elemType);
  if (targetType != HCAMD_I32 && targetType != HCAMD_I64)
    return c.fail("target type %d (int32, int64)", targetType);
  if (!dimsOk(c, tokens, d, vocab))
    return 1;
  if (d == 0 || vocab == 0)
    return c.fail("an empty dimension (%zu, vocabulary of %zu)", d, vocab);
  return tokens && c.checkAll({{"x", x, ldx, tokens, d, 2}, {"weight", weight, ldw, vocab, d, 2},
                               {"targets", targets, tokens, 1, tokens, targetType == HCAMD_I64 ? 8u : 4u}});
}
} // namespace

namespace {
// The workspace of the forward pass: the tiles' statistics and the targets' logits, then the
// copies of x and of a piece of the weight.  Without copies the vocabulary is one piece;
// with them a piece holds 64 Mi elements, so that its copy mostly stays in the 256 MiB
// memory-side cache, and 4096 rows at least.
struct XentFront {
  size_t piece, stats, bytes;
  bool lay;
};
XentFront xentFront(size_t tokens, size_t d, size_t vocab) {
  XentFront b;
  b.lay = laidOut(kForward, tokens, d, 2);
  b.stats = tokens * ceilDiv(vocab, statsCols(tokens)) * 8 + tokens * 4;
  b.piece = vocab;
  b.bytes = b.stats;
  if (b.lay) {
    b.piece = std::min(vocab, std::max<size_t>(((size_t)64 << 20) / d / 256 * 256, 4096));
    b.stats = alignUp(b.stats, 256);
    b.bytes = b.stats + layBytes(tokens, d, 2) + layBytes(b.piece, d, 2);
  }
  return b;
}
} // namespace

size_t hcamdLinearCrossEntropyWorkspace(size_t tokens, size_t d, size_t vocab) noexcept {
  if (tokens > kMaxDim || d > kMaxDim || vocab > kMaxDim || d == 0)
    return 0;
  return xentFront(tokens, d, vocab).bytes;
}

int hcamdLaunchLinearCrossEntropy(OlQueue q, int elemType, const void *x, size_t ldx, const void *weight, size_t ldw,
                                  const void *targets, int targetType, float *loss, float *lse, size_t tokens,
                                  size_t d, size_t vocab, void *work, size_t workBytes) noexcept {
  const Call c{q, "hcamdLaunchLinearCrossEntropy"};
  if (!q || xentCommon(c, elemType, x, ldx, weight, ldw, targets, targetType, tokens, d, vocab))
    return 1;
  if (tokens == 0)
    return 0;
  const XentFront b = xentFront(tokens, d, vocab);
  if (c.checkAll({{"loss", loss, tokens, 1, tokens, 4}, {"lse", lse, tokens, 1, tokens, 4}}) ||
      c.work(work, workBytes, b.bytes) || c.apart({loss, lse}, {x, weight, targets}))
    return 1;
  char *w = static_cast<char *>(work);
  const char *few = fewOf(tokens, vocab, d, 2, ceilDiv(vocab, 128), oddRows(x, ldx, 2) || oddRows(weight, ldw, 2));
  Lays lays;
  if (b.lay)
    lays.add(x, ldx, w + b.stats, tokens, d, 2);
  XentArgs a{};
  a.targets = targets, a.target_i64 = targetType == HCAMD_I64, a.vocab = (int)vocab;
  const bool fetch = fetchable(x, ldx, d, 2, b.lay) &&
                     (b.lay ? fetchable(w, padCols(d), d, 2, true) : fetchable(weight, ldw, d, 2, false));
  for (size_t v0 = 0; v0 < vocab; v0 += b.piece) {
    const size_t n = std::min(b.piece, vocab - v0);
    a.tiles += (int)ceilDiv(n, few ? fewColumns(tokens) : forwardKernel(tokens, n, d, fetch).tile);
  }
  a.stats = reinterpret_cast<float *>(w);
  a.zt = a.stats + tokens * a.tiles * 2;
  char name[64];
  for (size_t v0 = 0; v0 < vocab; v0 += b.piece) {
    const size_t n = std::min(b.piece, vocab - v0);
    const void *rows = static_cast<const char *>(weight) + v0 * ldw * 2;
    size_t ldr = ldw;
    if (b.lay) {
      lays.add(rows, ldr, w + b.stats + layBytes(tokens, d, 2), n, d, 2);
      if (lays.launch(c, 2))
        return 1;
    }
    const Kernel k = forwardKernel(tokens, n, d, fetch);
    const size_t tiles = ceilDiv(n, few ? fewColumns(tokens) : k.tile);
    a.mma.a[0] = x, a.mma.lda[0] = ldx, a.mma.b[0] = rows, a.mma.ldb[0] = ldr;
    a.mma.M = (int)tokens, a.mma.N = (int)n, a.mma.K = (int)d, a.mma.segments = a.mma.splits = 1;
    a.v0 = (int)v0;
    std::snprintf(name, sizeof(name), "hcamd_xent_stats_%s_%s", typeName(elemType), few ? few : k.suffix);
    const size_t groups = few ? tiles : groupsOf(k, ceilDiv(tokens, k.rows) * tiles, 1, a.mma.half_from);
    if (c.launch("xent", name, a, groups, 1, 1, few ? 512 : k.threads))
      return 1;
    a.tile0 += (int)tiles;
  }
  XentRowsArgs r{a.stats, a.zt, targets, a.target_i64, loss, lse, (uint32_t)tokens, (uint32_t)vocab,
                 (uint32_t)a.tiles};
  return c.launch("xent", "hcamd_xent_rows", r, ceilDiv(tokens, 4));
}

namespace {
// the workspace of the backward pass: the factor, p of a piece, the partial sums of dx,
// the partial sums of a piece's dW, the rows of x that take part, a copy of the piece's
// rows of W
struct XentBack {
  size_t piece, ldp, p, dx, dw, live, lay, bytes;
  Product px, pw;
};
XentBack xentBack(size_t tokens, size_t d, size_t vocab, size_t piece) {
  XentBack b;
  // by default a piece holds 64 Mi elements of p (128 MiB): what the two products of
  // the piece read again then mostly stays in the 256 MiB memory-side cache, and a
  // piece is work enough to fill the card
  if (piece == 0)
    piece = std::max<size_t>(alignUp(((size_t)64 << 20) / std::max<size_t>(tokens, 1), 256), 1024);
  b.piece = std::min(alignUp(piece, 8), vocab);
  b.ldp = padCols(b.piece);
  b.p = alignUp(tokens * b.ldp * 2, 256);
  b.px = productOf(tokens, d, b.piece, 1, 1, kMaxSplits);
  b.pw = productOf(b.piece, d, tokens, 1, 1, kMaxSplits);
  pairOf(b.px, b.pw, productOf(tokens, d, b.piece, 1, 1, kMaxSplits, 128),
         productOf(b.piece, d, tokens, 1, 1, kMaxSplits, 128));
  b.dx = alignUp((size_t)b.px.splits * tokens * padCols(d) * 4, 256);
  b.dw = partialBytes(b.pw, b.piece, d);
  b.live = alignUp(tokens * padCols(d) * 2, 256);
  b.lay = 256 + b.p + b.dx + b.dw + b.live;
  b.bytes = b.lay + (laidOut(kBackward, tokens, d, 2) ? layBytes(b.piece, d, 2) : 0);
  return b;
}
} // namespace

size_t hcamdLinearCrossEntropyBackwardWorkspace(size_t tokens, size_t d, size_t vocab, size_t piece) noexcept {
  if (tokens == 0 || d == 0 || vocab == 0 || tokens > kMaxDim || d > kMaxDim || vocab > kMaxDim || piece > kMaxDim)
    return 0;
  return xentBack(tokens, d, vocab, piece).bytes;
}

int hcamdLaunchLinearCrossEntropyBackward(OlQueue q, int elemType, const void *x, size_t ldx, const void *weight,
                                          size_t ldw, const void *targets, int targetType, const float *lse,
                                          const float *gradLoss, void *gradX, size_t ldgx, void *gradWeight,
                                          size_t ldgw, size_t tokens, size_t d, size_t vocab, size_t piece,
                                          void *work, size_t workBytes) noexcept {
  const Call c{q, "hcamdLaunchLinearCrossEntropyBackward"};
  if (!q || xentCommon(c, elemType, x, ldx, weight, ldw, targets, targetType, tokens, d, vocab))
    return 1;
  if (piece > kMaxDim)
    return c.fail("a piece of %zu rows", piece);
  if (tokens == 0)
    gradX = nullptr; // no rows; the weight's gradient is zero
  if ((tokens && c.checkAll({{"lse", lse, tokens, 1, tokens, 4}, {"grad_loss", gradLoss, tokens, 1, tokens, 4}})) ||
      (gradX && c.check({"grad_x", gradX, ldgx, tokens, d, 2})) ||
      (gradWeight && c.check({"grad_weight", gradWeight, ldgw, vocab, d, 2})))
    return 1;
  const XentBack b = xentBack(tokens, d, vocab, piece);
  if ((tokens && c.work(work, workBytes, b.bytes)) ||
      c.apart({gradX, gradWeight}, {x, weight, targets, lse, gradLoss}))
    return 1;
  if (!gradX && !gradWeight)
    return 0;
  char *w = static_cast<char *>(work);
  char name[64];
  float *factor = reinterpret_cast<float *>(w);
  const void *live = w + 256 + b.p + b.dx + b.dw;
  const bool lay = tokens && laidOut(kBackward, tokens, d, 2); // (without tokens there is no workspace, and nothing to read)
  if (tokens) {
    XentPrepareArgs a{};
    a.x = x, a.targets = targets, a.grad_loss = gradLoss, a.target_i64 = targetType == HCAMD_I64;
    a.top = elemType == HCAMD_F16 ? 0x1p15f : 1.0f, a.factor = factor;
    a.live_x = const_cast<void *>(live), a.ldx = ldx, a.ldl = padCols(d);
    a.rows = (uint32_t)tokens, a.cols = (uint32_t)d, a.vocab = (uint32_t)vocab;
    const size_t rest = gradWeight || lay ? std::min<size_t>(ceilDiv(tokens * ceilDiv(d, 8), 1024), 1024) : 0;
    if (c.launch("xent", "hcamd_xent_prepare", a, 1 + rest, 1, 1, 1024))
      return 1;
  }
  if (lay) // (the logits of rows that take no part are not looked at)
    x = live, ldx = padCols(d);
  const float *undo = tokens ? factor + 1 : nullptr;
  float *dx = reinterpret_cast<float *>(w + 256 + b.p);
  Folds folds;
  for (size_t v0 = 0; v0 < vocab; v0 += b.piece) {
    const size_t n = std::min(b.piece, vocab - v0);
    const void *rows = static_cast<const char *>(weight) + v0 * ldw * 2;
    size_t ldr = ldw;
    if (lay) {
      Lays l;
      l.add(rows, ldr, w + b.lay, n, d, 2);
      if (l.launch(c, 2))
        return 1;
    }
    XentArgs a{};
    a.mma.a[0] = x, a.mma.lda[0] = ldx, a.mma.b[0] = rows, a.mma.ldb[0] = ldr;
    a.mma.M = (int)tokens, a.mma.N = (int)n, a.mma.K = (int)d, a.mma.segments = a.mma.splits = 1;
    a.targets = targets, a.target_i64 = targetType == HCAMD_I64, a.v0 = (int)v0, a.vocab = (int)vocab;
    a.lse = lse, a.grad_loss = gradLoss, a.factor = factor, a.p = w + 256, a.ldp = b.ldp;
    const Kernel k = forwardKernel(tokens, n, d, fetchable(x, ldx, d, 2, lay) && fetchable(rows, ldr, d, 2, lay));
    const char *few = fewOf(tokens, n, d, 2, ceilDiv(n, 128), oddRows(x, ldx, 2) || oddRows(rows, ldr, 2));
    std::snprintf(name, sizeof(name), "hcamd_xent_p_%s_%s", typeName(elemType), few ? few : k.suffix);
    const size_t groups = few ? ceilDiv(n, fewColumns(tokens))
                        : groupsOf(k, ceilDiv(tokens, k.rows) * ceilDiv(n, k.tile), 1, a.mma.half_from);
    if (tokens && c.launch("xent", name, a, groups, 1, 1, few ? 512 : k.threads))
      return 1;
    Products products;
    if (gradX) {
      StoreArgs &s = products.args.nn;
      s.mma.a[0] = a.p, s.mma.lda[0] = b.ldp, s.mma.b[0] = rows, s.mma.ldb[0] = ldr;
      s.mma.M = (int)tokens, s.mma.N = (int)d, s.mma.K = (int)n, s.mma.segments = 1, s.mma.splits = b.px.splits;
      s.partial = dx, s.ldp = padCols(d), s.accumulate = v0 != 0;
      products.nn = kernelOf(b.px.tile, tokens, d, fetchable(a.p, b.ldp, n, 2, true) && fetchable(rows, ldr, d, 2, lay),
                             true);
      products.gn = groupsOf(
          products.nn, ceilDiv(tokens, products.nn.tile) * ceilDiv(d, products.nn.tile), b.px.splits, s.mma.half_from);
    }
    if (gradWeight) {
      StoreArgs &t = products.args.tn.p[0];
      t.mma.a[0] = a.p, t.mma.lda[0] = b.ldp, t.mma.b[0] = live, t.mma.ldb[0] = padCols(d);
      t.mma.M = (int)n, t.mma.N = (int)d, t.mma.K = (int)tokens, t.mma.segments = 1, t.mma.splits = b.pw.splits;
      t.out = static_cast<char *>(gradWeight) + v0 * ldgw * 2, t.ldo = ldgw, t.undo = undo;
      t.partial = b.dw ? reinterpret_cast<float *>(w + 256 + b.p + b.dx) : nullptr, t.ldp = padCols(d);
      products.tn = kernelOf(b.pw.tile, n, d,
                             fetchable(a.p, b.ldp, n, 2, true) && fetchable(live, padCols(d), d, 2, true), false);
      products.args.tn.tiles = (int)(ceilDiv(n, products.tn.tile) * ceilDiv(d, products.tn.tile));
      products.gt = groupsOf(products.tn, products.args.tn.tiles, b.pw.splits, t.mma.half_from);
      if (b.dw)
        folds.add({t.partial, t.out, t.ldp, ldgw, (uint32_t)n, (uint32_t)d, (uint32_t)b.pw.splits, undo});
    }
    if (products.launch(c, elemType))
      return 1;
    if (gradX && v0 + n == vocab)
      folds.add({dx, gradX, padCols(d), ldgx, (uint32_t)tokens, (uint32_t)d, (uint32_t)b.px.splits, undo});
    if (folds.launch(c, elemType)) // (the next piece writes the partial sums of dW again)
      return 1;
  }
  return 0;
}

// ===========================================================================
// clipping by the global norm
// ===========================================================================
namespace {
constexpr size_t kClipCells = 1024;
// elements to a chunk: small totals are cut finer, so that more workgroups share them
size_t clipChunk(size_t elems) { return elems >= ((size_t)16 << 20) ? 16384 : 4096; }
// workgroups of the launch that takes `chunks` of `all` chunks
size_t clipGroups(size_t chunks, size_t all) {
  return std::max<size_t>(1, std::min(chunks, all <= kClipCells ? chunks : chunks * kClipCells / all));
}
// Every clipped tensor is written once, over nothing that another workgroup reads: an output is
// neither another one nor another tensor's input, and the norm is none of them.
int clipApart(const Call &c, const HcamdClipTensor *tensors, size_t count, const float *norm) {
  std::vector<std::pair<const void *, size_t>> outs; // by address, with the tensor's index
  outs.reserve(count);
  for (size_t i = 0; i < count; ++i)
    if (tensors[i].count)
      outs.emplace_back(tensors[i].out, i);
  const std::less<const void *> below;
  std::sort(outs.begin(), outs.end(), [&](const auto &a, const auto &b) { return below(a.first, b.first); });
  for (size_t i = 1; i < outs.size(); ++i)
    if (outs[i].first == outs[i - 1].first)
      return c.fail("tensor %zu: two outputs are one buffer", std::max(outs[i].second, outs[i - 1].second));
  for (size_t i = 0; i < count; ++i) {
    const HcamdClipTensor &t = tensors[i];
    if (!t.count)
      continue;
    if (t.in == norm || t.out == norm)
      return c.fail("tensor %zu: the norm is a tensor's buffer", i);
    const auto at = std::lower_bound(outs.begin(), outs.end(), t.in,
                                     [&](const auto &o, const void *p) { return below(o.first, p); });
    if (at != outs.end() && at->first == t.in && at->second != i)
      return c.fail("tensor %zu: an output is another tensor's input", i);
  }
  return 0;
}
} // namespace

size_t hcamdClipGradNormWorkspace(size_t tensors) noexcept { return (kClipCells + ceilDiv(tensors, kClipTensors)) * 8; }

int hcamdLaunchClipGradNorm(OlQueue q, const HcamdClipTensor *tensors, size_t count, float maxNorm, float *norm,
                            void *work, size_t workBytes) noexcept {
  const Call c{q, "hcamdLaunchClipGradNorm"};
  if (!q)
    return 1;
  if (!(maxNorm >= 0.0f))
    return c.fail("the largest norm must not be negative");
  if ((count && !tensors) || count > 0x7fffffff)
    return c.fail("tensors is null, or too many");
  if (c.check({"norm", norm, 1, 1, 1, 4}) || c.work(work, workBytes, hcamdClipGradNormWorkspace(count)))
    return 1;
  size_t all = 0, elems = 0;
  for (size_t i = 0; i < count; ++i) {
    const HcamdClipTensor &t = tensors[i];
    if (t.type != HCAMD_F32 && !half16(t.type))
      return c.fail("tensor %zu: type %d (fp32, fp16, bf16)", i, t.type);
    if (t.count > ((size_t)1 << 40))
      return c.fail("tensor %zu: too many elements", i);
    if (t.count && (c.check({"a tensor", t.in, t.count, 1, t.count, elemBytes(t.type)}) ||
                    c.check({"a clipped tensor", t.out, t.count, 1, t.count, elemBytes(t.type)})))
      return 1;
    elems += t.count;
  }
  try {
    if (clipApart(c, tensors, count, norm))
      return 1;
  } catch (...) {
    return c.fail("out of host memory");
  }
  const size_t chunk = clipChunk(elems);
  for (size_t i = 0; i < count; ++i)
    all += ceilDiv(tensors[i].count, chunk);
  if (all > 0x7fffffff)
    return c.fail("too many elements");
  const size_t launches = std::max<size_t>(1, ceilDiv(count, (size_t)kClipTensors));
  size_t cells = 0;
  for (int pass = 0; pass < 2; ++pass) {
    size_t cell = 0;
    for (size_t l = 0; l < launches; ++l) {
      ClipArgs a{};
      const size_t first = l * kClipTensors, n = std::min<size_t>(kClipTensors, count - std::min(count, first));
      size_t chunks = 0;
      for (size_t i = 0; i < n; ++i) {
        const HcamdClipTensor &t = tensors[first + i];
        a.in[i] = t.in, a.out[i] = t.out, a.count[i] = t.count, a.type[i] = (uint8_t)t.type;
        a.first_chunk[i] = (uint32_t)chunks;
        chunks += ceilDiv(t.count, chunk);
      }
      a.first_chunk[n] = (uint32_t)chunks;
      a.tensors = (uint32_t)n, a.chunk = (uint32_t)chunk;
      a.partial = static_cast<double *>(work), a.first_cell = (uint32_t)cell;
      a.max_norm = maxNorm, a.norm = norm, a.cells = (uint32_t)cells;
      const size_t groups = clipGroups(chunks, all);
      if (pass == 0 ? c.launch("clip", "hcamd_clip_sums", a, groups)
                    : c.launch("clip", "hcamd_clip_scale", a, std::max<size_t>(1, std::min<size_t>(chunks, 4096))))
        return 1;
      cell += groups;
    }
    cells = cell;
  }
  return 0;
}

} // extern "C"
