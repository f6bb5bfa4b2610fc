// Argument blocks of the language-model kernels, passed by value and shared by
// the launchers (operators.cpp) and the kernels.  Pointers are device pointers,
// leading dimensions are in elements.
#pragma once
#include <stddef.h>
#include <stdint.h>

namespace hcamd {

// h = x + residual, y = h / rms(h) * weight (rmsnorm.hip)
struct NormArgs {
  const void *x, *residual, *weight; // residual, weight may be null
  void *summed, *out;                // summed may be null
  float *scale, *rstd;               // scale: 8-bit output only; rstd may be null
  size_t ldx, ldr, lds, ldo;
  uint32_t rows, cols;
  float eps;
  int weight_f32; // weight is fp32 (else the element type)
};
struct NormBackArgs {
  const void *grad_out, *summed, *weight, *grad_summed; // weight, grad_summed may be null
  const float *rstd;
  void *grad_in, *grad_weight; // grad_weight may be null
  float *partial;              // [bands][cols]
  size_t ldg, ldh, ldgs, ldgi;
  uint32_t rows, cols, band, bands; // rows to a band, bands
  int weight_f32;
};

// One tiled product C[M,N] = sum_k A(m,k) B(n,k) (mma.h).  A second pair
// continues the sum over k where `segments` is 2; a second B alone interleaves
// its rows with the first's (the gated block).
struct MmaArgs {
  const void *a[2], *b[2];
  size_t lda[2], ldb[2];
  int M, N, K;
  int segments;   // 1, or 2: k runs through (a[0], b[0]), then (a[1], b[1])
  int splits;     // k tiles are dealt to this many workgroups (grid y)
  int half_from;  // 256 x 256 tiles from here on are worked as two halves
};

struct GatedArgs {
  MmaArgs mma; // a[0] = x [T,D], b = {gate, up} [F,D]; N = F
  const float *x_scale, *gate_scale, *up_scale; // 8-bit operands only
  void *out, *gate, *up;                        // gate, up may be null
  size_t ldo, ldgate, ldup;
  int activation;
  int out_f16; // 8-bit operands: the output is fp16 (else bf16)
};
struct GatedBackArgs { // pre-activation gradients, element by element
  const void *grad_out, *gate, *up;
  void *dgate, *dup;
  size_t ldg, ldgate, ldup, ldd;
  uint32_t rows, cols;
  int activation;
  // fp16: the largest magnitude each workgroup of a launch before this one has met, and what
  // undoes the scaling that follows from them (written by the first workgroup)
  float *most, *undo;
  uint32_t mosts;
};

// a product whose result is stored: in the element type (`out`), or as fp32
// partial sums (`partial`: [splits][M][ldp]) that a second kernel adds up
struct StoreArgs {
  MmaArgs mma;
  void *out;
  float *partial;
  size_t ldo, ldp;
  const float *undo; // when not null: *undo multiplies what goes to `out`
  int accumulate;      // add to `partial` instead of replacing it
};
struct PairStoreArgs { // two products of one shape, one after the other in grid x
  StoreArgs p[2];
  int tiles; // of one of them
};
struct ProductsArgs { // dx and dW of a backward pass; workgroups of one split of each, 0: not wanted
  StoreArgs nn;
  PairStoreArgs tn;
  int nn_groups, tn_groups;
};
struct FoldArgs { // out = sum over splits of partial (* *undo)
  const float *partial;
  void *out;
  size_t ldp, ldo;
  uint32_t rows, cols, splits;
  const float *undo;
};

struct FoldJobs { // grid y selects
  FoldArgs job[3];
};

struct LayArgs { // a matrix copied to rows of ld_to, a multiple of 16 bytes, zeros behind each row's last element
  const void *from;
  void *to;
  size_t ld_from, ld_to;
  uint32_t rows, cols;
};
struct LayJobs { // grid y selects
  LayArgs job[3];
};

struct XentArgs {
  MmaArgs mma; // a = x [T,D], b = weight rows of this piece; N = rows of the piece
  const void *targets;
  int target_i64;
  int v0;            // first vocabulary row of the piece
  int tile0;         // column tiles before the piece
  int vocab;         // rows of the whole weight matrix
  // forward: per row and column tile (max, sum of exp(z - max)), target logit
  float *stats;      // [T][tiles][2]
  float *zt;         // [T]
  int tiles;
  // backward
  const float *lse, *grad_loss, *factor;
  void *p;           // [T][ldp] (softmax - onehot) * grad_loss * *factor
  size_t ldp;
};
struct XentPrepareArgs { // before the backward pass
  const void *x, *targets;
  const float *grad_loss;
  int target_i64;
  float top;        // what the largest |grad_loss| becomes
  float *factor;    // [2]
  void *live_x;     // x with zeros in the rows that take no part, padded to pieces of 8 (null: not wanted)
  size_t ldx, ldl;
  uint32_t rows, cols, vocab;
};
struct XentRowsArgs {
  const float *stats, *zt;
  const void *targets;
  int target_i64;
  float *loss, *lse;
  uint32_t rows, vocab, tiles;
};

// Clipping by the global norm (clip.hip): the tensors of one launch.
constexpr int kClipTensors = 64;
struct ClipArgs {
  const void *in[kClipTensors];
  void *out[kClipTensors];
  uint64_t count[kClipTensors];
  uint32_t first_chunk[kClipTensors + 1]; // chunks before this tensor
  uint8_t type[kClipTensors];
  uint32_t tensors, chunk;                // elements to a chunk
  double *partial;       // one cell per workgroup of every launch of the call
  uint32_t first_cell, cells;
  float max_norm;
  float *norm;
};

} // namespace hcamd
