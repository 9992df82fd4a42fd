// Local products whose epilogue is more than a conversion, on the tcgen05 core of the plain GEMM (CTA pairs, 256-row tiles):
//   kGated       h = act(x Wg) * (x Wu), and what its gradient needs
//   kGatedGrad   dg, du from dh = dy Wd^T
//   kPlain       C (+)= alpha (A0 B0 (+ A1 B1)), bf16 or fp32
//   kHead        logits of a tile as statistics and exponentials relative to the tile's maximum
//   kGram        alpha A A^T + beta C of a batch, symmetric: half of the tiles, mirrored (fp16)
//   kStep        a X + gamma B X of a batch (fp32, with an fp16 copy, or the last one as the result)
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace msb {

enum ProductKind : int { kNone = -1, kGated = 0, kGatedGrad = 1, kPlain = 2, kHead = 3, kGram = 4, kStep = 5 };

// Features of a row that share an exponent in what kGated keeps.
constexpr int kGatedChunk = 32;

struct Product {
  CUtensorMap a[2], b[2];      // operands: two ranges of the contraction (kPlain), b of kGated: gate and up
  CUtensorMap o[3];            // outputs that leave as TMA stores of 32 x 32
  int M, N;                    // of an item of the batch
  int kblocks[2];              // of the two ranges
  int items;                   // batch
  int a_mn_major, a_map3d, b_mn_major, b_map3d;
  int a_item, b_item;          // rows of the operand's map from one item to the next
  int k_item;                  // of a contraction in parts, which are the items: its length from one to the next
  int group, along_n;          // tile order: panels of `group` blocks along M or N
  // ---- kGated, kGatedGrad ----
  int act;                     // 0: silu, 1: tanh-GeLU
  int keep;                    // kGated: write what the gradient needs
  const void* g;               // kGatedGrad: fp16 [M, N], scaled per row and chunk
  const void* u;
  uint16_t* exps;              // [M, chunks]: exponents of gate (low byte) and up
  // ---- kHead ----
  float2* stats;               // [2 tiles_n, M], of each half of a tile's columns: maximum, sum of exp(z - maximum)
  float* label;                // [M]: the label's logit, where there is one
  const int64_t* targets;
  int vocab;
  int write;                   // exponentials are written
  int parts;                   // of the contraction, added in fp32 outside the tensor pipe; none is empty
  // ---- kPlain ----
  int out_item_rows;           // rows of the output from one item to the next, a multiple of 32
  int accumulate;              // add to what is there: c (bf16) is read, fp32 is added by the copy engine
  int64_t ldc;
  // ---- kPlain, kGram, kStep ----
  void* out;                   // kGram: fp16 [items, M, M]; kStep: the last step's result, or null
  const void* c;               // kPlain: the output; kGram: fp16 [items, M, M] or null; kStep: X in fp32 [items, M, N]
  float alpha, beta;
  void* copy;                  // kStep: fp16 copy of X, times
  float scale;
  int rows, cols;              // kStep: extent of the result that is wanted
  int64_t out_item, out_row, out_col;   // its strides in elements, one of the last two 1
  int out_fp32;                // kPlain too
};
struct ProductArgs {
  Product p[3];
  int tiles[3];                // tiles of the first problem, of the first two, of all (set by the launcher)
  int lead, rounds;            // tiles of the longer contraction, and of tile_walk.h (set by the launcher)
  uint32_t* status;            // [4]: code, blockIdx, detail, detail2
  uint64_t timeout_ns;
};

// An operand as the builder takes it: [rows, K] (K-major) or [K, rows] (mn_major), 16-bit; `k_rows`: rows of the latter over all items
// of a batch (0: K).
struct ProductOperand {
  const void* base;
  int64_t ld;
  int mn_major;
  int64_t k_rows;
};
// Maps of the operands for tiles of `tile_n` columns (0, or an error code).  `rows_a` / `rows_b`: extent along M / N over all items, `K`: of
// the contraction.  For kGated the columns of either half count.
int product_operands(Product* p, int kind, int tile_n, const ProductOperand* a, const ProductOperand* b, int ranges, int64_t rows_a,
                     int64_t rows_b, const int64_t* K);
// Output map of 16-bit or fp32 [rows, cols].
int product_output(Product* p, int which, const void* base, int64_t cols, int64_t rows, int64_t ld, bool fp32);
// Tiles of a problem.
int64_t product_tiles(const Product& p, int kind, int tile_n);

// `problems` problems: the first of kind k0, the others of kind k1, on at most `sms` SMs.  The first `longer` of them have one contraction, not
// shorter than the one of the others.  Supported: kGated, kHead alone (k1 kNone); (kGatedGrad, kPlain), (kPlain, kGatedGrad),
// (kPlain, kPlain).
cudaError_t launch_sm100_products(ProductArgs& args, int k0, int k1, int problems, int longer, int tile_n, int sms, cudaStream_t stream);

// All products of the orthogonal update of a batch in one launch: step by step X X^T, b A + c A^2 and a X + B X, in which a tile waits for the
// tiles that its matrix's product before it consists of.
struct ChainArgs {
  Product gram[2];             // kGram, of either copy of X
  Product square;              // kGram
  Product step[3];             // kStep: of either copy of X, and the last
  int items, steps;
  int tiles[2];                // of an item, kGram and kStep (set by the launcher)
  uint32_t* counters;          // [3 steps, items], 0 at launch: CTAs that have written their part of a tile, two a tile
  uint32_t* status;
  uint64_t timeout_ns;
};
// Columns of a tile, and the launch on at most `sms` SMs.
int chain_tile_n(int64_t m, int64_t n, int64_t items, int sms);
cudaError_t launch_sm100_chain(ChainArgs& args, int tile_n, int sms, cudaStream_t stream);

}  // namespace msb
