// Gradient of an embedding lookup by sorted tokens (embed.hip), shared with the score network's backward pass.
#pragma once
#include "token_common.h"

struct EmbedGrad {
  const void* d_out; int32_t dtype; int64_t d_stride;   // [n, width] gradient of the looked-up rows
  TokenView tok; int64_t n;                             // tokens; outside [0, tok.n_rows): no row
  int32_t rows;                                         // rows of d_table: tok.n_rows, or one more, which takes the tokens outside
  int32_t width;
  float scale;
  void* d_table; int32_t grad_dtype; int64_t t_stride;
  bool accumulate;
};
size_t embed_grad_workspace(int64_t n, int32_t rows, int32_t width);
void embed_grad(const EmbedGrad& g, void* workspace, hipStream_t s);   // sizes checked by the caller

// The atom branch of the score network's input embedding for integer atom types: a table of LD_A + 1 rows, before LayerNorm and
// after GELU, and the weight gradients from those of the rows before LayerNorm.
void type_embed(const float* Wa, const float* ba, const float* ga, const float* bea, float* pre, float* emb, hipStream_t s);
void type_embed_dw(const float* du, float* dWa, float* dba, hipStream_t s);
