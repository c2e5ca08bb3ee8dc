// Tensor-core (tcgen05) products grouped by expert: declarations; the kernel
// lives in expert_tc.cu.
#pragma once

#include "common.cuh"

namespace stade {

// Rows of one group that a product tile covers; expert < 0: rows of no group.
struct ExpertTile {
  int expert, row, rows, pad;
};
constexpr int kExpertTcRows = 256;   // rows of a tensor-core tile

// An operand as the tensor cores read it: `planes` 16-bit planes of an array
// of d2 x d1 rows of d0 values (row pitch `pitch`, a multiple of 8), one after
// the other.
struct ExpertOperand {
  const void* p;
  int64_t d0, d1, d2, pitch;
};

// The calls below, and expert_pack, are launched so that they overlap the end of
// the kernel before them; that has to be a kernel of the same call.
// out[s, :] (+)= in[s, :] W[e] (n_i -> n_o) or in[s, :] W[e]^T (trans)
stade_status expert_tc_rows(int dtype, const ExpertOperand& in, const ExpertOperand& w, void* out,
                            const ExpertTile* tiles, const int* count, int64_t max_tiles,
                            int64_t n_i, int64_t n_o, bool trans, bool add, cudaStream_t s);
// wb[e] (+)= sum over the group's rows of x^T yb (Float32)
stade_status expert_tc_wgrad(int dtype, const ExpertOperand& x, const ExpertOperand& yb, float* wb,
                             const int64_t* bounds, int64_t n_e, int64_t n_i, int64_t n_o, bool add,
                             cudaStream_t s);

// 16-bit planes of a rows x cols array at a pitch of `pitch` values: one plane
// of the type itself for the 16-bit types, three bf16 planes for Float32.
int64_t expert_planes(int dtype);
stade_status expert_pack(int dtype, const void* src, void* dst, int64_t rows, int64_t cols,
                         int64_t pitch, cudaStream_t s);

int expert_tc_take_error();

}  // namespace stade
