// Host launchers of the mixture-of-experts row kernels (no counterpart in the reference, whose all-to-all takes rows
// that are sorted already): the order of the rows by expert, the rows into it and back, and their gradients.
#pragma once
#include <cuda_runtime.h>
#include <cstdint>

namespace fo {

constexpr int kMaxExperts = 1024;
constexpr int kMaxTopK = 64;

// ids [tokens * top_k] (int32, or int64 with ids64): the experts chosen for each token, in [0, experts); any other
// value is a choice that this GPU does not serve.  slot [tokens * top_k]: the row of each choice, -1 if not served;
// source [tokens * top_k]: the choice of each row, -1 behind the last row; offsets [experts + 1]: each expert's first row.
// Rows of an expert keep the order of their choices.  The sort is one cluster of at most `most_ctas` CTAs, of 16, 8 or 1.
cudaError_t moe_sort_launch(const void* ids, bool ids64, int64_t choices, int experts, int most_ctas, int32_t* slot,
                            int32_t* source, int32_t* offsets, cudaStream_t stream);
// The cluster that sorts that many choices where clusters of `most` CTAs have a place.
int moe_sort_ctas(int64_t choices, int most);

// The router's weights or their gradients: fp32, or the rows' 16-bit type.
struct MoeWeights {
  const void* p;
  bool f32;
};

// One call's shape.  `rows` of `dim` 16-bit elements; dim a multiple of 8, every row 16-byte aligned.
struct MoeShape {
  int tokens, top_k, dim, experts;
  bool bf16;
};

// What tells the two calls below which rows no slot names (they are zeros in what is written): the sort's `source`, or `scratch`
// of moe_scratch_words int32 whatever it holds, where that is not 0.  The slots decide, not the sources: those save the search.
struct MoeSources {
  const int32_t* source;
  int32_t* scratch;
};
int64_t moe_scratch_words(const MoeShape& s, bool sources);

// R[slot[t, k]] = X[t]; every other row, and those from offsets[experts] on: zero.
cudaError_t moe_dispatch_launch(const MoeShape& s, const void* X, const int32_t* slot, const int32_t* offsets,
                                const MoeSources& from, void* R, cudaStream_t stream);
// O[t] = sum over k of w[t, k] * R[slot[t, k]] (w.p == nullptr: 1), choices without a row left out.
cudaError_t moe_combine_launch(const MoeShape& s, const void* R, MoeWeights w, const int32_t* slot, void* O,
                               cudaStream_t stream);
// DR[slot[t, k]] = w[t, k] * GO[t]; every other row, and those from offsets[experts] on: zero; DW[t, k] = <GO[t], R[slot[t, k]]>,
// 0 without a row, in w's type.  DR (then `from` is not used) or DW may be nullptr.
cudaError_t moe_combine_backward_launch(const MoeShape& s, const void* GO, const void* R, MoeWeights w,
                                        const int32_t* slot, const int32_t* offsets, const MoeSources& from, void* DR,
                                        void* DW, cudaStream_t stream);

}  // namespace fo
