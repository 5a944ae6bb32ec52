// Launch API of the decoder-block kernels: rotary positions, counter-based
// dropout (alone and in the residual add + LayerNorm) and attention with a
// decay per head.
#pragma once
#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include <cstddef>
#include <cstdint>

namespace nexar {

// ---------------------------------------------------------------- rotary positions
// One rotated tensor: x [B, T, heads, D] with strides (in elements) and unit
// inner stride, y contiguous. Heads from `rotated` on are copied.
struct RotaryPart {
  const void* x;
  void* y;
  long long sb, st, sh;
  int heads, rotated;
};
struct RotaryArgs {
  RotaryPart part[2];
  int nparts;
  const float* table;      // [rows, R]: (cos, sin) of pair 0, 1, ...
  const void* positions;   // nullptr: start + t
  int positions_64;        // int64 (1) or int32 (0)
  long long pb, pt;        // strides of positions
  long long start, rows;
  long long B, T;
  int D, R;
  int interleaved;
  float sign;              // +1, or -1 for the inverse turn
};
// elem: bytes per element (2 or 4); half: fp16 instead of bf16.
cudaError_t rotary(const RotaryArgs& a, int elem, bool half, cudaStream_t s);
// table[p, 2 i], table[p, 2 i + 1] = magnitude * (cos, sin)(p * freq[i]), angles in 64 bits.
cudaError_t rotary_table(const double* freq, float* table, long long rows, int R, double magnitude, cudaStream_t s);

// ---------------------------------------------------------------- dropout
// state: (seed, step) on the device. snapshot (may be null) receives the two
// values used, for the backward pass. dtype: 0 bf16, 1 fp16, 2 fp32.
cudaError_t dropout(const void* x, void* y, long long n, int dtype, const int64_t* state, uint32_t site,
                    uint32_t threshold, float scale, int64_t* snapshot, cudaStream_t s);
// s = bf16(x + drop(r + rb)), y = LayerNorm(s); C % 8 == 0, C <= 2048.
cudaError_t dropout_ln_fwd(const __nv_bfloat16* x, const __nv_bfloat16* r, const __nv_bfloat16* rb,
                           __nv_bfloat16* sum_out, const __nv_bfloat16* w, const __nv_bfloat16* b, __nv_bfloat16* y,
                           float* mean, float* rstd, int R, int C, float eps, const int64_t* state, uint32_t site,
                           uint32_t threshold, float scale, int64_t* snapshot, cudaStream_t s);
// dx = dres + dLN/ds, dr = drop'(dx), column sums dw, db and (if not null) drb = column sums of dr.
// scratch: dropout_ln_bwd_scratch_floats(R, C) floats.
size_t dropout_ln_bwd_scratch_floats(int R, int C);
cudaError_t dropout_ln_bwd(const __nv_bfloat16* dy, const __nv_bfloat16* s_in, const float* mean, const float* rstd,
                           const __nv_bfloat16* w, const __nv_bfloat16* dres, __nv_bfloat16* dx, __nv_bfloat16* dr,
                           __nv_bfloat16* dw, __nv_bfloat16* db, __nv_bfloat16* drb, float* scratch, int R, int C,
                           const int64_t* state, uint32_t site, uint32_t threshold, float scale, cudaStream_t s);

// ---------------------------------------------------------------- decay attention
// One use of the chunked recurrence (see decay_attention.cu): out_i = intra *
// sum_{j <= i} lam^(i-j) (q_i . k_j) v_j + inter * lam^(i+a) X q_i, tokens
// taken from the first (reverse = 0) or the last (reverse = 1).
struct DecayRole {
  const __nv_bfloat16 *q, *k, *v;
  __nv_bfloat16* out;
  long long qb, qt, qh, kb, kt, kh, vb, vt, vh, ob, ot, oh;  // strides in elements
  int reverse;
  float intra, inter, kv;   // factors of the scores, of the state's part and of the state's update
  const float* init;        // [B, H, D, D] state before the first token, or null
  int init_transposed;
  float* final_state;       // state behind the last token, or null
  // When the tokens are split: states before every piece of seg_tokens, [B, H, nseg, D, D]. seg_own: computed here and
  // read as they are; else another role's or the forward pass's, read transposed. Roles with states of their own come
  // first.
  float* segments;
  int seg_own;
};
struct DecayArgs {
  DecayRole role[3];
  int nroles;
  const float* log_decay;   // [H]
  const int* lengths;       // [B] or null
  int B, T, H, D;
  // The states are computed for nseg pieces of seg_tokens, side by side; the outputs then by blocks that take `step`
  // pieces one after the other.
  int nseg, seg_tokens, step;
};
// Chunks of 64 tokens to a segment of the forward pass (ragged: sequences have lengths of their own).
int decay_segment_chunks(int B, int T, int H, int D, bool ragged);
// Segments of so many chunks that a block of the backward pass takes; 0: whole sequences.
int decay_backward_step(int B, int T, int H, int D, int chunks);
cudaError_t decay_attention(const DecayArgs& a, cudaStream_t s, int* launches);
unsigned int decay_error_flag();  // current GPU: not 0 once a wait inside decay_attention has given up (synchronises)
// One token: state = lam state + k v^T in place, o = scale * state^T q. q, k, v rows with strides, o contiguous.
struct DecayStepArgs {
  const __nv_bfloat16 *q, *k, *v;
  __nv_bfloat16* o;
  float* state;             // [B, H, D, D]
  const float* log_decay;
  long long qb, qh, kb, kh, vb, vh;
  int B, H, D;
  float scale;
};
cudaError_t decay_step(const DecayStepArgs& a, cudaStream_t s);

}  // namespace nexar
