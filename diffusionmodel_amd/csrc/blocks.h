// Operators of transformer blocks (layernorm.hip, rotary.hip, linear.hip).  Strides are in elements.
#pragma once
#include "common.h"

namespace ldm {

int launch_layer_norm(int dtype, const void* x, long xs, const float* w, const float* b, float eps, void* y, long ys,
                      float* mean, float* rstd, long rows, int C, hipStream_t s);
long ln_ws_floats(int dtype, long rows, long C);
// dw null: no parameter gradients (db and ws are then unused)
int launch_layer_norm_backward(int dtype, const void* dy, long dys, const void* x, long xs, const void* add, long as,
                               const float* mean, const float* rstd, const float* w, void* dx, long dxs, float* dw,
                               float* db, float* ws, long rows, int C, hipStream_t s);

struct RopeArgs {
    const void* in[2];             // queries, keys (H[1] = 0: no keys)
    void* out[2];
    long isb[2], isn[2], ish[2];   // input strides: batch, token, head
    long osb[2], osn[2], osh[2];
    int H[2];
    int N, D, P;                   // tokens per batch entry, elements per head, rotated pairs
    long tokens;                   // B * N
    const void* pos;
    int pos_dtype;                 // 0 int32, 1 int64, 2 f32
    long pos_sb, pos_sa, pos_sn;
    int axes;
    int sec_end[4];                // first pair behind each axis; D for the last one and those that are not there
    const float* inv_freq;         // [P]
    int inverse;
    int nrot, nchunk, tpb, hpg;    // set by launch_rope
    unsigned groups;
    bool through;
};
int launch_rope(int dtype, int interleaved, RopeArgs a, hipStream_t s);

enum LinAct { LIN_NONE = 0, LIN_SILU = 1, LIN_RELU = 2, LIN_GELU = 3 };
// C[m, n] = act(sum_k A(m, k) B(k, n) + bias[n] + res[m, n]); pre: the value before the activation, optional.
// An operand that is contiguous along k (kc) holds A(m, k) at m * lda + k, B(k, n) at n * ldb + k; otherwise A(m, k) at
// k * lda + m, B(k, n) at k * ldb + n.
struct GemmArgs {
    const void *A, *B;
    const float* bias;
    const void* res;
    void *pre, *C;
    long lda, ldb, ldr, ldp, ldc;
    long M, N, K;
    int act;
    float* part;                   // set by launch_gemm: partial sums [parts][M][N rounded up to 8] of a split contraction
    int kper;                      // set by launch_gemm: steps of the contraction per part
    bool through;                  // set by launch_gemm: outputs are written through the L2
};
// the join of a split contraction that the caller launches later; blocks = 0: none
struct GemmJoin {
    GemmArgs a;
    int parts;
    unsigned blocks;
};
long gemm_ws_floats(int dtype, long M, long N, long K);
// later null: the product is complete; otherwise a join may be left there, and ws holds its parts until then
int launch_gemm(int dtype, const GemmArgs& a, bool akc, bool bkc, float* ws, GemmJoin* later, hipStream_t s);
// dz = dy act'(pre) (not written without an activation: dz is dy) and, in ws [*groups][N], what adds up to db = column sums
// of dz; *groups = -1: db is complete, or null and not taken
long linear_dz_ws_floats(int dtype, long M, long N);
int launch_linear_dz(int dtype, const void* dy, long lddy, const void* pre, long ldp, void* dz, long lddz, float* db, float* ws,
                     long M, long N, int act, int* groups, hipStream_t s);
// what the products and the dz kernel left, in one launch
int launch_linear_finish(int dtype, const GemmJoin& x, const GemmJoin& w, const float* part, int groups, long N, float* db,
                         hipStream_t s);

}  // namespace ldm
