// Host-side entry points of the kernel families, called by capi.cu.
#pragma once
#include "common.cuh"

namespace msx {

void spmm_run(int value_dtype, int index_dtype, const void *data, const void *indices, const void *indptr,
              const void *rhs, int64_t k, void *out, int64_t n_rows, int64_t n_cols, int64_t nnz,
              cudaStream_t stream);

void spgemm_run(bool write, int value_dtype, int lhs_it, const void *ld, const void *li, const void *lp, int rhs_it,
                const void *rd, const void *ri, const void *rp, int64_t m, int64_t rhs_rows, int64_t n_cols,
                int out_it, void *out_indptr, void *out_idx, void *out_data, int64_t *out_nnz, bool prune,
                cudaStream_t s);

void csr_batched_matvec_run(int value_dtype, int index_dtype, const void *data, const void *indices,
                            const void *indptr, int64_t nnz, int64_t n_rows, int64_t n_cols, int64_t batch,
                            const void *rhs, void *out, cudaStream_t s);
void csr_batched_matmul_run(int value_dtype, int index_dtype, const void *data, const void *indices,
                            const void *indptr, int64_t nnz, int64_t n_rows, int64_t n_cols, int64_t batch,
                            int64_t k, const void *rhs, void *out, cudaStream_t s);

void csr_diagonal_run(int value_dtype, int index_dtype, const void *data, const void *indices, const void *indptr,
                      int64_t n_diag, void *out, cudaStream_t stream);

// COO -> CSR (by_col: rows sorted by (column, source position) as the
// reference's coo_tocsr; else by source position only). out_data may be null
// (structure only); out_perm (int64[nnz], the source position of every output
// entry) may be null. Synchronises `s` once (coordinate check).
void coo_tocsr_run(int value_dtype, int index_dtype, const void *data, const void *row, const void *col, int64_t nnz,
                   int64_t n_rows, int64_t n_cols, bool by_col, void *out_data, void *out_indices, void *out_indptr,
                   int64_t *out_perm, cudaStream_t s);
// CSR of A^T: row c lists A's entries of column c by ascending row.
void csr_transpose_run(int value_dtype, int index_dtype, const void *data, const void *indices, const void *indptr,
                       int64_t nnz, int64_t n_rows, int64_t n_cols, void *out_data, void *out_indices,
                       void *out_indptr, int64_t *out_perm, cudaStream_t s);
// out[p] = sum_j cot[row(p), j] * rhs[col(p), j], j in order (k = 1: matvec).
void csr_data_vjp_run(int value_dtype, int index_dtype, const void *indices, const void *indptr, int64_t nnz,
                      int64_t n_rows, const void *rhs, const void *cot, int64_t k, void *out, cudaStream_t s);

// Distillation against a CSR matrix of teacher logits (rows x vocab). With
// `loss`: the forward pass (`stats`, 16 bytes a row, may be null); with `grad`
// too: both in one pass; without `loss`: the backward pass from `stats`.
struct DistillCall {
  const void *logits;
  int64_t ld;  // elements between rows of the logits
  const void *t_data, *t_indices, *t_indptr;
  int64_t nnz, rows, vocab;
  float temperature;
  const float *cotangent;  // per row; null: ones
  float *loss;
  void *stats, *grad;
};
void distill_run(int value_dtype, int index_dtype, const DistillCall &call, cudaStream_t s);

// Windowed attention. q, k, v: (batch, tokens, heads, dim) with any batch,
// token and head strides (in elements) and stride 1 along dim; out, grad_out and
// the gradients are contiguous in that order. lse and delta: float (batch,
// q_heads, q_len rounded up to a multiple of 128), delta followed by more workspace
// (window_backward_floats in all). A null dq (dk and dv) is not computed.
struct WindowTensor {
  const void *ptr;
  int64_t batch, token, head;
};
struct WindowCall {
  WindowTensor q, k, v;
  const void *grad_out;
  void *out, *dq, *dk, *dv;
  void *out_low;  // what rounding out to its 16-bit type took off, in that type; may be null
  float *lse, *delta;
  int64_t batch, q_len, k_len;
  int q_heads, k_heads, dim;
  int64_t window, sinks;
  float scale;
  const void *indptr;  // packed sequences (batch 1, q_len = k_len), or null
  int indptr_dtype;    // of indptr or lengths
  int64_t n_seq;
  const void *lengths;  // keys of each batch entry (type indptr_dtype), or null: k_len
};
void window_forward_run(int value_dtype, const WindowCall &c, cudaStream_t s);
int64_t window_backward_floats(const WindowCall &c);
void window_decode_run(int value_dtype, const WindowCall &c, cudaStream_t s);
bool window_take_error();  // reads and clears the device's wait error flag
void window_set_wait_limit(long long ns);  // negative: the default
void window_backward_run(int value_dtype, const WindowCall &c, cudaStream_t s);

}  // namespace msx
