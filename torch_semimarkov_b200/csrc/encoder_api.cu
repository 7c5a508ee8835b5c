// encoder_api.cu -- the extern "C" entry points of the encoder operators
// (include/semicrf.h).  Each validates its arguments before any CUDA call and
// enqueues kernels on the given stream; nothing allocates or synchronises.

#include <initializer_list>

#include "encoder_internal.cuh"

using namespace semicrf;

namespace {

bool known_type(int dtype) {
  return dtype == SEMICRF_F32 || dtype == SEMICRF_BF16 || dtype == SEMICRF_F16;
}

// sizes within which every index below fits 63 bits and every grid 31
constexpr int64_t kMaxT = (int64_t)1 << 40, kMaxD = (int64_t)1 << 20, kMaxB = (int64_t)1 << 31;
constexpr int64_t kMaxRows = (int64_t)1 << 42, kMaxValues = (int64_t)1 << 46;
constexpr int64_t kMaxNormWidth = 8192;  // a row's registers in one CTA of 16 warps

int check_sizes(int64_t B, int64_t T, int64_t D, int dtype) {
  if (B < 0 || T < 0 || D < 1 || !known_type(dtype)) return SEMICRF_ERR_INVALID_ARGUMENT;
  if (B > kMaxB || T > kMaxT || D > kMaxD) return SEMICRF_ERR_UNSUPPORTED;
  if (B && T > kMaxRows / B) return SEMICRF_ERR_UNSUPPORTED;
  if (B * T > kMaxValues / D) return SEMICRF_ERR_UNSUPPORTED;
  return SEMICRF_OK;
}

int check_recurrence(const semicrf_recurrence* p) {
  if (!p) return SEMICRF_ERR_INVALID_ARGUMENT;
  const int st = check_sizes(p->batch, p->T, p->D, p->dtype);
  if (st != SEMICRF_OK) return st;
  // one CTA per 64 positions and 64 channels
  const int64_t tiles = (p->D + 63) / 64, chunks = (p->T + 63) / 64;
  if (p->batch && chunks * tiles > 0x7fffffff / p->batch) return SEMICRF_ERR_UNSUPPORTED;
  return SEMICRF_OK;
}

int check_norm(const semicrf_block_norm* p) {
  if (!p) return SEMICRF_ERR_INVALID_ARGUMENT;
  const int st = check_sizes(p->batch, p->T, p->D, p->dtype);
  if (st != SEMICRF_OK) return st;
  if (p->D > kMaxNormWidth) return SEMICRF_ERR_UNSUPPORTED;
  return SEMICRF_OK;
}

int check_norm_inputs(const semicrf_block_norm* p) {
  if (!(p->eps >= 0.f) || !p->next_weight) return SEMICRF_ERR_INVALID_ARGUMENT;
  if (p->batch && p->T && !p->residual.data) return SEMICRF_ERR_INVALID_ARGUMENT;
  const bool branch = p->branch.data != nullptr;
  if (branch && (!p->gate.data || !p->branch_weight || !p->residual_scale))
    return SEMICRF_ERR_INVALID_ARGUMENT;
  return SEMICRF_OK;
}

// What the kernels read and write codes by: half a group's 16 bytes or less.
bool codes_aligned(const int8_t* codes) { return reinterpret_cast<uintptr_t>(codes) % 8 == 0; }

// Whether every tensor starts on a multiple of its element's size.
bool elements_aligned(int dtype, std::initializer_list<const semicrf_sequence*> list) {
  for (const semicrf_sequence* s : list)
    if (reinterpret_cast<uintptr_t>(s->data) % (dtype == SEMICRF_F32 ? 4 : 2)) return false;
  return true;
}

cudaStream_t as_stream(void* s) { return static_cast<cudaStream_t>(s); }

}  // namespace

extern "C" {

size_t semicrf_recurrence_saved_size(const semicrf_recurrence* p) {
  return check_recurrence(p) == SEMICRF_OK ? recurrence_saved_bytes(p) : 0;
}

size_t semicrf_recurrence_workspace_size(const semicrf_recurrence* p) {
  return check_recurrence(p) == SEMICRF_OK ? recurrence_workspace_bytes(p) : 0;
}

int semicrf_recurrence_forward(const semicrf_recurrence* p, const semicrf_sequence* h,
                               float* final_state, void* saved, void* workspace,
                               size_t workspace_bytes, void* stream) {
  const int st = check_recurrence(p);
  if (st != SEMICRF_OK) return st;
  if (p->batch == 0) return SEMICRF_OK;
  if (!h || !final_state) return SEMICRF_ERR_INVALID_ARGUMENT;
  if (p->T && (!p->x.data || !p->gate.data || !h->data)) return SEMICRF_ERR_INVALID_ARGUMENT;
  if (!elements_aligned(p->dtype, {&p->x, &p->gate, h})) return SEMICRF_ERR_INVALID_ARGUMENT;
  const size_t need = recurrence_workspace_bytes(p);
  if (workspace_bytes < need || (need && !workspace)) return SEMICRF_ERR_WORKSPACE;
  return recurrence_forward(p, *h, final_state, saved, workspace, as_stream(stream));
}

int semicrf_recurrence_backward(const semicrf_recurrence* p, const void* saved,
                                const semicrf_sequence* grad_h, const float* grad_state,
                                const semicrf_sequence* grad_x,
                                const semicrf_sequence* grad_gate, float* grad_initial,
                                void* workspace, size_t workspace_bytes, void* stream) {
  const int st = check_recurrence(p);
  if (st != SEMICRF_OK) return st;
  if (p->batch == 0) return SEMICRF_OK;
  if (!grad_h || !grad_x || !grad_gate) return SEMICRF_ERR_INVALID_ARGUMENT;
  if (p->T && (!p->x.data || !p->gate.data || !grad_x->data || !grad_gate->data || !saved))
    return SEMICRF_ERR_INVALID_ARGUMENT;
  if (!elements_aligned(p->dtype, {&p->x, &p->gate, grad_h, grad_x, grad_gate}))
    return SEMICRF_ERR_INVALID_ARGUMENT;
  const size_t need = recurrence_workspace_bytes(p);
  if (workspace_bytes < need || (need && !workspace)) return SEMICRF_ERR_WORKSPACE;
  return recurrence_backward(p, saved, *grad_h, grad_state, *grad_x, *grad_gate, grad_initial,
                             workspace, as_stream(stream));
}

int semicrf_recurrence_step(int64_t B, int64_t D, int dtype, const void* x, int64_t x_stride,
                            const void* gate, int64_t gate_stride, const uint8_t* active,
                            const float* state, float* state_out, void* h, void* stream) {
  const int st = check_sizes(B, 1, D, dtype);
  if (st != SEMICRF_OK) return st;
  if (B == 0) return SEMICRF_OK;
  if (!x || !gate || !state || !state_out || !h) return SEMICRF_ERR_INVALID_ARGUMENT;
  if (B > (int64_t)0x7fffffff * 128 / D) return SEMICRF_ERR_UNSUPPORTED;
  return recurrence_step(B, D, dtype, x, x_stride, gate, gate_stride, active, state, state_out, h,
                         as_stream(stream));
}

int semicrf_block_norm_forward(const semicrf_block_norm* p, const semicrf_sequence* residual_out,
                               const semicrf_sequence* normed, float* statistics, int8_t* codes,
                               uint8_t* scales, void* stream) {
  int st = check_norm(p);
  if (st == SEMICRF_OK) st = check_norm_inputs(p);
  if (st != SEMICRF_OK) return st;
  if (p->batch == 0 || p->T == 0) return SEMICRF_OK;
  if (!residual_out || !normed || !normed->data || (p->branch.data && !residual_out->data) ||
      !codes != !scales)
    return SEMICRF_ERR_INVALID_ARGUMENT;
  if (!codes_aligned(codes) ||
      !elements_aligned(p->dtype, {&p->residual, &p->branch, &p->gate, residual_out, normed}))
    return SEMICRF_ERR_INVALID_ARGUMENT;
  return block_norm_forward(p, *residual_out, *normed, statistics, codes, scales,
                            as_stream(stream));
}

size_t semicrf_block_norm_workspace_size(const semicrf_block_norm* p) {
  return check_norm(p) == SEMICRF_OK ? block_norm_workspace_bytes(p) : 0;
}

int semicrf_block_norm_backward(const semicrf_block_norm* p, const float* statistics,
                                const semicrf_sequence* grad_residual_out,
                                const semicrf_sequence* grad_normed,
                                const semicrf_sequence* grad_residual,
                                const semicrf_sequence* grad_branch,
                                const semicrf_sequence* grad_gate, float* grad_weights,
                                void* workspace, size_t workspace_bytes, void* stream) {
  int st = check_norm(p);
  if (st == SEMICRF_OK) st = check_norm_inputs(p);
  if (st != SEMICRF_OK) return st;
  if (!grad_residual_out || !grad_normed || !grad_residual || !grad_branch || !grad_gate ||
      !grad_weights)
    return SEMICRF_ERR_INVALID_ARGUMENT;
  if (p->batch && p->T &&
      (!statistics || !grad_residual->data ||
       (p->branch.data && (!grad_branch->data || !grad_gate->data))))
    return SEMICRF_ERR_INVALID_ARGUMENT;
  if (!elements_aligned(p->dtype, {&p->residual, &p->branch, &p->gate, grad_residual_out, grad_normed,
                                   grad_residual, grad_branch, grad_gate}))
    return SEMICRF_ERR_INVALID_ARGUMENT;
  if (p->batch == 0 || p->T == 0)
    return cudaMemsetAsync(grad_weights, 0, sizeof(float) * 3 * p->D, as_stream(stream)) ==
                   cudaSuccess
               ? SEMICRF_OK
               : SEMICRF_ERR_CUDA;
  const size_t need = block_norm_workspace_bytes(p);
  if (workspace_bytes < need || !workspace) return SEMICRF_ERR_WORKSPACE;
  return block_norm_backward(p, statistics, *grad_residual_out, *grad_normed, *grad_residual,
                             *grad_branch, *grad_gate, grad_weights, workspace,
                             as_stream(stream));
}

int semicrf_pack(int64_t B, int64_t T, int64_t D, int dtype, const semicrf_sequence* x,
                 const int64_t* lengths, int8_t* codes, uint8_t* scales, void* stream) {
  const int st = check_sizes(B, T, D, dtype);
  if (st != SEMICRF_OK) return st;
  if (B == 0 || T == 0) return SEMICRF_OK;
  if (!x || !x->data || !codes || !scales) return SEMICRF_ERR_INVALID_ARGUMENT;
  if (!codes_aligned(codes) || !elements_aligned(dtype, {x})) return SEMICRF_ERR_INVALID_ARGUMENT;
  return pack_rows(B, T, D, dtype, *x, lengths, codes, scales, as_stream(stream));
}

int semicrf_unpack(int64_t rows, int64_t D, int dtype, const int8_t* codes,
                   const uint8_t* scales, void* out, void* stream) {
  const int st = check_sizes(1, rows, D, dtype);
  if (st != SEMICRF_OK) return st;
  if (rows == 0) return SEMICRF_OK;
  if (!codes || !scales || !out || !codes_aligned(codes)) return SEMICRF_ERR_INVALID_ARGUMENT;
  return unpack_rows(rows, D, dtype, codes, scales, out, as_stream(stream));
}

size_t semicrf_packed_weight_grad_workspace_size(int64_t B, int64_t T, int64_t D, int64_t M,
                                                 int dtype) {
  if (check_sizes(B, T, D, dtype) != SEMICRF_OK || M < 1 || M > kMaxD) return 0;
  return packed_weight_grad_workspace_bytes(B, T, D, M, dtype);
}

int semicrf_packed_weight_grad(int64_t B, int64_t T, int64_t D, int64_t M, int dtype,
                               const semicrf_sequence* grad_output, const int8_t* codes,
                               const uint8_t* scales, int packed_dtype, const int64_t* lengths,
                               int out_dtype, void* out, void* workspace, size_t workspace_bytes,
                               void* stream) {
  int st = check_sizes(B, T, D, dtype);
  if (st == SEMICRF_OK) st = M < 1 ? SEMICRF_ERR_INVALID_ARGUMENT : check_sizes(B, T, M, dtype);
  if (st != SEMICRF_OK) return st;
  if (!known_type(out_dtype) || !known_type(packed_dtype) || !out) return SEMICRF_ERR_INVALID_ARGUMENT;
  if (!grad_output || (B && T && (!grad_output->data || !codes || !scales)))
    return SEMICRF_ERR_INVALID_ARGUMENT;
  if (!codes_aligned(codes) || !elements_aligned(dtype, {grad_output}))
    return SEMICRF_ERR_INVALID_ARGUMENT;
  const size_t need = packed_weight_grad_workspace_bytes(B, T, D, M, dtype);
  if (workspace_bytes < need || !workspace) return SEMICRF_ERR_WORKSPACE;
  return packed_weight_grad(B, T, D, M, dtype, packed_dtype, *grad_output, codes, scales, lengths,
                            out_dtype, out, workspace, as_stream(stream));
}

}  // extern "C"
