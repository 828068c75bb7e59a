// C entry points of the sequence operators' kernel libraries. Each launches
// on the given device and stream and returns a hipError_t; none allocates,
// synchronises or throws. Types and what may be null: see the .hip files.
#pragma once
#include <stdint.h>

extern "C" {

int rlsched_norm_fwd(int device, void* stream, const void* x, const void* w,
                     const void* b, void* y, float* mean, float* rstd,
                     int64_t rows, int64_t dim, int64_t x_stride, double eps,
                     int type, int wtype);
int64_t rlsched_norm_parts(int64_t rows, int64_t dim, int type);
int rlsched_norm_bwd(int device, void* stream, const void* dy, const void* x,
                     const void* w, const float* mean, const float* rstd,
                     void* dx, void* dw, void* db, float* partial,
                     int64_t rows, int64_t dim, int64_t x_stride,
                     int64_t dy_stride, int type, int wtype);

int64_t rlsched_scan_scratch(int64_t T, int64_t E, int64_t H, int type,
                             int back);
int64_t rlsched_scan_states(int64_t T);
int64_t rlsched_scan_reach(int64_t H);
int rlsched_scan_fwd(int device, void* stream, const void* gate, const void* x,
                     const float* h0, const uint8_t* done, void* hs,
                     float* h_last, float* states, float* scratch, int64_t T,
                     int64_t E, int64_t H, int64_t gate_t, int64_t gate_e,
                     int64_t x_t, int64_t x_e, int type);
int rlsched_scan_bwd(int device, void* stream, const void* dhs,
                     const float* dh_last, const void* gate, const void* x,
                     const float* states, const uint8_t* done, void* dgate,
                     void* dx, float* dh0, float* scratch, int64_t T,
                     int64_t E, int64_t H, int64_t gate_t, int64_t gate_e,
                     int64_t x_t, int64_t x_e, int64_t dhs_t, int64_t dhs_e,
                     int type);
int rlsched_scan_step(int device, void* stream, const void* gate,
                      const void* x, const uint8_t* done, float* h, void* hs,
                      int64_t E, int64_t H, int64_t gate_e, int64_t x_e,
                      int type);

int64_t rlsched_logp_scratch(int64_t rows, int64_t A, int k, int type);
int rlsched_logp_fwd(int device, void* stream, const void* logits,
                     const int64_t* actions, const uint8_t* mask, float* logp,
                     float* entropy, float* stats, float* top_logp,
                     int64_t* top_index, void* scratch, int64_t rows,
                     int64_t A, int64_t x_stride, int64_t mask_stride, int k,
                     int type);
int rlsched_logp_bwd(int device, void* stream, const float* dlogp,
                     const float* dentropy, const void* logits,
                     const int64_t* actions, const uint8_t* mask,
                     const float* stats, void* dlogits, int64_t rows,
                     int64_t A, int64_t x_stride, int64_t mask_stride,
                     int type);

}  // extern "C"
