// Internal interface of the sequence operators: crnn_seq_api.hip (C entry points, argument checks), crnn_seq.hip (kernels),
// crnn_api.hip (the handle).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/crnn_hip.h"

namespace crnn {

// Makes the handle's device current for a call and the caller's again after it.
struct SeqDevice {
  int before = -1;
  ~SeqDevice();
};
// Device state and current device for a call on `stream` (locked: the caller holds the handle's mutex).
int seq_enter(crnn_handle* h, void* stream, SeqDevice* dev, bool need_weights = false, bool locked = false);
int seq_fail(crnn_handle* h, int code, const char* msg);

void launch_warm_seq(hipStream_t s);
void launch_linear(const crnn_linear_args& a, hipStream_t s);
void launch_rms_norm(const crnn_rms_norm_args& a, hipStream_t s);
int64_t cross_attention_workspace(const crnn_cross_attention_args& a);
void launch_cross_attention(const crnn_cross_attention_args& a, hipStream_t s);
// out [n,T,512] = rec, zeros from tlen[i] on; out_len (may be null) = tlen, T where tlen is null
void launch_copy_states(const void* rec, void* out, int32_t* out_len, const int32_t* tlen, int n, int T, bool b16,
                        hipStream_t s);

}  // namespace crnn
