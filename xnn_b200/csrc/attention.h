// Host entry points of the structure-attention kernels (attention.cu, attention_tc*.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace attn {

template <typename T> struct Params;

template <typename T> cudaError_t forward(const Params<T>&, cudaStream_t);
template <typename T> cudaError_t forward_join(const Params<T>&, cudaStream_t);
template <typename T> cudaError_t sum_splits(int64_t n, int splits, const T* work, T* out0, T* out1, cudaStream_t);
template <typename T> cudaError_t backward_short(const Params<T>&, cudaStream_t);
template <typename T> cudaError_t second_short(const Params<T>&, cudaStream_t);

// float64 on the FP64 tensor instructions, and the second derivative of wide float32 heads in 64 bits (attention_f64.cu)
cudaError_t forward64(const Params<double>&, cudaStream_t);
cudaError_t backward64(const Params<double>&, cudaStream_t);
template <typename T> int64_t second64_words(const Params<T>&);
template <typename T> cudaError_t second64(const Params<T>&, double* work, cudaStream_t);

// tensor-core forms for float32; `work` holds the operands' images (the byte counts say how much), `status` is set
// where a bounded wait ran out
int64_t tc_forward_bytes(const Params<float>&);
int64_t tc_backward_bytes(const Params<float>&);
cudaError_t tc_forward(const Params<float>&, char* work, int* status, cudaStream_t);
cudaError_t tc_backward(const Params<float>&, char* work, int* status, cudaStream_t);
cudaError_t tc_wide_backward(const Params<float>&, char* work, int* status, cudaStream_t);   // 65 .. 128 columns, images written
int64_t tc_second_bytes(const Params<float>&);
cudaError_t tc_second(const Params<float>&, char* work, int* status, cudaStream_t);          // up to 64 columns

}  // namespace attn
