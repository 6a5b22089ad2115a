// thork_internal.h — declarations shared by the host-side translation units of
// libthork_rt.so (not part of the public C-ABI).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

int thork_set_error(int code, const char *fmt, ...);
int thork_cuda_error(cudaError_t e, const char *what);
int thork_encode_tmap_2d(void *out128, int dtype, const void *base, uint64_t rows, uint64_t cols,
                         uint64_t row_stride_bytes, uint32_t box_rows, uint32_t box_cols,
                         int swizzle_bytes);
// Dense 3-D tensor map (d0 innermost, in elements) with a box0 x box1 x 1 box
// and 128-byte swizzle; out128 is 64-byte aligned.
int thork_encode_tmap_3d(void *out128, int dtype, const void *base, uint64_t d0, uint64_t d1, uint64_t d2,
                         uint32_t box0, uint32_t box1);
// Per-device status word (4 x u32, cudaMalloc'd and zeroed on first use).
int thork_status_word(unsigned **d_status);
// The linear-layer operators' status word, one per device in page-locked host
// memory that kernels write when something went wrong: the host reads it after
// a wait for the stream without a copy (a synchronising linear of 16 x 4096 x
// 4096 took 19.7 us without a read, 28-29 with one of a word on the device).
int thork_host_status_word(unsigned **word);
// Cached multiprocessor count of the current device.
int thork_sm_count(int *n);
// Pipelined copies through pinned slots for pageable host memory (staging.cu).
bool thork_is_pageable(const void *host_ptr);
size_t thork_staged_min_bytes();
int thork_staged_htod(void *d_dst, const void *h_src, size_t n, cudaStream_t s);
int thork_staged_dtoh(void *h_dst, const void *d_src, size_t n, cudaStream_t s);
