// Library-internal helpers shared by the translation units of libvidax_cuda.so.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

// Records `msg` as the calling thread's last error (vx_last_error) and
// returns `code`.
int vx_internal_fail(int code, const char* msg);

// The same, printf-style, and for a CUDA error (VX_ECUDA).
int vx_internal_failf(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int vx_internal_cuda_fail(cudaError_t e, const char* what);

// Device address of the current device's status word (the one
// vx_device_status reads), looked up once per device.
int vx_internal_status_word(int** out);

// The current device, its SM count, and a kernel's dynamic shared memory
// limit (raised once per kernel and device).
int vx_internal_device(int* dev, int* sms);
int vx_internal_prepare_kernel(const void* fn, int dev, size_t smem);

// 2-D tensor map over `rows` rows of `row_bytes` bytes, `stride` bytes apart,
// of elements of `elem` (1, 2 or 4) bytes, in boxes of box_bytes (128, 64 or
// 32, swizzled over that width) x box_rows; loads read 0 past the end, stores
// are clipped there.
int vx_internal_byte_tmap(CUtensorMap* tm, const void* base, uint64_t row_bytes, uint64_t rows,
                          uint64_t stride, uint32_t box_bytes, uint32_t box_rows, int elem = 1);
