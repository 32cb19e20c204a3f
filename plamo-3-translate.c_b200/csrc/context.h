// What the library's other translation units use of a context (struct
// plamo_cuda is private to backend.cu): its device and stream, its launch
// counter and its notes.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include "../../include/plamo_cuda.h"

namespace plamo {

// Makes the context's device current for a scope.
class ContextDevice {
public:
    explicit ContextDevice(const plamo_cuda *c);
    ~ContextDevice();
    ContextDevice(const ContextDevice &) = delete;
    ContextDevice &operator=(const ContextDevice &) = delete;

private:
    int before_, device_;
};

cudaStream_t context_stream(const plamo_cuda *c);
int context_sms(const plamo_cuda *c);
bool context_pdl(const plamo_cuda *c);
// Two device words: status bits of paged calls that were given no word of their own, and a copy being read.
uint32_t *context_paged_status(const plamo_cuda *c);
// Returns 0 (declined) with `why` in the context's note.
int context_decline(plamo_cuda *c, const char *why);
// Records an error, if any. True when there is none.
bool context_note(plamo_cuda *c, const char *what, cudaError_t e);
// Counts a launch; records its error, if any. True when it was enqueued.
bool context_launched(plamo_cuda *c, const char *what, cudaError_t e);

// Row-major 2-D tensor map [rows][cols] with a {box_cols x box_rows} box and
// 128-byte swizzle, rows row_stride elements apart (0: cols); false when the driver refuses it.
bool tensor_map_2d(CUtensorMap *map, CUtensorMapDataType type, uint32_t element_bytes, const void *ptr, uint64_t rows,
                   uint64_t cols, uint32_t box_cols, uint32_t box_rows, uint64_t row_stride = 0);

// BF16 rows of heads, [rows][heads][128], rows row_stride elements apart: boxes of 64 dimensions of box_heads heads of
// box_rows rows, 128-byte swizzle.
bool tensor_map_heads(CUtensorMap *map, const void *ptr, uint64_t rows, uint64_t heads, uint64_t row_stride, uint32_t box_heads,
                      uint32_t box_rows);

// One-time setup of the paged kernels on the context's device.
cudaError_t paged_configure();

}  // namespace plamo
