// skv_tree.cuh -- tree attention over the engine's own records.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/seoulkv_b200.h"

namespace skv {

// The K and V maps of one cell's FP8 records [rows][512] (K | V).
int record_maps(CUtensorMap *two, const uint8_t *records, int64_t rows);
// Attention over a cache given by `d`, or (cells != null: device array of the K
// and V maps of every cell) over FP8 records with the context at `tlen`.
// `status` (null: the device's word) gets the bits of waits that
// gave up.
int tree_attention(const SkvTree *d, const CUtensorMap *cells, const int32_t *tlen, uint32_t *status, cudaStream_t st);

}  // namespace skv
