// The tensor-core form of the packed attention (packed_tc.cu) for sequences of many rows of an f16 or 8-bit pool, as packed.cu launches it.
#pragma once
#include "packed.cuh"

constexpr uint32_t PACKED_TC_ROWS = 256;     // rows of an item
constexpr uint32_t PACKED_TC_MIN_ROWS = 33;  // sequences of fewer rows are the other kernel's
// (16 sequences behind 3000 positions, the other kernel against this one: 32 rows f16 88 against 90 us, 8 bit 97 against 108; 48 rows 118 against 92, 138 against 111)

// one block per SM; part: two slots of PACKED_TC_ROWS rows each; notes: one each
int32_t brasa_packed_tc_launch(brasa_cmd *cmd, const brasa_dev::PackedView &v, int32_t kv, const float *q, const uint8_t *kpool, const uint8_t *vpool, void *o,
                               float *part, brasa_dev::PackedNote *notes, uint32_t hq, float scale);
