// 8-bit checkpoints inside the library.
#pragma once

#include "common.hpp"

namespace glt {

// glt_ckpt8_swiglu with inter wanted for the columns of [lo, hi) only; what it
// holds elsewhere is undefined.
glt_status ckpt8_swiglu(const void* gate8, const void* up8, int64_t rows, int32_t cols, uint16_t* gate, uint16_t* up,
                        uint16_t* inter, int lo, int hi, hipStream_t st);

}  // namespace glt
