// lds_device.h -- reads of tiles in LDS by their addresses there.
#pragma once

#include "attention_device.h"

namespace iq4xs {

__device__ inline uint32_t lds_address(const void* p) {
    return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)(const_cast<void*>(p));
}

__device__ inline u4 read_row(uint32_t lds) {
    return *reinterpret_cast<__attribute__((address_space(3))) const u4*>((uintptr_t)lds);
}
// Four keys of the lane's channel: 16 lanes read 4 rows of 16 channels and each gets a column.
__device__ inline u2 read_column(uint32_t lds) {
    typedef short s4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(
        u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<__attribute__((address_space(3))) s4*>((uintptr_t)lds)));
}

}  // namespace iq4xs
