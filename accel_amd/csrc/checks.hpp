// What the operator layer's checks share: tensors' names in messages and the
// refusal itself.  Included into one anonymous namespace per translation unit.
#pragma once

#include <string>

#include "internal.hpp"

namespace accel {
namespace {

const char* dtype_name(int32_t d) {
    switch (d) {
        case ACCEL_F32: return "f32";
        case ACCEL_F16: return "f16";
        case ACCEL_BF16: return "bf16";
        case ACCEL_U32: return "u32";
        case ACCEL_I8: return "i8";
        default: return "an unknown dtype";
    }
}

std::string shape_str(const accel_tensor_t* t) {
    std::string s = "[";
    for (int i = 0; i < t->rank && i < 4; i++) {
        if (i) s += ' ';
        s += std::to_string((long long)t->shape[i]);
    }
    return s + "]";
}

int64_t elements(const accel_tensor_t* t) {
    int64_t n = 1;
    for (int i = 0; i < t->rank && i < 4; i++) n *= t->shape[i];
    return n;
}

int refuse(const char* op, const std::string& why) {
    return fail(ACCEL_E_INVALID, "accel/tensor: %s: %s", op, why.c_str());
}

bool valid_tensor(const accel_tensor_t* t) {
    return t && t->rank >= 0 && t->rank <= 4;
}

}  // namespace
}  // namespace accel
