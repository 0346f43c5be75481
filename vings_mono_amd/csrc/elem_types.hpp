// 16-byte accesses to rows of float32, bfloat16 and float16 elements.  The vector types are
// declared with their element's alignment: gfx950 serves a 16-byte global access at any element
// boundary, so views that start inside a larger array need no path of their own.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace vings {

enum ElemType { ELEM_F32 = 0, ELEM_BF16 = 1, ELEM_F16 = 2 };   // VINGS_F32 / _BF16 / _F16

template <typename T> struct Elem;
template <> struct Elem<float> {
    static constexpr int kVec = 4;
    typedef float vec __attribute__((ext_vector_type(4), aligned(4)));
};
template <> struct Elem<__bf16> {
    static constexpr int kVec = 8;
    typedef __bf16 vec __attribute__((ext_vector_type(8), aligned(2)));
};
template <> struct Elem<_Float16> {
    static constexpr int kVec = 8;
    typedef _Float16 vec __attribute__((ext_vector_type(8), aligned(2)));
};

static inline int elem_bytes(int type) { return type == ELEM_F32 ? 4 : 2; }
static inline bool elem_known(int type) { return type >= ELEM_F32 && type <= ELEM_F16; }

}  // namespace vings
