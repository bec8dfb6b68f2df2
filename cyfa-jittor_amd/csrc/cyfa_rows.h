// cyfa_rows.h -- 16-byte vectors of bf16, fp16 or fp32 rows that start anywhere:
// rows of odd lengths lie off the 16-byte grid, which gfx950's global loads and
// stores take as they are (unaligned access mode), so every row is whole
// vectors and fewer than one vector of single elements at its end.
#pragma once

#include "cyfa_device.h"

namespace cyfa {

template <class E>
struct RowVec {
    static constexpr int N = 16 / sizeof(E);
    typedef E type __attribute__((ext_vector_type(16 / sizeof(E))));
};

// PAST: of a 16-byte aligned vector that nothing reads again soon, past the caches.
template <class E, bool PAST = false>
__device__ __forceinline__ typename RowVec<E>::type load_row(const E* p) {
    typename RowVec<E>::type v;
    if (PAST)
        v = __builtin_nontemporal_load(reinterpret_cast<const typename RowVec<E>::type*>(p));
    else
        __builtin_memcpy(&v, p, 16);
    return v;
}

template <class E, bool PAST = false>
__device__ __forceinline__ void store_row(E* p, const typename RowVec<E>::type& v) {
    if (PAST)
        __builtin_nontemporal_store(v, reinterpret_cast<typename RowVec<E>::type*>(p));
    else
        __builtin_memcpy(p, &v, 16);
}

}  // namespace cyfa
