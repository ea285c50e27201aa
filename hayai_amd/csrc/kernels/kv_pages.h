// Where a page's keys and values lie.  A page holds its keys as [heads][tokens][dim] and its values
// turned, as [heads][dim][tokens]: both operands of an attention's products, keys by queries and
// weights by values, are then 16 bytes of neighbours of the summed axis in memory, so they go to the
// matrix cores without a transposition in registers or LDS.
#ifndef HH_KERNELS_KV_PAGES_H
#define HH_KERNELS_KV_PAGES_H

#include "act_types.h"

typedef uint32_t hh_u4 __attribute__((ext_vector_type(4)));

// Bytes from a page's start to its keys' (head h, token t) and its values' (head h, element d) rows.
template <class C>
HH_DEV uint32_t hh_kv_key(const hh_kv_args& a, uint32_t h, uint32_t t) {
    return (((h << a.shift) + t) * a.dim) * (uint32_t)sizeof(typename C::E);
}
template <class C>
HH_DEV uint32_t hh_kv_value(const hh_kv_args& a, uint32_t h, uint32_t d) {
    return (((a.heads + h) * a.dim + d) << a.shift) * (uint32_t)sizeof(typename C::E);
}

#endif
