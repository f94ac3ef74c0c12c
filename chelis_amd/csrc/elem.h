// Element types of kernels that read and write any float dtype and compute
// wider: bf16 and f16 at binary32, f32 and f64 at their own width. The
// 16-bit conversions are the hardware's (nearest even, subnormals kept);
// every NaN is stored as the canonical quiet NaN of its dtype ([04-NUM-2]).
#pragma once

#include "hip_common.h"

namespace chelis {

template <typename T>
struct Wide {
    using type = float;
};
template <>
struct Wide<double> {
    using type = double;
};

template <typename T>
__device__ inline typename Wide<T>::type widen(T v) {
    return (typename Wide<T>::type)v;
}
template <typename T>
__device__ inline T finalize(typename Wide<T>::type v) {
    return (T)canon_bits(v);
}

// V elements, loaded and stored as one access that needs no more than the
// element's own alignment.
template <typename T, int V>
struct Pack {
    typedef T Q __attribute__((ext_vector_type(V)));
    typedef T U __attribute__((ext_vector_type(V), aligned(sizeof(T))));
    Q q;
    __device__ void load(const T *p) { q = *reinterpret_cast<const U *>(p); }
    __device__ void load_streamed(const T *p) { q = __builtin_nontemporal_load(reinterpret_cast<const U *>(p)); }
    __device__ void store(T *p) const { *reinterpret_cast<U *>(p) = q; }
    __device__ void store_streamed(T *p) const { __builtin_nontemporal_store(q, reinterpret_cast<U *>(p)); }
    __device__ typename Wide<T>::type get(int i) const { return widen<T>(q[i]); }
    __device__ void set(int i, typename Wide<T>::type v) { q[i] = finalize<T>(v); }
};
template <typename T>
struct Pack<T, 1> {
    T q;
    __device__ void load(const T *p) { q = *p; }
    __device__ void load_streamed(const T *p) { q = *p; }
    __device__ void store(T *p) const { *p = q; }
    __device__ void store_streamed(T *p) const { *p = q; }
    __device__ typename Wide<T>::type get(int) const { return widen<T>(q); }
    __device__ void set(int, typename Wide<T>::type v) { q = finalize<T>(v); }
};

// f(T()) with the element type of a float dtype.
template <class F>
int32_t with_elem(chelis_dtype dt, F &&f) {
    switch (dt) {
        case CHELIS_DTYPE_F32: return f(float());
        case CHELIS_DTYPE_F64: return f(double());
        case CHELIS_DTYPE_BF16: return f(__bf16());
        default: return f(_Float16());
    }
}

}  // namespace chelis
