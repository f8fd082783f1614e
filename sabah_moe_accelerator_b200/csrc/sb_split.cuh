// A list of places cut into equal parts, for a kernel whose warps each take one.
// A list has from 1 to 2^31 - 1 places, so no sum here goes past its end.
#pragma once

#include <cuda_runtime.h>

// a / b; the integer division is a long subroutine, and most numbers here are small
__host__ __device__ inline int div_fast(int a, int b) {
#ifdef __CUDA_ARCH__
    if (a >= 1 << 22) return (int)((unsigned)a / (unsigned)b);
    int q = (int)__fdividef((float)a, (float)b);   // within one of the quotient
    q -= q * b > a;
    return q + (a - q * b >= b);
#else
    return a / b;
#endif
}
// places of a part, at least `least`
__host__ __device__ inline int part_of(int places, int warps, int least) {
    const int part = div_fast(places - 1, warps) + 1;
    return part > least ? part : least;
}
// how many parts there are
__host__ __device__ inline int parts_in(int places, int part) { return div_fast(places - 1, part) + 1; }
// where part w ends; it starts at w * part
__host__ __device__ inline int part_end(int places, int part, int w) {
    return places - w * part > part ? w * part + part : places;
}
