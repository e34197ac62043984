// adapters.hip -- low-rank adapters of many requests beside a shared projection (gfx950).
//
// y_r = base_r + s_a B_a (A_a x_r), with a = which[r] the row's own adapter, A_a of rank x cols and B_a of
// out x rank.  Rows without an adapter are base_r.
#include <algorithm>

#include "paged_ops.h"

namespace mh {
namespace {

constexpr int kThreads = 256;

template <class T>
__device__ __forceinline__ float get(const T *p) {
    if constexpr (sizeof(T) == 2)
        return __half2float(*(const __half *)p);
    else
        return *p;
}
template <class T>
__device__ __forceinline__ void put(T *p, float x) {
    if constexpr (sizeof(T) == 2)
        *p = __float2half_rn(x);
    else
        *p = x;
}

// A workgroup a row and a share of its outputs.
template <class X, class Y>
__global__ __launch_bounds__(kThreads) void adapter_kernel(AdapterArgs a) {
    __shared__ float t[kAdapterRankMax];
    const int r = blockIdx.x, w = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int id = a.which[r];
    const bool has = id >= 0 && id < a.n;
    const int rank = !has ? 0 : (a.rank == nullptr ? a.max_rank : min(max(a.rank[id], 0), a.max_rank));
    const X *x = (const X *)a.x + r * a.x_row;
    for (int k = w; k < rank; k += kThreads / 64) {
        const __half *row = (const __half *)a.a + ((size_t)id * a.max_rank + k) * a.cols;
        float sum = 0.0f;
        for (int c = lane; c < a.cols; c += 64) sum = fmaf(get(x + c), __half2float(row[c]), sum);
        sum = wave_sum(sum);
        if (lane == 0) t[k] = sum;
    }
    __syncthreads();
    const float scale = !has || a.scale == nullptr ? 1.0f : a.scale[id];
    for (int o = blockIdx.y * kThreads + threadIdx.x; o < a.out; o += gridDim.y * kThreads) {
        float sum = 0.0f;
        if (has) {
            const __half *row = (const __half *)a.b + ((size_t)id * a.out + o) * a.max_rank;
            for (int k = 0; k < rank; ++k) sum = fmaf(t[k], __half2float(row[k]), sum);
        }
        const float base = get((const Y *)a.base + r * a.base_row + o);
        put((Y *)a.y + r * a.y_row + o, has ? fmaf(scale, sum, base) : base);
    }
}

template <class X, class Y>
hipError_t launch(const AdapterArgs &a, hipStream_t s) {
    (void)hipGetLastError();
    hipLaunchKernelGGL((adapter_kernel<X, Y>), dim3(a.rows, std::min((a.out + kThreads - 1) / kThreads, 16)), dim3(kThreads), 0, s, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_adapter_rows(const AdapterArgs &a, hipStream_t s) {
    if (a.x_dtype == ELEM_F16) return a.y_dtype == ELEM_F16 ? launch<__half, __half>(a, s) : launch<__half, float>(a, s);
    return a.y_dtype == ELEM_F16 ? launch<float, __half>(a, s) : launch<float, float>(a, s);
}

}  // namespace mh
