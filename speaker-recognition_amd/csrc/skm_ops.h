// skm_ops.h -- what skm_route.hip and skm_fp8.hip share: element types, device guard, wave reductions (gfx950 only).
#pragma once
#include "skm_common.h"

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

// element size of an SKM_DT_* code, 0 for an unknown one
static inline int skm_dt_size(int dt)
{
    return dt == SKM_DT_F32 ? 4 : dt == SKM_DT_BF16 || dt == SKM_DT_F16 ? 2 : dt == SKM_DT_F64 ? 8 : 0;
}

// The workgroups of 256 threads that one launch takes.  A launch has fewer than 2^32 threads along x; the runtime cuts a
// larger grid's number of threads to 32 bits without an error, so the rows behind them would have no result.  Calls
// of more rows are several launches.
#define SKM_MAX_GROUPS 0xFFFFFFL

// The launches go to the ctx's GPU whatever device the calling thread has current.
struct SkmDeviceGuard {
    int prev;
    bool changed;
    explicit SkmDeviceGuard(const SkmCtx *ctx) : prev(-1), changed(false)
    {
        if (hipGetDevice(&prev) == hipSuccess && prev != ctx->device) changed = hipSetDevice(ctx->device) == hipSuccess;
    }
    ~SkmDeviceGuard()
    {
        if (changed) (void)hipSetDevice(prev);
    }
};

// 16 bytes and the like at any address that a T may have: global memory takes unaligned vector accesses, one instruction
// where a loop over the elements is one each
template <typename V, typename T>
__device__ __forceinline__ V load_any(const T *p)
{
    V v;
    __builtin_memcpy(&v, p, sizeof(V));
    return v;
}
template <typename V, typename T>
__device__ __forceinline__ void store_any(T *p, const V &v)
{
    __builtin_memcpy(p, &v, sizeof(V));
}

// What the lanes of a wave wrote to LDS before is what its lanes read behind it.  The hardware carries a wave's LDS
// instructions out in order; this keeps the compiler from exchanging them (no instruction comes of it).
__device__ __forceinline__ void wave_sync()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <typename T>
__device__ __forceinline__ T wave_max(T v)
{
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) {
        const T o = __shfl_xor(v, m);
        v = o > v ? o : v;
    }
    return v;
}

template <typename T>
__device__ __forceinline__ T wave_sum(T v)
{
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) v += __shfl_xor(v, m);
    return v;
}
