// serve.cuh -- shared by the serving operators' files (kv_pages.cu, kv8.cu,
// attn_prompt.cu, attn_prefix.cu, attn_kv8.cu, spec_verify.cu, beam_select.cu): argument checks, the
// device's view of a paged cache, launches.
#pragma once

#include <atomic>
#include <cuda_runtime.h>
#include <cuda_fp16.h>

#include "backend.cuh"
#include "common.cuh"

namespace sllm {

constexpr int kServeDim = 128;      // the head dimension of every model the library runs
constexpr float kServeScale = 0.08838834764831845f;     // 1 / sqrt(128)

// OK when p is memory of the current device (a kernel given a host pointer or
// another device's would fault); the message names the argument.
int need_device(const void* p, const char* who, const char* arg);

// the fields of a sllm_cuda_kv_pages, checked (no device call); and whether its
// values are 8-bit codes or not, as the caller takes them
int check_pages(const sllm_cuda_kv_pages* p, const char* who);
int check_pages(const sllm_cuda_kv_pages* p, const char* who, bool eight);

// the error words of the attention kernels' bounded waits, read and cleared
int take_prompt_error();
int take_prefix_error();
int take_kv8_error();
// the limit of those waits for the next launches (2 s; tests set a short one), and
// of one try's sleep, ns
struct WaitLimit {
    uint32_t ns, nap;
};
WaitLimit attn_wait_limit();

int current_sms();

// an attribute of a kernel, set once per device
template <auto Kernel, cudaFuncAttribute Attr>
cudaError_t set_once(int value) {
    static std::atomic<unsigned long long> done{0};
    int dev = 0;
    const cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const unsigned long long bit = dev < 64 ? 1ull << dev : 0;
    if (bit != 0 && (done.load(std::memory_order_relaxed) & bit) != 0) return cudaSuccess;
    const cudaError_t r = cudaFuncSetAttribute(Kernel, Attr, value);
    if (r == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
    return r;
}
template <auto Kernel>
cudaError_t allow_smem(int bytes) { return set_once<Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize>(bytes); }
// clusters of 16 CTAs
template <auto Kernel>
cudaError_t allow_cluster() { return set_once<Kernel, cudaFuncAttributeNonPortableClusterSizeAllowed>(1); }

struct PagesDev {
    int32_t* refs;
    int32_t* tables;
    int32_t* lens;
    int n_pages, n_slots, width, page;
    int cap;                        // width * page: the most tokens a slot holds
};

inline PagesDev pages_dev(const sllm_cuda_kv_pages& p) {
    return PagesDev{p.refs, p.tables, p.lens, p.n_pages, p.n_slots, p.table_width, p.page_size,
                    p.table_width * p.page_size};
}

inline size_t kv_elt_bytes(int type) { return type == SLLM_CUDA_KV_I8 ? 1 : type == SLLM_CUDA_KV_F16 ? 2 : 4; }

constexpr int kKvBlock = 16;        // tokens that share a scale of an 8-bit cache

// sets *status (nullable) to an error; it is never cleared here
__device__ __forceinline__ void raise(int32_t* status, int code) {
    if (status != nullptr) *status = code;
}

// a kernel launch; pdl: the launch may start while the kernel before it on
// the stream still runs, and orders itself with griddepcontrol.wait
template <class... KArgs, class... Args>
cudaError_t launch(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, bool pdl,
                   Args... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = pdl ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, KArgs(args)...);
}

__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_trigger() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
template <class T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <class T> __device__ __forceinline__ void from_f32_to(T* p, float x) { *p = from_f32<T>(x); }

// four consecutive elements as floats (8- or 16-byte aligned)
__device__ __forceinline__ float4 ld4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 ld4(const __half* p) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&u.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
    return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ void st4(float* p, float4 v) { *reinterpret_cast<float4*>(p) = v; }
__device__ __forceinline__ void st4(__half* p, float4 v) {
    const __half2 a = __floats2half2_rn(v.x, v.y), b = __floats2half2_rn(v.z, v.w);
    uint2 u;
    u.x = *reinterpret_cast<const uint32_t*>(&a);
    u.y = *reinterpret_cast<const uint32_t*>(&b);
    *reinterpret_cast<uint2*>(p) = u;
}

}  // namespace sllm
