// Shared device helpers for the sm_100a kernels: PTX wrappers for asynchronous copies,
// shared-memory matrix loads and the bf16 warp-level MMA, plus launch-error bookkeeping.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <utility>

#include "../../include/gaudirt_b200.h"

namespace gk {

// cudaError_t of the last failed launch on this host thread.
extern thread_local int g_last_cuda_error;

inline int check_launch() {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    g_last_cuda_error = static_cast<int>(e);
    return GK_ERR_CUDA;
  }
  return GK_OK;
}

// The opt-in for more than 48 KB of dynamic shared memory is per device and has to be made once
// before the first launch there.  `done` is one flag per device ordinal; the entry points may be
// called from several host threads, so the flags are atomics (setting the attribute twice is
// harmless, reading a half-written flag would not be).
template <typename Kernel>
inline int opt_in_shared_memory(Kernel kernel, int bytes, std::atomic<bool> (&done)[64]) {
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return check_launch();
  const bool tracked = device >= 0 && device < 64;
  if (tracked && done[device].load(std::memory_order_acquire)) return GK_OK;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
    return check_launch();
  if (tracked) done[device].store(true, std::memory_order_release);
  return GK_OK;
}

// Programmatic dependent launch.  A kernel launched through launch_after_predecessor may be set up on
// the GPU while the kernel before it in the stream is still running; its first statement is
// wait_for_predecessor(), which lets the kernel AFTER it start its own set-up and then blocks until the
// kernel before it has completed and its writes are visible, so every access of the kernel body is
// ordered exactly as by plain stream order.  What overlaps is the launch latency and the scheduling of
// the CTAs, which is most of a decode layer's gap between kernels.  Launched the ordinary way (or with
// the switch off) both instructions do nothing.
extern std::atomic<int> g_programmatic_launch;

__device__ __forceinline__ void wait_for_predecessor() {
  asm volatile("griddepcontrol.launch_dependents;\ngriddepcontrol.wait;\n" ::: "memory");
}

template <typename... Params, typename... Args>
inline void launch_programmatic(bool on, void (*kernel)(Params...), dim3 grid, dim3 block, size_t shared_bytes,
                                cudaStream_t stream, Args&&... args) {
  cudaLaunchConfig_t config{};
  config.gridDim = grid;
  config.blockDim = block;
  config.dynamicSmemBytes = shared_bytes;
  config.stream = stream;
  cudaLaunchAttribute attribute[1];
  attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute[0].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attribute;
  config.numAttrs = on ? 1 : 0;
  (void)cudaLaunchKernelEx(&config, kernel, static_cast<Params>(args)...);   // the caller reads the error with check_launch()
}

template <typename... Params, typename... Args>
inline void launch_after_predecessor(void (*kernel)(Params...), dim3 grid, dim3 block, size_t shared_bytes,
                                     cudaStream_t stream, Args&&... args) {
  launch_programmatic(g_programmatic_launch.load(std::memory_order_relaxed) != 0, kernel, grid, block, shared_bytes, stream,
                      std::forward<Args>(args)...);
}

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

// 16-byte asynchronous global->shared copy, bypassing L1.  With src_bytes == 0 nothing is
// read and the 16 destination bytes are zero-filled.
__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src, int src_bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(src_bytes)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory");
}

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

// D(16x8, fp32) += A(16x16, bf16, row) * B(16x8, bf16, col)
__device__ __forceinline__ void mma_bf16_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);   // .x = lo (low 16 bits)
  return *reinterpret_cast<const uint32_t*>(&v);
}

__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}

// softcap * tanh(scale * s / softcap) in log2 units, from tanh(x) = 1 - 2 / (exp(2x) + 1): `e` is 2 log2(e) scale / softcap
// and `c` softcap * log2(e).  Both ends come out exactly (exp2 gives 0 or infinity).  The absolute error is a few 2^-23 of
// the cap whatever the score: a few 2^-22 of the result where |scale * s / softcap| is above 1/2, and 2^-14 (of a score
// that enters an exponential, where a probability's rounding to bf16 is 2^-9) up to kTightCap.  At a cap of 10^6 it would be
// 0.2 of a score of ordinary size.
constexpr float kTightCap = 256.f;
__device__ __forceinline__ float capped_large_score(float s, float e, float c) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(r) : "f"(fast_exp2(s * e) + 1.f));
  return fmaf(-2.f * c, r, c);
}

// The same for two scores with |scale * s / softcap| <= 1/2 (`in` = scale / softcap, `out` = scale * log2(e)), from the
// series of tanh: the first term left out is 21844/6081075 x^12 of the result, under 9e-7 of it, so the error is relative to
// the score and does not know the cap.  Multiplies instead of the two special-function instructions per score.
__device__ __forceinline__ float2 capped_small_scores(float2 s, float in, float out) {
  const float2 x = __fmul2_rn(s, make_float2(in, in)), y = __fmul2_rn(x, x);
  float2 t = make_float2(-1382.f / 155925.f, -1382.f / 155925.f);
  t = __ffma2_rn(t, y, make_float2(62.f / 2835.f, 62.f / 2835.f));
  t = __ffma2_rn(t, y, make_float2(-17.f / 315.f, -17.f / 315.f));
  t = __ffma2_rn(t, y, make_float2(2.f / 15.f, 2.f / 15.f));
  t = __ffma2_rn(t, y, make_float2(-1.f / 3.f, -1.f / 3.f));
  t = __ffma2_rn(t, y, make_float2(1.f, 1.f));
  return __fmul2_rn(t, __fmul2_rn(s, make_float2(out, out)));
}

// Two scores under a cap above kTightCap, each by its own size, so that one huge score does not cost its neighbours their
// digits.  Tight caps need only the logistic form: 460 against 542 us where most scores are past half a cap of 1 (4 chunks of
// up to 1024 rows on 4096 tokens, 32 query / 8 KV heads, head_dim 128).
__device__ __forceinline__ float2 capped_scores(float2 s, float in, float out, float e, float c) {
  const float2 small = capped_small_scores(s, in, out);
  return make_float2(fabsf(s.x * in) <= 0.5f ? small.x : capped_large_score(s.x, e, c),
                     fabsf(s.y * in) <= 0.5f ? small.y : capped_large_score(s.y, e, c));
}

}  // namespace gk
