// attn_host.h -- the host half that the entry points of the attention operators share.
#pragma once
#include <cuda_runtime.h>

#include <cstdio>
#include <initializer_list>

#include "../../include/fusedmm_b200.h"

namespace fmm {
namespace attn {

// the status of the CUDA error that is pending on this thread (and clears it)
inline int cuda_status()
{
   const cudaError_t e = cudaGetLastError();
   if (e == cudaSuccess) return 0;
   fprintf(stderr, "fusedmm_b200: %s\n", cudaGetErrorString(e));
   return e == cudaErrorMemoryAllocation ? FUSEDMM_B200_ERR_NOMEM : FUSEDMM_B200_ERR_CUDA;
}

// multiprocessors of the current device; 0 or a status
inline int sm_count(int *out)
{
   int dev = 0;
   if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(out, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
      cudaGetLastError();
      return FUSEDMM_B200_ERR_CUDA;
   }
   return 0;
}

// true if every pointer that is not null is memory of the current device, or managed memory
inline bool on_device(std::initializer_list<const void *> ptrs)
{
   int dev = 0;
   if (cudaGetDevice(&dev) != cudaSuccess) { cudaGetLastError(); return false; }
   for (const void *p : ptrs) {
      if (!p) continue;
      cudaPointerAttributes a;
      if (cudaPointerGetAttributes(&a, p) != cudaSuccess) { cudaGetLastError(); return false; }
      if (!(a.type == cudaMemoryTypeManaged || (a.type == cudaMemoryTypeDevice && a.device == dev))) return false;
   }
   return true;
}

// after the last launch of an entry point: its errors, and the wait of a call without a stream
inline int finish_call(void *stream)
{
   if (int s = cuda_status()) return s;
   if (!stream && cudaStreamSynchronize(nullptr) != cudaSuccess) return cuda_status();
   return 0;
}

}  // namespace attn
}  // namespace fmm
