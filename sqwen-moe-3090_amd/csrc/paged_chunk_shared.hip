// paged_chunk_shared.hip - the launch of paged_chunk.hpp's kernel for a call whose groups share
// prefixes: tiles of their members over the prefixes' keys, and of requests of many tokens over
// their own.
#include <mutex>

#include "paged_chunk.hpp"

namespace sqa {
namespace paged {

int launch_many(const Parts &c, hipStream_t s) {
    const bool opt = c.cap2 != 0.0f || c.bias != 0.0f;
    typedef void (*Kernel)(Parts);
    static const Kernel kernels[4] = {paged_many_kernel<1, false, Parts>, paged_many_kernel<2, false, Parts>,
                                      paged_many_kernel<1, true, Parts>, paged_many_kernel<2, true, Parts>};
    static std::once_flag once;  // the LDS limit is raised once per process
    static hipError_t err = hipSuccess;
    std::call_once(once, [] {
        for (Kernel k : kernels)
            if (err == hipSuccess) err = raise_chunk_lds((const void *)k);
    });
    if (err != hipSuccess) return hip_status(err, "paged_attn_shared LDS attribute");
    const int prof = profile_start("paged_shared", s);
    kernels[(c.rows_c == 128) + 2 * opt]<<<dim3((unsigned)c.grid_c), dim3(kThreads), kLdsBytes, s>>>(c);
    profile_stop(prof, s);
    return hip_status(hipGetLastError(), "paged_attn_shared launch");
}

}  // namespace paged
}  // namespace sqa
