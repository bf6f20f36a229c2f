// kvd_op.h -- what the operators on device memory (include/sp_hipkv.h) share:
// errors, the device of a call, row formats.
#pragma once
#include "sp_hipkv.h"
#include "kvd_internal.h"
#include "kvd_spinor.h"
#include <cmath>
#include <cstdio>

namespace kvd {

inline int op_fail(const char *who, const char *what) {
    char b[300];
    snprintf(b, sizeof b, "%s: %s", who, what);
    sp_set_error(b);
    return 1;
}
#define OP_NEED(cond, what) do { if (!(cond)) return op_fail(who, what); } while (0)

inline bool aligned(const void *p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// Makes the stream's device the current one for the life of a call.
class OpDevice {
    int was = -1;
    bool moved = false;
public:
    hipError_t err;
    explicit OpDevice(hipStream_t s) {
        int dev = 0;
        err = hipGetDevice(&was);
        if (err == hipSuccess && s) {
            err = hipStreamGetDevice(s, &dev);
            if (err == hipSuccess && dev != was) { err = hipSetDevice(dev); moved = err == hipSuccess; }
        }
    }
    OpDevice(const OpDevice &) = delete;
    ~OpDevice() { if (moved) hipSetDevice(was); }
};

// One launch and its own error: hipGetLastError would give, and take, an error that an
// earlier call of the same thread left.
template <typename T> struct op_param { typedef T type; };
template <typename... P>
hipError_t op_launch(void (*k)(P...), dim3 grid, dim3 wg, hipStream_t s, const typename op_param<P>::type &...p) {
    void *args[] = {const_cast<void *>(static_cast<const void *>(&p))...};
    return hipLaunchKernel(reinterpret_cast<const void *>(k), grid, wg, args, 0, s);
}

// The end of a call, e its launches' error; an error of its own is reported here and not left behind.
inline int op_done(const char *who, hipError_t e) {
    if (e == hipSuccess) return 0;
    (void)hipGetLastError();
    return op_fail(who, hipGetErrorString(e));
}

// The operators' launches, for arguments that their entry points accept.  On an error
// the launches behind it are left out.
hipError_t launch_tree(const sp_hipkv_tree_args &a, hipStream_t s);
hipError_t launch_logprob(const sp_hipkv_logprob_args &a, hipStream_t s);
hipError_t launch_keep(const sp_hipkv_keep_args &a, hipStream_t s);
hipError_t launch_append(const sp_hipkv_append_args &a, hipStream_t s);
hipError_t launch_prompt(const sp_hipkv_prompt_args &a, hipStream_t s);
hipError_t launch_cache(const sp_hipkv_cache_args &a, hipStream_t s);

__host__ __device__ constexpr int row_bytes_of(int rows, int hd) { return rows == SP_HIPKV_ROWS_SPINOR ? spn_row_bytes(hd) : 4 * hd; }

}  // namespace kvd
