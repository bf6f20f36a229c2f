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

// The end of a call: its launches' error, if any.
inline int op_done(const char *who, const OpDevice &d) {
    const hipError_t e = d.err != hipSuccess ? d.err : hipGetLastError();
    return e == hipSuccess ? 0 : op_fail(who, hipGetErrorString(e));
}

// The operators' launches, for arguments that their entry points accept.
void launch_tree(const sp_hipkv_tree_args &a, hipStream_t s);
void launch_logprob(const sp_hipkv_logprob_args &a, hipStream_t s);
void launch_keep(const sp_hipkv_keep_args &a, hipStream_t s);

__host__ __device__ constexpr int row_bytes_of(int rows, int hd) { return rows == SP_HIPKV_ROWS_SPINOR ? spn_row_bytes(hd) : 4 * hd; }

}  // namespace kvd
