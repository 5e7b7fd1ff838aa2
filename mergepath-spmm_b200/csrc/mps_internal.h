// Shared by the translation units of libmps_b200.so; not part of the public ABI.
#pragma once
#include <stdint.h>

#include <atomic>

#include "mps.h"

namespace mps {
// Records a printf-style message for mps_last_error() on this thread and returns `code`.
int fail(int code, const char *fmt, ...);

// Host-side scans of a caller's CSR (host_check.cpp), each on up to `threads` host threads (0 = all):
// index of the first row whose row_ptr decreases / of the first column index outside [0, n_cols), or -1.
long long first_decreasing_row(const int32_t *row_ptr, long long n_rows, int threads);
long long first_bad_column(const int32_t *col_idx, long long nnz, int32_t n_cols, int threads);
int32_t max_column(const int32_t *col_idx, long long nnz, int threads);
// row_ptr[0] == 0, row_ptr non-decreasing, every column index inside [0, n_cols) (col_idx may be NULL): MPS_OK or
// MPS_ERR_ARG with the offending position in the message.
int check_csr_host(const char *who, int32_t n_rows, int32_t n_cols, const int32_t *row_ptr, const int32_t *col_idx, int threads);
// A value that is looked up once per device and then kept for the life of the process (a function's attribute that was set, an
// address): get() is 0 until put() was called on that device.
template <typename T>
struct PerDevice {
    static constexpr int kDevices = 64;
    std::atomic<T> value[kDevices] = {};
    T get(int device) const { return device >= 0 && device < kDevices ? value[device].load(std::memory_order_acquire) : T(); }
    void put(int device, T v) {
        if (device >= 0 && device < kDevices) value[device].store(v, std::memory_order_release);
    }
};

// SMs of the current device (mps_route.cu).
int sm_count(int *n);
// Status word of the routing kernels on the current device (mps_route.cu): waits for the stream, returns it and clears it.
int take_route_status(void *stream, int *status);
// Rows listed by id as by mps_group_rows (device arrays), those without a valid id as a last group behind the others:
// group_ptr has n_groups + 2 entries (mps_route.cu).
int list_rows_and_rest(int n_rows, int n_groups, const int32_t *ids, int32_t *group_ptr, int32_t *slot_row, void *stream);
}  // namespace mps
