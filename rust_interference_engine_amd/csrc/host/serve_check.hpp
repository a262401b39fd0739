// serve_check.hpp — what the C ABI of the batched serving operators checks before a launch.
#pragma once

#include "../../../include/rie_hip.h"

#include "../serve.hpp"
#include "guard.hpp"

#include <algorithm>
#include <string>

namespace rie {

inline Error bad(const std::string &m) { return Error{E_RUNTIME, m}; }

// The stream's device is the current one while this lives.
class OnDevice {
  public:
    explicit OnDevice(hipStream_t st) {
        RIE_HIP_CHECK(hipGetDevice(&was_));
        device = was_;
        if (st) {
            hipDevice_t d;
            RIE_HIP_CHECK(hipStreamGetDevice(st, &d));
            device = (int)d;
        }
        if (device != was_) RIE_HIP_CHECK(hipSetDevice(device));
    }
    ~OnDevice() {
        if (device != was_) (void)hipSetDevice(was_);
    }
    OnDevice(const OnDevice &) = delete;
    OnDevice &operator=(const OnDevice &) = delete;

    // p is memory that a kernel on this device may use
    void check(const void *p, const char *what) const {
        if (!p) throw bad(std::string(what) + " is NULL");
        hipPointerAttribute_t a;
        const hipError_t e = hipPointerGetAttributes(&a, p);
        if (e != hipSuccess) (void)hipGetLastError();  // not an error of the launch
        if (e != hipSuccess || (a.type != hipMemoryTypeDevice && a.type != hipMemoryTypeManaged))
            throw bad(std::string(what) + " is not device memory");
        if (a.type == hipMemoryTypeDevice && a.device != device)
            throw bad(std::string(what) + " is on device " + std::to_string(a.device) + ", the stream on device " + std::to_string(device));
    }

    int device;

  private:
    int was_;
};

inline bool is16(int ty) { return ty == T_F16 || ty == T_BF16; }

// A dimension of one entry is at 0, whatever its stride says (that of a tensor's is arbitrary)
inline int64_t used(int64_t n, int64_t stride) { return n > 1 ? stride : 0; }

// Rows of values of es bytes each start at p + any multiples of the strides: all 16-byte
// aligned, and strides of 2^26 bytes at most, so that 16 rows stay within 31 bits
inline void check_rows(const void *p, int64_t row, int64_t head, int es, const char *what) {
    const int64_t a = 16 / es, most = ((int64_t)1 << 26) / es;
    if ((uintptr_t)p % 16 || row % a || head % a) throw bad(std::string(what) + ": rows have to be 16-byte aligned");
    if (row < 0 || row > most || head < 0 || head > most) throw bad(std::string(what) + ": strides have to lie in 0.." + std::to_string(most));
}

// Rows that are written, n of each dimension a stride apart: no two of them share a value.  Every
// stride has to cover what the smaller ones span.
struct Dim {
    int64_t n, stride;
};
template <size_t N>
void check_apart(Dim (&&dims)[N], int hd, const char *what) {
    std::sort(dims, dims + N, [](const Dim &a, const Dim &b) { return a.stride < b.stride; });
    __int128 span = hd;  // strides of up to 2^40 by counts of up to 2^31
    for (const Dim &d : dims) {
        if (d.n <= 1) continue;
        if (d.stride < span) throw bad(std::string(what) + ": strides below head_dim, or below what the smaller ones span, would make rows overlap");
        span += (__int128)(d.n - 1) * d.stride;
    }
}

constexpr int MOST = 1 << 30;  // positions
constexpr int MOST_ROWS = (1 << 26) - 4;  // 4 to a workgroup of 256: a launch has under 2^32 threads

inline BatchView batch(const rie_hip_seqs *s, bool lens) {
    if (!s) throw bad("seqs is NULL");
    if (s->n_seq < 1 || s->n_rows < 1 || s->n_seq >= 1 << 24 || s->n_rows > MOST_ROWS) throw bad("n_seq has to lie in 1..2^24-1, n_rows in 1..2^26-4");
    if (s->max_new < 1 || s->max_len < 1 || s->max_new > MOST || s->max_len > MOST) throw bad("max_new and max_len have to lie in 1..2^30");
    BatchView b;
    b.starts = s->starts;
    b.lens = lens ? s->lens : nullptr;
    b.n_seq = s->n_seq;
    b.n_rows = s->n_rows;
    b.max_new = std::min(s->max_new, s->n_rows);
    b.max_len = s->max_len;
    return b;
}

}  // namespace rie
