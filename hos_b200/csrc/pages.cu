// Pages of a cache copied to other pages, in all arrays of a group of layers in one launch: array a is `n_pages` pages of
// bytes[a] each at address[a]; pair p copies page src[p] to page dst[p] of every array.  Nothing but bytes moves, so a page may hold
// numbers of any type.  A pair with a page outside the arrays, or with src == dst, copies nothing (a list may be padded with -1); no
// page may be written twice, or read and written, in one launch.
// Bound by memory: a block asks for 32 KB before it writes any (100 pages in 46 arrays of 16 kv heads of 128, 1.2 GB read and 1.2 written: 367 us,
// the rate of a plain copy); a handful of pages by the launch.
#include "common.cuh"

namespace hos {

constexpr int kCopyThreads = 256, kCopyUnroll = 8;
constexpr int kCopyBytes = kCopyThreads * kCopyUnroll * 16;       // 32 KB a block

__global__ void __launch_bounds__(kCopyThreads)
copy_pages_kernel(const long long* __restrict__ table, const int* __restrict__ src, const int* __restrict__ dst, int n_pages) {
    pdl_enter();
    const int p = blockIdx.z, a = blockIdx.y;
    const int from = src[p], to = dst[p];
    if (from < 0 || to < 0 || from >= n_pages || to >= n_pages || from == to) return;
    const long long bytes = table[2 * a + 1];
    const long long at = (long long)blockIdx.x * kCopyBytes + threadIdx.x * 16;
    const char* s = (const char*)table[2 * a] + from * bytes;
    char* d = (char*)table[2 * a] + to * bytes;
    uint4 v[kCopyUnroll];
#pragma unroll
    for (int i = 0; i < kCopyUnroll; ++i)
        if (at + i * kCopyThreads * 16 < bytes) v[i] = *(const uint4*)(s + at + i * kCopyThreads * 16);
#pragma unroll
    for (int i = 0; i < kCopyUnroll; ++i)
        if (at + i * kCopyThreads * 16 < bytes) *(uint4*)(d + at + i * kCopyThreads * 16) = v[i];
}

}  // namespace hos

using namespace hos;

// table: int64 [n_arrays][2] on the device (address, bytes of a page); most_bytes: the largest of the pages' sizes, all multiples of 16.
extern "C" int hos_copy_pages(const long long* table, int n_arrays, long long most_bytes, const int* src, const int* dst, int n_pairs, int n_pages,
                              cudaStream_t stream) {
    if (n_pairs <= 0 || n_arrays <= 0) return 0;
    if (most_bytes <= 0 || most_bytes % 16) HOS_REFUSE("copy_pages: pages of %lld bytes (multiples of 16)", most_bytes);
    if (n_arrays > 65535) HOS_REFUSE("copy_pages: %d arrays", n_arrays);
    for (int lo = 0; lo < n_pairs; lo += 65535) {
        const int n = n_pairs - lo < 65535 ? n_pairs - lo : 65535;
        launch_pdl(copy_pages_kernel, dim3((unsigned)((most_bytes + kCopyBytes - 1) / kCopyBytes), (unsigned)n_arrays, (unsigned)n), dim3(kCopyThreads), 0, stream,
                   table, src + lo, dst + lo, n_pages);
    }
    return check_launch("copy_pages");
}
