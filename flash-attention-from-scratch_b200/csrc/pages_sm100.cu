// The cache's pages: copies of whole pages, kept tokens moved together, and the bookkeeping of who holds
// which page (forks, frees, room for new tokens).
//
// None of it computes; what bounds it is bytes for the copies and, for the rest, the latency of a few
// dependent loads. Counts are changed by integer atomics, whose order does not show; which free page
// goes where is decided by prefix sums, so that every call gives the same answer for the same state.
//
// Measured in captured graphs: a path of one sequence kept 2.9 us, the paths of a batch 7.1; one sample forked four times (fork,
// reserve, copy, free) 11.8, of which the copy is 2.0; 256 beams of 64 54.9, of which 255 pages of 0.5 MB copied are 44.1 (6.06 TB/s).
// Calls from Python take 11 to 14 us each, which is what bounds the small ones.

#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "sm100_ptx.cuh"
#include "stream_internal.h"

namespace fa_sm100 {

namespace {

// --------------------------------------------------------------------------------------- copies

constexpr int kCopyThreads = 256;

// A CTA copies one head's tokens of k or of v of a pair of pages: page_size x head_dim values on end, 8 words of 16 bytes
// a thread in flight. Bound by bytes where there are many pairs, by two dependent loads where there are few.
__global__ void __launch_bounds__(kCopyThreads) copy_kernel(const __grid_constant__ FaCopyParams p, DeviceStatus* status) {
    const FaCache& c = p.cache;
    int unit = static_cast<int>(blockIdx.x);
    const bool is_v = unit & 1;
    unit >>= 1;
    const int h = unit % c.kv_heads;
    const int i = unit / c.kv_heads;
    const int src = __ldg(p.src + i);
    const int dst = __ldg(p.dst + i);
    if (src < 0 || dst < 0) {
        return;
    }
    if (src >= c.num_pages || dst >= c.num_pages) {
        if (threadIdx.x == 0) {
            atomicOr(&status->code, kStatusBadPage);
        }
        return;
    }
    const int elem = c.dtype == FA_DTYPE_FLOAT8_E4M3 ? 1 : 2;
    const int64_t* st = is_v ? c.v_stride : c.k_stride;
    uint8_t* base = static_cast<uint8_t*>(is_v ? c.v : c.k) + h * st[1] * elem;
    const uint4* from = reinterpret_cast<const uint4*>(base + src * st[0] * elem);
    uint4* to = reinterpret_cast<uint4*>(base + dst * st[0] * elem);
    const int words = c.page_size * c.head_dim * elem / 16;
#pragma unroll 8
    for (int w = static_cast<int>(threadIdx.x); w < words; w += kCopyThreads) {
        to[w] = __ldcs(from + w);
    }
    if (elem == 1 && threadIdx.x == 0) {
        float* scale = (is_v ? c.v_scale : c.k_scale) + h;
        scale[static_cast<int64_t>(dst) * c.kv_heads] = scale[static_cast<int64_t>(src) * c.kv_heads];
    }
}

// --------------------------------------------------------------------------------- kept tokens

constexpr int kKeepThreads = 128;
constexpr int kMostTokens = 256;                          // of a call
constexpr int kMostPages = kMostTokens / 8 + 1;           // that they lie in
constexpr int kKeepWords = 4;                             // 16-byte words of a thread in flight

// A CTA moves one head's rows of k or of v of a sequence, in the order of their targets: a row's source is
// never below its target, so what a round of rows has read is all that its writes can reach. A page's
// other tokens are rescaled last, when nothing reads the old codes any more.
__global__ void __launch_bounds__(kKeepThreads) keep_kernel(const __grid_constant__ FaKeepParams p, DeviceStatus* status) {
    const FaCache& c = p.cache;
    int unit = static_cast<int>(blockIdx.x);
    const bool is_v = unit & 1;
    unit >>= 1;
    const int h = unit % c.kv_heads;
    const int b = unit / c.kv_heads;
    const bool e4m3 = c.dtype == FA_DTYPE_FLOAT8_E4M3;
    const int elem = e4m3 ? 1 : 2;
    const int log2_page = 31 - __clz(c.page_size);
    const int len = max(c.lengths[b], 0);
    const int count = c.counts != nullptr ? min(max(c.counts[b], 0), c.tokens) : c.tokens;
    const int start = len - count;
    const bool leader = threadIdx.x == 0 && h == 0 && !is_v;

    __shared__ int list[kMostTokens];
    __shared__ int kept;
    __shared__ int page_id[kMostPages];
    __shared__ float before[kMostPages], after[kMostPages];
    if (threadIdx.x == 0) {
        kept = min(p.most, c.tokens);
    }
    __syncthreads();
    for (int j = static_cast<int>(threadIdx.x); j < min(p.most, c.tokens); j += kKeepThreads) {
        const int x = __ldg(p.kept + b * p.kept_stride + j);
        const int last = j > 0 ? __ldg(p.kept + b * p.kept_stride + j - 1) : -1;
        list[j] = x;
        if (x <= last || x >= count) {
            atomicMin(&kept, j);
        }
    }
    // The pages from the first drafted token's on. A position is (start + i), its page number relative to `page0`.
    const int page0 = max(start, 0) >> log2_page;
    const int pages = count > 0 && len > 0 ? ((len - 1) >> log2_page) - page0 + 1 : 0;
    for (int i = static_cast<int>(threadIdx.x); i < pages; i += kKeepThreads) {
        int id = page0 + i < c.max_pages ? __ldg(c.page_table + b * c.table_stride + page0 + i) : -1;
        id = id >= c.num_pages ? -1 : id;
        page_id[i] = id;
        if (e4m3) {
            const float s = id < 0 ? 0.0f : (is_v ? c.v_scale : c.k_scale)[static_cast<int64_t>(id) * c.kv_heads + h];
            before[i] = s;
            after[i] = s;
        }
    }
    __syncthreads();
    const int n = kept;
    if (leader) {
        p.new_lengths[b] = start + n;
        if (n < p.most && n < c.tokens && list[n] != -1) {
            atomicOr(&status->code, kStatusBadPage);  // the row ends with what is no -1
        }
    }
    if (n == 0) {
        return;
    }
    // Whether token j moves: its places exist.
    auto place = [&](int token, int& page, int& slot) {
        const int position = start + token;
        page = position < 0 ? -1 : (position >> log2_page) - page0;
        slot = position & (c.page_size - 1);
        return position >= 0 && page_id[page] >= 0;
    };
    if (e4m3) {
        // Scales are positive, so that their order is that of their bits.
        for (int j = static_cast<int>(threadIdx.x); j < n; j += kKeepThreads) {
            int fp, fs, tp, ts;
            if (place(list[j], fp, fs) && place(j, tp, ts)) {
                atomicMax(reinterpret_cast<int*>(&after[tp]), __float_as_int(before[fp]));
            }
        }
        __syncthreads();
        for (int i = static_cast<int>(threadIdx.x); i < pages; i += kKeepThreads) {
            if (after[i] != before[i]) {
                (is_v ? c.v_scale : c.k_scale)[static_cast<int64_t>(page_id[i]) * c.kv_heads + h] = after[i];
            }
        }
    }
    const int64_t* st = is_v ? c.v_stride : c.k_stride;
    uint8_t* base = static_cast<uint8_t*>(is_v ? c.v : c.k) + h * st[1] * elem;
    const int64_t page_bytes = st[0] * elem;
    const int row_bytes = c.head_dim * elem;
    const int lanes = row_bytes / 16;  // 4, 8 or 16 threads of a row
    const int chunk = static_cast<int>(threadIdx.x) & (lanes - 1);
    const int group = static_cast<int>(threadIdx.x) / lanes;
    const int groups = kKeepThreads / lanes;
    auto rescaled = [](uint32_t w, float ratio) {
        const float2 x = unpack_half2(e4m3x2_to_half2(w & 0xFFFFu));
        const float2 y = unpack_half2(e4m3x2_to_half2(w >> 16));
        return pack_e4m3x2(x.x * ratio, x.y * ratio) | (pack_e4m3x2(y.x * ratio, y.y * ratio) << 16);
    };
    bool bad = false;
    for (int j0 = 0; j0 < n; j0 += groups * kKeepWords) {
        uint4 w[kKeepWords];
        uint8_t* to[kKeepWords];
#pragma unroll
        for (int i = 0; i < kKeepWords; ++i) {
            const int j = j0 + i * groups + group;
            to[i] = nullptr;
            if (j < n) {
                int fp, fs, tp, ts;
                const bool there = place(list[j], fp, fs);
                if (!(place(j, tp, ts) && there)) {
                    bad = true;
                } else if (list[j] != j) {
                    w[i] = *reinterpret_cast<const uint4*>(base + page_id[fp] * page_bytes + fs * row_bytes + chunk * 16);
                    to[i] = base + page_id[tp] * page_bytes + ts * row_bytes + chunk * 16;
                    if (e4m3 && before[fp] != after[tp]) {
                        const float ratio = before[fp] / after[tp];
                        w[i] = make_uint4(rescaled(w[i].x, ratio), rescaled(w[i].y, ratio), rescaled(w[i].z, ratio),
                                          rescaled(w[i].w, ratio));
                    }
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kKeepWords; ++i) {
            if (to[i] != nullptr) {
                *reinterpret_cast<uint4*>(to[i]) = w[i];
            }
        }
    }
    if (bad && chunk == 0 && h == 0 && !is_v) {
        atomicOr(&status->code, kStatusBadPage);
    }
    if (!e4m3) {
        return;
    }
    for (int i = 0; i < pages; ++i) {
        if (after[i] == before[i]) {
            continue;
        }
        const float ratio = before[i] / after[i];
        const int position0 = (page0 + i) << log2_page;
        const int filled = min(c.page_size, len - position0);
        for (int r = group; r < filled; r += groups) {
            const int token = position0 + r - start;
            if (token >= 0 && token < n && list[token] != token) {
                // A token that came in, unless its source was out of reach.
                int fp, fs;
                if (place(list[token], fp, fs)) {
                    continue;
                }
            }
            uint4* at = reinterpret_cast<uint4*>(base + page_id[i] * page_bytes + r * row_bytes + chunk * 16);
            const uint4 w = *at;
            *at = make_uint4(rescaled(w.x, ratio), rescaled(w.y, ratio), rescaled(w.z, ratio), rescaled(w.w, ratio));
        }
    }
}

// ---------------------------------------------------------------------------------- bookkeeping

constexpr int kPageThreads = 256;

// A thread an entry.
__global__ void __launch_bounds__(kPageThreads) fork_kernel(const __grid_constant__ FaPages p, DeviceStatus* status) {
    const long long at = static_cast<long long>(blockIdx.x) * kPageThreads + threadIdx.x;
    const int b = static_cast<int>(at / p.width);
    const int i = static_cast<int>(at - static_cast<long long>(b) * p.width);
    if (b >= p.batch) {
        return;
    }
    const int row = __ldg(p.rows + b);
    int id = -1;
    bool bad = row < -1 || row >= p.from_batch;
    if (row >= 0 && !bad) {
        id = __ldg(p.from + row * p.from_stride + i);
        bad = id < -1 || id >= p.num_pages;
    }
    if (bad) {
        atomicOr(&status->code, kStatusBadPage);
        id = -1;
    }
    if (id >= 0) {
        atomicAdd(p.refs + id, 1);
    }
    p.table[b * p.table_stride + i] = id;
}

__global__ void __launch_bounds__(kPageThreads) free_kernel(const __grid_constant__ FaPages p, DeviceStatus* status) {
    const long long at = static_cast<long long>(blockIdx.x) * kPageThreads + threadIdx.x;
    const int b = static_cast<int>(at / p.width);
    const int i = static_cast<int>(at - static_cast<long long>(b) * p.width);
    if (b >= p.batch || (p.keep != nullptr && i < __ldg(p.keep + b))) {
        return;
    }
    int32_t* entry = p.table + b * p.table_stride + i;
    const int id = *entry;
    if (id == -1) {
        return;
    }
    bool bad = id < 0 || id >= p.num_pages;
    if (!bad && atomicSub(p.refs + id, 1) <= 0) {
        atomicAdd(p.refs + id, 1);  // it had none left to give
        bad = true;
    }
    if (bad) {
        atomicOr(&status->code, kStatusBadPage);
    }
    *entry = -1;
}

constexpr int kReserveThreads = 1024;

// Entries of a row that get new tokens: at most so many, and no more than the row has.
__host__ __device__ __forceinline__ int reserve_entries(const FaPages& p) {
    const int most = (p.tokens + p.page_size - 2) / p.page_size + 1;
    return most < p.width ? most : p.width;
}

// Exclusive prefix sum over the CTA and the total. All threads call.
__device__ __forceinline__ int block_prefix(int mine, int& total) {
    __shared__ int warp_sum[kReserveThreads / 32];
    const int lane = static_cast<int>(threadIdx.x) % 32;
    const int warp = static_cast<int>(threadIdx.x) / 32;
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, incl, o);
        incl += lane >= o ? up : 0;
    }
    __syncthreads();  // the last call's sums have been read
    if (lane == 31) {
        warp_sum[warp] = incl;
    }
    __syncthreads();
    int sum = warp_sum[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, sum, o);
        sum += lane >= o ? up : 0;
    }
    total = __shfl_sync(0xffffffffu, sum, 31);
    const int before = __shfl_sync(0xffffffffu, sum, warp > 0 ? warp - 1 : 0);
    return incl - mine + (warp > 0 ? before : 0);
}

// Entries [first, end) of a row that get new tokens; empty where the row cannot be served at all (`fits` false).
struct NewEntries {
    int first, end;
    bool fits, older;  // older: the first of them holds older tokens
};

__device__ __forceinline__ NewEntries new_entries(const FaPages& p, int b) {
    NewEntries e;
    const int len = p.lengths[b];
    const int count = p.counts != nullptr ? min(max(p.counts[b], 0), p.tokens) : p.tokens;
    const int log2_page = 31 - __clz(p.page_size);
    const long long start = static_cast<long long>(len) - count;
    e.fits = start >= 0 && len <= static_cast<long long>(p.width) * p.page_size;
    e.first = e.fits ? static_cast<int>(start >> log2_page) : 0;
    e.end = e.fits && count > 0 ? ((len - 1) >> log2_page) + 1 : e.first;
    e.older = (start & (p.page_size - 1)) != 0;
    return e;
}

// The new entries of all rows, row after row, and for each the rank of the free page that it needs; then the free pages
// as far as they are needed; then the pages' new places: three passes of one CTA with barriers between them, since needs
// and free pages are those that the call finds. Several CTAs would need a launch a pass (2 us each) and save part of 4 to
// 6 us, up to some ten thousand entries. Entries are taken in order, four a thread, so that a long prompt's are not one
// thread's. Workspace: before[batch + 1] (needs of the rows before), rank[batch][entries] (-1: none needed), free[...].
__global__ void __launch_bounds__(kReserveThreads) reserve_kernel(const __grid_constant__ FaPages p, DeviceStatus* status,
                                                                  int32_t* before, int32_t* rank, int32_t* free_list) {
    const int entries = reserve_entries(p);
    const long long all = static_cast<long long>(p.batch) * entries;
    int needed = 0;
    for (long long at0 = 0; at0 < all; at0 += 4 * kReserveThreads) {
        bool want[4];
        int mine = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const long long at = at0 + 4 * static_cast<int>(threadIdx.x) + k;
            want[k] = false;
            if (at < all) {
                const int b = static_cast<int>(at / entries);
                const NewEntries e = new_entries(p, b);
                const int i = e.first + static_cast<int>(at - static_cast<long long>(b) * entries);
                if (i < e.end) {
                    const int id = p.table[b * p.table_stride + i];
                    const bool bad = id < -1 || id >= p.num_pages;
                    if (bad) {
                        atomicOr(&status->code, kStatusBadPage);
                    }
                    want[k] = id < 0 || bad || p.refs[id] > 1;
                }
            }
            mine += want[k];
        }
        int total;
        int next = needed + block_prefix(mine, total);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const long long at = at0 + 4 * static_cast<int>(threadIdx.x) + k;
            if (at < all) {
                rank[at] = want[k] ? next : -1;
                if (at % entries == 0) {
                    before[at / entries] = next;
                }
            }
            next += want[k];
        }
        needed += total;
    }
    if (threadIdx.x == 0) {
        before[p.batch] = needed;
    }
    // Free pages in order, as many as are needed.
    int found = 0;
    for (int i0 = 0; i0 < p.num_pages && found < needed; i0 += 4 * kReserveThreads) {
        const int i = i0 + 4 * static_cast<int>(threadIdx.x);
        bool is_free[4];
        int mine = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            is_free[k] = i + k < p.num_pages && p.refs[i + k] == 0;
            mine += is_free[k];
        }
        int total;
        int next = found + block_prefix(mine, total);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (is_free[k]) {
                if (next < needed) {
                    free_list[next] = i + k;
                }
                ++next;
            }
        }
        found += total;
    }
    __syncthreads();
    for (long long at = threadIdx.x; at < all; at += kReserveThreads) {
        const int b = static_cast<int>(at / entries);
        const int nth = static_cast<int>(at - static_cast<long long>(b) * entries);
        const NewEntries e = new_entries(p, b);
        const bool granted = e.fits && (before[b + 1] == before[b] || before[b + 1] <= found);
        int src = -1, dst = -1;
        if (granted && rank[at] >= 0) {
            int32_t* entry = p.table + b * p.table_stride + e.first + nth;
            const int id = *entry;
            const int page = free_list[rank[at]];
            if (id >= 0 && id < p.num_pages) {
                atomicSub(p.refs + id, 1);
                if (nth == 0 && e.older) {
                    src = id;
                    dst = page;
                }
            }
            p.refs[page] = 1;
            *entry = page;
        }
        if (nth == 0) {
            if (!e.fits) {
                atomicOr(&status->code, kStatusBadPage);
            }
            p.granted[b] = granted;
            p.src[b] = src;
            p.dst[b] = dst;
        }
    }
}

// Parts of the reserve workspace, each on 16 bytes.
unsigned long long rounded(unsigned long long n) { return (n + 15) / 16 * 16; }

}  // namespace

cudaError_t launch_copy_pages(const FaCopyParams& p, DeviceStatus* status, cudaStream_t stream) {
    const long long grid = 2ll * p.count * p.cache.kv_heads;
    if (grid > 0x7fffffffLL) {
        return cudaErrorInvalidConfiguration;
    }
    copy_kernel<<<static_cast<unsigned>(grid), kCopyThreads, 0, stream>>>(p, status);
    return cudaGetLastError();
}

cudaError_t launch_keep_tokens(const FaKeepParams& p, DeviceStatus* status, cudaStream_t stream) {
    const long long grid = 2ll * p.cache.batch * p.cache.kv_heads;
    if (grid > 0x7fffffffLL) {
        return cudaErrorInvalidConfiguration;
    }
    keep_kernel<<<static_cast<unsigned>(grid), kKeepThreads, 0, stream>>>(p, status);
    return cudaGetLastError();
}

cudaError_t launch_fork_pages(const FaPages& p, DeviceStatus* status, cudaStream_t stream) {
    const long long grid = (static_cast<long long>(p.batch) * p.width + kPageThreads - 1) / kPageThreads;
    if (grid > 0x7fffffffLL) {
        return cudaErrorInvalidConfiguration;
    }
    fork_kernel<<<static_cast<unsigned>(grid), kPageThreads, 0, stream>>>(p, status);
    return cudaGetLastError();
}

cudaError_t launch_free_pages(const FaPages& p, DeviceStatus* status, cudaStream_t stream) {
    const long long grid = (static_cast<long long>(p.batch) * p.width + kPageThreads - 1) / kPageThreads;
    if (grid > 0x7fffffffLL) {
        return cudaErrorInvalidConfiguration;
    }
    free_kernel<<<static_cast<unsigned>(grid), kPageThreads, 0, stream>>>(p, status);
    return cudaGetLastError();
}

unsigned long long reserve_workspace_bytes(const FaPages& p) {
    const unsigned long long all = static_cast<unsigned long long>(p.batch) * reserve_entries(p);
    return rounded(4ull * (p.batch + 1ull)) + rounded(4ull * all) + 4ull * std::min<unsigned long long>(all, p.num_pages);
}

cudaError_t launch_reserve_pages(const FaPages& p, DeviceStatus* status, void* workspace, cudaStream_t stream) {
    uint8_t* at = static_cast<uint8_t*>(workspace);
    int32_t* before = reinterpret_cast<int32_t*>(at);
    at += rounded(4ull * (p.batch + 1ull));
    int32_t* rank = reinterpret_cast<int32_t*>(at);
    at += rounded(4ull * p.batch * reserve_entries(p));
    reserve_kernel<<<1, kReserveThreads, 0, stream>>>(p, status, before, rank, reinterpret_cast<int32_t*>(at));
    return cudaGetLastError();
}

}  // namespace fa_sm100
