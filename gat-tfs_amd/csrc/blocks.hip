// Block tables of a paged cache: pages taken and given back, slots and positions of a step's rows.
//
//   had = ceil(cached / page),  need = ceil((cached + fresh) / page) - had
//   pages of request r: free[count - 1 - k], k from the exclusive sum of need;  slot = table[pos / page] page + pos % page
//
// Bound by a launch and its chain of dependent reads (lengths, sums over the requests, a row's request, its page):
// one block forms the sums over the requests, 4096 at a time, and, where the batch is small, goes on with the
// rows from LDS; else a second launch finds each row's request by bisection.  A new block's page is taken from the
// list by each of its rows, so that no row waits for the table; the row at offset 0 writes it there.
//
// A step of 12 requests: 5.0 us.  2500 prompts of 471 thousand rows: sums 6.9 us, rows 5.6; 300 requests that end 2.5 + 3.5.
#include <algorithm>
#include <string>

#include "cache.hpp"
#include "cache_index.hpp"

namespace gatgpu {
namespace {

constexpr int kScan = 1024;                        // threads of a block that sums
// Requests of each of them at a time, where there are more than 1024 (1024 at once: four each 8.5 us, one 8.0).
constexpr uint32_t kEach = 4;
// Rows that the block of the sums takes itself.  64 requests of 16 rows: 5.5 us, in two launches 7.6; of 64 rows 8.3 and 7.6.
constexpr uint32_t kOneBlockRows = 2048;
// Requests of a release in one block.  8 requests: 4.0 us, in two launches 4.7; 32 4.8 and 5.1; 64 6.4 and 5.0.
constexpr uint32_t kOneBlockRelease = 32;
// Counts that each block of a release sums itself.  16384: 24 us, by one block between 33; 32768 54 and 61, 65536 154 and 115.
constexpr uint32_t kFewCounts = 32768;
constexpr uint32_t kMaxRequests = 1u << 20;

struct BlocksArgs {
    uint32_t requests = 0, page_log = 0, pages = 0, rows = 0, blocks = 0;
    uint64_t ld = 0;
    const uint32_t *cached = nullptr, *fresh = nullptr, *free_count = nullptr;
    uint32_t *table = nullptr, *free = nullptr, *free_left = nullptr, *stored = nullptr, *k_len = nullptr, *q_begin = nullptr, *slot = nullptr,
             *position = nullptr, *unserved = nullptr;
    uint32_t* behind = nullptr;  // workspace: [requests] pages taken (given back) before each request's
    uint32_t* count = nullptr;   // workspace: [1] pages in the list at the start
};

struct Sums {
    uint64_t pages, rows;
};
// Inclusive sums over the block's threads; `total`: of all of them.
__device__ inline Sums block_sums(Sums x, Sums& total) {
    __shared__ Sums wave_total[kScan / kWave];
    const int lane = int(threadIdx.x) % kWave, wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / kWave);
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) {
        const uint64_t p = __shfl_up(x.pages, d), r = __shfl_up(x.rows, d);
        if (lane >= d) {
            x.pages += p;
            x.rows += r;
        }
    }
    __syncthreads();  // (the totals of the call before have been read)
    if (lane == kWave - 1) wave_total[wave] = x;
    __syncthreads();
    // A lane a wave's total: sums up to this wave, and of all.
    Sums t = lane < kScan / kWave ? wave_total[lane] : Sums{0, 0};
#pragma unroll
    for (int d = 1; d < kScan / kWave; d *= 2) {
        const uint64_t p = __shfl_up(t.pages, d), r = __shfl_up(t.rows, d);
        if (lane >= d) {
            t.pages += p;
            t.rows += r;
        }
    }
    total = {__shfl(t.pages, kScan / kWave - 1), __shfl(t.rows, kScan / kWave - 1)};
    if (wave) {
        x.pages += __shfl(t.pages, wave - 1);
        x.rows += __shfl(t.rows, wave - 1);
    }
    return x;
}

// One row's slot and position.  begin, k_len, behind: its request's.
__device__ inline void assign_row(const BlocksArgs& a, uint32_t row, uint32_t request, uint32_t begin, uint32_t end, uint32_t k_len, uint32_t behind,
                                  uint32_t count) {
    uint32_t slot = GATGPU_NO_PAGE, pos = 0;
    if (row >= begin && row < end && k_len) {
        const uint32_t cached = k_len - (end - begin), page = 1u << a.page_log, had = uint32_t((uint64_t(cached) + page - 1) >> a.page_log);
        pos = cached + (row - begin);
        const uint32_t block = pos >> a.page_log;
        uint32_t* const at = a.table + uint64_t(request) * a.ld + block;
        uint32_t p;
        if (block >= had) {
            p = a.free[count - 1 - (behind + (block - had))];
            if (!(pos & (page - 1))) *at = p;
        } else {
            p = *at;
        }
        if (p < a.pages) slot = (p << a.page_log) + (pos & (page - 1));
    }
    a.slot[row] = slot;
    a.position[row] = pos;
}
// The last i of [lo, hi] with begin[i] <= row, for begin[lo] <= row (equal begins: the last).
template <class P>
__device__ inline uint32_t find_request(P begin, uint32_t lo, uint32_t hi, uint32_t row) {
    while (lo < hi) {
        const uint32_t mid = lo + (hi - lo + 1) / 2;
        if (begin[mid] <= row) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// Sums over the requests, EACH of a thread at a time; ROWS: the rows as well (at most kScan requests).
template <bool ROWS, uint32_t EACH>
__global__ __launch_bounds__(kScan) void k_blocks_assign(const BlocksArgs a) {
    __shared__ uint32_t s_left, s_unserved;
    __shared__ uint32_t s_begin[ROWS ? kScan + 1 : 1], s_len[ROWS ? kScan : 1], s_behind[ROWS ? kScan : 1];
    const uint32_t tid = threadIdx.x;
    const uint32_t count = min(*a.free_count, a.pages);
    if (tid == 0) {
        s_left = count;
        s_unserved = 0;
        a.q_begin[0] = 0;
        if (ROWS) s_begin[0] = 0;
    }
    __syncthreads();
    Sums before = {0, 0};
    uint32_t left = count, unserved = 0;  // after the thread's requests that take pages, and of the wave's
    for (uint32_t first = 0; first < a.requests; first += kScan * EACH) {
        const uint64_t page = uint64_t(1) << a.page_log;
        uint64_t c[EACH], f[EACH], need[EACH];
        Sums own = {0, 0};
#pragma unroll
        for (uint32_t i = 0; i < EACH; ++i) {
            const uint32_t r = first + tid * EACH + i;
            c[i] = r < a.requests ? a.cached[r] : 0;
            f[i] = r < a.requests ? a.fresh[r] : 0;
        }
#pragma unroll
        for (uint32_t i = 0; i < EACH; ++i) {
            const bool fits = c[i] + f[i] <= uint64_t(a.blocks) << a.page_log;
            need[i] = fits ? ((c[i] + f[i] + page - 1) >> a.page_log) - ((c[i] + page - 1) >> a.page_log) : 0;
            own.pages += need[i];
            own.rows += f[i];
        }
        Sums total;
        const Sums all = block_sums(own, total);
        Sums upto = {before.pages + all.pages - own.pages, before.rows + all.rows - own.rows};
        before.pages += total.pages;
        before.rows += total.rows;
#pragma unroll
        for (uint32_t i = 0; i < EACH; ++i) {
            const uint32_t r = first + tid * EACH + i;
            upto.pages += need[i];
            upto.rows += f[i];
            const bool fits = c[i] + f[i] <= uint64_t(a.blocks) << a.page_log;
            const bool served = fits && (need[i] == 0 || upto.pages <= count) && upto.rows <= a.rows;
            unserved += uint32_t(__popcll(__ballot(r < a.requests && !served)));
            if (r >= a.requests) continue;
            const uint32_t behind = uint32_t(upto.pages - need[i]), len = served ? uint32_t(c[i] + f[i]) : 0;
            const uint32_t end = upto.rows > 0xffffffffu ? 0xffffffffu : uint32_t(upto.rows);
            a.stored[r] = uint32_t(served ? c[i] + f[i] : c[i]);
            a.k_len[r] = len;
            a.q_begin[r + 1] = end;
            if (ROWS) {
                s_begin[r + 1] = end;
                s_len[r] = len;
                s_behind[r] = behind;
            } else {
                a.behind[r] = behind;
            }
            if (served && need[i]) left = count - uint32_t(upto.pages);  // (less with each request, so the least of all threads' counts)
        }
    }
#pragma unroll
    for (int d = kWave / 2; d; d /= 2) left = min(left, uint32_t(__shfl_xor(int(left), d)));
    if (tid % kWave == 0) {
        atomicMin(&s_left, left);
        atomicAdd(&s_unserved, unserved);
    }
    __syncthreads();
    if (tid == 0) {
        if (!ROWS) *a.count = count;
        *a.free_left = s_left;
        *a.unserved = s_unserved;
    }
    if constexpr (ROWS) {
        for (uint32_t row = tid; row < a.rows; row += kScan) {
            const uint32_t q = find_request(s_begin, 0, a.requests, row);
            if (q < a.requests) assign_row(a, row, q, s_begin[q], s_begin[q + 1], s_len[q], s_behind[q], count);
            else assign_row(a, row, 0, 0, 0, 0, 0, count);
        }
    }
}

// Rows of many requests: the requests of a block's first and last row bound its other rows'.
__global__ __launch_bounds__(256) void k_blocks_rows(const BlocksArgs a) {
    __shared__ uint32_t s_ends[2];
    const uint32_t count = *a.count, tid = threadIdx.x;
    for (uint64_t first = uint64_t(blockIdx.x) * 256; first < a.rows; first += uint64_t(gridDim.x) * 256) {
        const uint32_t last = index_min(first + 255, a.rows - 1), row = uint32_t(first) + tid;
        if (tid < 2 * kWave) {
            const uint32_t end = last_at_most(a.q_begin, a.requests + 1, tid < kWave ? uint32_t(first) : last, int(tid % kWave));
            if (tid % kWave == 0) s_ends[tid / kWave] = end;
        }
        __syncthreads();
        if (row <= last) {
            const uint32_t q = find_request(a.q_begin, s_ends[0], s_ends[1], row);
            if (q < a.requests) assign_row(a, row, q, a.q_begin[q], a.q_begin[q + 1], a.k_len[q], a.behind[q], count);
            else assign_row(a, row, 0, 0, 0, 0, 0, count);
        }
        __syncthreads();
    }
}

// Blocks of a table row that hold its request's tokens.
__device__ inline uint32_t held_blocks(const BlocksArgs& a, uint32_t r) {
    const uint64_t n = (uint64_t(a.cached[r]) + (uint64_t(1) << a.page_log) - 1) >> a.page_log;
    return uint32_t(n < a.blocks ? n : a.blocks);
}
// A wave's count of the pages in request r's row; WRITE: into the list from `place` on.
template <bool WRITE>
__device__ inline uint32_t give_back(const BlocksArgs& a, uint32_t r, uint64_t place) {
    const int lane = int(threadIdx.x) % kWave;
    const uint32_t n = held_blocks(a, r);
    uint32_t found = 0;
    for (uint32_t b = 0; b < n; b += kWave) {
        const uint32_t p = b + uint32_t(lane) < n ? a.table[uint64_t(r) * a.ld + b + uint32_t(lane)] : GATGPU_NO_PAGE;
        const uint64_t some = __ballot(p < a.pages);
        if (WRITE && p < a.pages) {
            const uint64_t at = place + found + uint64_t(__popcll(some & ((uint64_t(1) << lane) - 1)));
            if (at < a.pages) a.free[at] = p;
        }
        found += uint32_t(__popcll(some));
    }
    return found;
}
__global__ __launch_bounds__(256) void k_release_count(const BlocksArgs a) {
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.count = min(*a.free_count, a.pages);
    const uint32_t r = blockIdx.x * 4 + threadIdx.x / kWave;
    if (r >= a.requests) return;
    const uint32_t n = give_back<false>(a, r, 0);
    if (threadIdx.x % kWave == 0) a.behind[r] = n;
}
// A block's four requests, behind the sum of the counts before them.
__global__ __launch_bounds__(256) void k_release_write(const BlocksArgs a) {
    __shared__ uint64_t s_sum[4];
    const uint32_t first = blockIdx.x * 4, wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    uint64_t sum = 0;
    for (uint32_t r = threadIdx.x; r < first; r += 256) sum += a.behind[r];
#pragma unroll
    for (int d = kWave / 2; d; d /= 2) sum += __shfl_xor(sum, d);
    if (lane == 0) s_sum[wave] = sum;
    __syncthreads();
    uint64_t place = uint64_t(*a.count) + s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3];
    for (uint32_t r = first; r < a.requests && r < first + 4; ++r) {
        if (r == first + wave) (void)give_back<true>(a, r, place);
        place += a.behind[r];
    }
    if (blockIdx.x == gridDim.x - 1 && threadIdx.x == 0) *a.free_left = index_min(place, a.pages);
}
// Counts to sums; ALL: counts and writes too (at most kOneBlockRelease requests).
template <bool ALL>
__global__ __launch_bounds__(kScan) void k_release(const BlocksArgs a) {
    __shared__ uint32_t s_count[ALL ? kOneBlockRelease : 1];
    const uint32_t tid = threadIdx.x, count = ALL ? min(*a.free_count, a.pages) : *a.count;
    if constexpr (ALL) {
        for (uint32_t r = tid / kWave; r < a.requests; r += kScan / kWave) {
            const uint32_t n = give_back<false>(a, r, 0);
            if (tid % kWave == 0) s_count[r] = n;
        }
    }
    __syncthreads();
    uint64_t before = 0;
    for (uint32_t first = 0; first < a.requests; first += kScan) {
        const uint32_t r = first + tid;
        const uint32_t n = r >= a.requests ? 0 : ALL ? s_count[ALL ? r : 0] : a.behind[r];
        Sums total;
        const Sums upto = block_sums({n, 0}, total);
        // (what stands beyond the list's `pages` places is not written, so 32 bits do)
        const uint32_t behind = uint32_t(min(before + upto.pages - n, uint64_t(0xffffffffu)));
        if (r < a.requests) {
            if (ALL) s_count[ALL ? r : 0] = behind;
            else a.behind[r] = behind;
        }
        before += total.pages;
    }
    __syncthreads();
    if (tid == 0) {
        *a.free_left = uint32_t(min(uint64_t(count) + before, uint64_t(a.pages)));
    }
    if constexpr (ALL)
        for (uint32_t r = tid / kWave; r < a.requests; r += kScan / kWave) (void)give_back<true>(a, r, uint64_t(count) + s_count[r]);
}
// The same, behind sums that k_release has formed.
__global__ __launch_bounds__(256) void k_release_place(const BlocksArgs a) {
    const uint32_t r = blockIdx.x * 4 + threadIdx.x / kWave;
    if (r < a.requests) (void)give_back<true>(a, r, uint64_t(*a.count) + a.behind[r]);
}

}  // namespace
}  // namespace gatgpu

namespace {

using namespace gatgpu;

int check_words(gatgpu_ctx* c, const char* name, const void* p, uint64_t n = 1) {
    if (!n) return GATGPU_OK;
    if (!p) return fail(c, GATGPU_EINVAL, std::string("null ") + name);
    if (reinterpret_cast<uintptr_t>(p) % 4) return fail(c, GATGPU_EINVAL, std::string(name) + " must be 4-byte aligned");
    return check_device_array(c, p, name);
}
int check_sizes(gatgpu_ctx* c, const gatgpu_blocks_io* io) {
    if (!io) return fail(c, GATGPU_EINVAL, "null arrays");
    if (io->requests > kMaxRequests) return fail(c, GATGPU_EOVERFLOW, "more than 2^20 requests");
    if (io->page < 16 || io->page > 256 || (io->page & (io->page - 1))) return fail(c, GATGPU_EINVAL, "page must be 16, 32, 64, 128 or 256");
    if (uint64_t(io->pages) * io->page >= (uint64_t(1) << 32)) return fail(c, GATGPU_EOVERFLOW, "pages * page must be below 2^32");
    if (uint64_t(io->blocks) * io->page >= (uint64_t(1) << 32)) return fail(c, GATGPU_EOVERFLOW, "blocks * page must be below 2^32");
    if (io->table_stride < io->blocks || io->table_stride > (uint64_t(1) << 40)) return fail(c, GATGPU_EINVAL, "table has a bad row stride");
    return GATGPU_OK;
}
uint64_t blocks_bytes(const gatgpu_blocks_io* io) { return (uint64_t(io->requests) + 1 + 3) / 4 * 16; }

int check_call(gatgpu_ctx* c, const gatgpu_blocks_io* io, void* ws, uint64_t bytes) {
    if (int r = check_sizes(c, io)) return r;
    if (int r = check_words(c, "cached", io->cached, io->requests)) return r;
    if (int r = check_words(c, "table", io->table, uint64_t(io->requests) * io->blocks)) return r;
    if (int r = check_words(c, "free", io->free, io->pages)) return r;
    if (int r = check_words(c, "free_count", io->free_count)) return r;
    if (int r = check_words(c, "free_left", io->free_left)) return r;
    const uint64_t need = blocks_bytes(io);
    if (bytes < need) return fail(c, GATGPU_EINVAL, "workspace of " + std::to_string(bytes) + " bytes, " + std::to_string(need) + " needed");
    if (!ws || reinterpret_cast<uintptr_t>(ws) % 16) return fail(c, GATGPU_EINVAL, "workspace must be 16-byte aligned device memory");
    return check_device_array(c, ws, "workspace");
}
BlocksArgs make_args(const gatgpu_blocks_io* io, void* ws) {
    BlocksArgs a;
    a.requests = io->requests;
    while ((1u << a.page_log) < io->page) ++a.page_log;
    a.pages = io->pages;
    a.rows = io->rows;
    a.blocks = io->blocks;
    a.ld = io->table_stride;
    a.cached = io->cached;
    a.fresh = io->fresh;
    a.free_count = io->free_count;
    a.table = io->table;
    a.free = io->free;
    a.free_left = io->free_left;
    a.stored = io->stored;
    a.k_len = io->k_len;
    a.q_begin = io->q_begin;
    a.slot = io->slot;
    a.position = io->position;
    a.unserved = io->unserved;
    a.behind = static_cast<uint32_t*>(ws);
    a.count = a.behind + io->requests;
    return a;
}

}  // namespace

extern "C" {

int gatgpu_blocks_workspace(gatgpu_ctx* c, const gatgpu_blocks_io* io, uint64_t* bytes) {
    if (!c) return fail(nullptr, GATGPU_EINVAL, "null context");
    if (!bytes) return fail(c, GATGPU_EINVAL, "null output");
    if (int r = check_sizes(c, io)) return r;
    *bytes = blocks_bytes(io);
    return GATGPU_OK;
}

int gatgpu_blocks_assign(gatgpu_ctx* c, const gatgpu_blocks_io* io, void* ws, uint64_t bytes) {
    if (!c) return fail(nullptr, GATGPU_EINVAL, "null context");
    DeviceGuard on(c->device);
    if (!on.ok) return fail(c, GATGPU_EDEVICE, "cannot select the context's device");
    if (int r = check_call(c, io, ws, bytes)) return r;
    if (int r = check_words(c, "fresh", io->fresh, io->requests)) return r;
    if (int r = check_words(c, "stored", io->stored, io->requests)) return r;
    if (int r = check_words(c, "k_len", io->k_len, io->requests)) return r;
    if (int r = check_words(c, "q_begin", io->q_begin)) return r;
    if (int r = check_words(c, "slot", io->slot, io->rows)) return r;
    if (int r = check_words(c, "position", io->position, io->rows)) return r;
    if (int r = check_words(c, "unserved", io->unserved)) return r;
    const BlocksArgs a = make_args(io, ws);
    if (a.requests <= uint32_t(kScan) && a.rows <= kOneBlockRows) {
        k_blocks_assign<true, 1><<<1, kScan, 0, c->stream>>>(a);
        HIPCHECK(c, hipGetLastError());
        return GATGPU_OK;
    }
    if (a.requests <= uint32_t(kScan)) k_blocks_assign<false, 1><<<1, kScan, 0, c->stream>>>(a);
    else k_blocks_assign<false, kEach><<<1, kScan, 0, c->stream>>>(a);
    HIPCHECK(c, hipGetLastError());
    if (!a.rows) return GATGPU_OK;
    k_blocks_rows<<<index_min((uint64_t(a.rows) + 255) / 256, 1u << 14), 256, 0, c->stream>>>(a);
    HIPCHECK(c, hipGetLastError());
    return GATGPU_OK;
}

int gatgpu_blocks_release(gatgpu_ctx* c, const gatgpu_blocks_io* io, void* ws, uint64_t bytes) {
    if (!c) return fail(nullptr, GATGPU_EINVAL, "null context");
    DeviceGuard on(c->device);
    if (!on.ok) return fail(c, GATGPU_EDEVICE, "cannot select the context's device");
    if (int r = check_call(c, io, ws, bytes)) return r;
    const BlocksArgs a = make_args(io, ws);
    if (a.requests <= kOneBlockRelease) {
        k_release<true><<<1, kScan, 0, c->stream>>>(a);
        HIPCHECK(c, hipGetLastError());
        return GATGPU_OK;
    }
    k_release_count<<<(a.requests + 3) / 4, 256, 0, c->stream>>>(a);
    HIPCHECK(c, hipGetLastError());
    if (a.requests <= kFewCounts) {
        k_release_write<<<(a.requests + 3) / 4, 256, 0, c->stream>>>(a);
        HIPCHECK(c, hipGetLastError());
        return GATGPU_OK;
    }
    k_release<false><<<1, kScan, 0, c->stream>>>(a);
    HIPCHECK(c, hipGetLastError());
    k_release_place<<<(a.requests + 3) / 4, 256, 0, c->stream>>>(a);
    HIPCHECK(c, hipGetLastError());
    return GATGPU_OK;
}

}  // extern "C"
