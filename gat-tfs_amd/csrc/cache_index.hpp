// Where the rows of a request and the bytes of its pages lie: plain arithmetic on what the caller's device arrays hold,
// clamped so that nothing outside the arrays is reached whatever they hold.  (A host compiler takes it too.)
#pragma once
#include <cstdint>

#ifdef __HIPCC__
#define GATGPU_INDEX __host__ __device__ inline
#else
#define GATGPU_INDEX inline
#endif

namespace gatgpu {

constexpr uint32_t kCacheTile = 64, kCacheRows = 16;  // keys a step, packed rows a wave
constexpr uint32_t kNoPage = 0xffffffffu;             // GATGPU_NO_PAGE

struct CacheSizes {
    uint64_t rows = 0;  // of q and out
    uint32_t requests = 0, most = 0, blocks = 0, pages = 0, page_log = 0;
    uint32_t heads = 0, kv_heads = 0, group = 0, dim = 0;
};

GATGPU_INDEX uint32_t index_min(uint64_t a, uint64_t b) { return uint32_t(a < b ? a : b); }

// One request of a call.
struct CacheRequest {
    uint32_t begin = 0, rows = 0, keys = 0;  // first row, rows that are computed, tokens
    int64_t shift = 0;                       // position of row 0
};
GATGPU_INDEX CacheRequest cache_request(const CacheSizes& c, uint32_t begin, uint32_t end, uint32_t k_len) {
    CacheRequest q;
    const uint32_t lo = index_min(begin, c.rows), hi = index_min(end, c.rows), len = hi > lo ? hi - lo : 0;
    q.begin = lo;
    q.rows = len < c.most ? len : c.most;
    q.keys = index_min(k_len, uint64_t(c.blocks) << c.page_log);
    q.shift = int64_t(q.keys) - int64_t(len);
    return q;
}
// Keys that row i of a request sees.
GATGPU_INDEX uint32_t cache_seen(const CacheRequest& q, uint32_t i) {
    const int64_t n = q.shift + int64_t(i) + 1;
    return n < 0 ? 0u : uint32_t(n);
}
// Tiles of a request: of keys (one, if it has none), and of its packed rows.
GATGPU_INDEX uint32_t key_tiles(const CacheRequest& q) { return q.keys ? (q.keys - 1) / kCacheTile + 1 : 1; }
GATGPU_INDEX uint32_t row_tiles(const CacheSizes& c, const CacheRequest& q) {
    return uint32_t((uint64_t(q.rows) * c.group + kCacheRows - 1) / kCacheRows);
}

// Index in the request's table row of the page of `key`, kNoPage beyond its tokens.
GATGPU_INDEX uint32_t block_of(const CacheSizes& c, uint32_t keys, uint32_t key) { return key < keys ? key >> c.page_log : kNoPage; }
// A page to take bytes from where a table entry is none: those bytes count for nothing.
GATGPU_INDEX uint32_t some_page(const CacheSizes& c, uint32_t page) { return page < c.pages ? page : 0; }
// Byte of a key's first column, and of column `col`'s entry for a key, in the keys' and the values' bytes.
GATGPU_INDEX uint64_t key_byte(const CacheSizes& c, uint32_t page, uint32_t head, uint32_t key) {
    return (((uint64_t(page) * c.kv_heads + head) << c.page_log) + (key & ((1u << c.page_log) - 1))) * c.dim;
}
GATGPU_INDEX uint64_t value_byte(const CacheSizes& c, uint32_t page, uint32_t head, uint32_t key, uint32_t col) {
    return (((uint64_t(page) * c.kv_heads + head) * c.dim + col) << c.page_log) + (key & ((1u << c.page_log) - 1));
}

}  // namespace gatgpu
