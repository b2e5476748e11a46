// Segment attention: plans and C entry points (declarations: include/gatgpu.h).
#include "attention.hpp"

#include <algorithm>
#include <cmath>
#include <memory>
#include <new>
#include <numeric>
#include <string>

struct gatgpu_attention {
    gatgpu_ctx* ctx = nullptr;
    gatgpu_attention_shape shape{};
    std::vector<gatgpu::AttnSeg> segs;
    uint64_t rows = 0, keys = 0, dist_bytes = 0;
    bool shared_keys = false;  // key rows of two segments overlap
    // Tables on the device: segments; tiles of the forward, the query and the key pass; joined tiles.
    // Short segments: forward of one and two blocks of 32 keys, backward of 1, 2 and 4 waves.
    gatgpu::DevBuf dsegs, dsmall[2], dsmall_bwd[3], dfwd, dbwd_q, dbwd_kv, djoin, djoin_q, djoin_kv;
    uint32_t own_delta = 0;  // segments of so many keys need no rest: their backward pass forms delta from its weights
    uint64_t nsmall[2] = {}, nsmall_bwd[3] = {}, small_parts = 0, nfwd = 0, nbwd_q = 0, nbwd_kv = 0, njoin = 0, njoin_q = 0, njoin_kv = 0;
    uint32_t join_rows = 0;  // rows of the fullest joined tile
    int wfwd = 1, wbwd_q = 1, wbwd_kv = 1;  // waves a block
    gatgpu::AttnCap capped;
    bool split = false;  // the forward pass leaves ranges of keys to be joined
    bool cut = false;    // its blocks cut the keys among their waves
    bool spread = false;
};

namespace gatgpu {

DeviceGuard::DeviceGuard(int device) {
    if (hipGetDevice(&before) != hipSuccess) before = -1;
    if (before != device) ok = hipSetDevice(device) == hipSuccess;
    else before = -1;
}
DeviceGuard::~DeviceGuard() {
    if (before >= 0) (void)hipSetDevice(before);
}

// A call must not reach a kernel with an array of the host or of another GPU.
int check_device_array(gatgpu_ctx* c, const void* p, const char* name) {
    hipPointerAttribute_t at{};
    if (hipPointerGetAttributes(&at, p) != hipSuccess || (at.type != hipMemoryTypeDevice && at.type != hipMemoryTypeManaged)) {
        (void)hipGetLastError();
        return fail(c, GATGPU_EINVAL, std::string(name) + " is not device memory");
    }
    if (at.type == hipMemoryTypeDevice && at.device != c->device)
        return fail(c, GATGPU_EINVAL, std::string(name) + " is not on the context's device");
    return GATGPU_OK;
}

}  // namespace gatgpu

namespace {

using namespace gatgpu;

constexpr uint64_t kMaxLen = uint64_t(1) << 30, kMaxRow = uint64_t(1) << 44;
constexpr uint64_t kMaxThreads = (uint64_t(1) << 32) - (1 << 16);  // of a launch

// Keys that query i of a segment sees by position.
uint32_t seen(const gatgpu_attention_shape& sh, const AttnSeg& s, int64_t i) {
    if (sh.mask == GATGPU_MASK_FULL) return s.k_len;
    const int64_t pos = i + int64_t(s.k_len) - int64_t(s.q_len);
    return uint32_t(std::min<int64_t>(s.k_len, std::max<int64_t>(pos + 1, s.prefix)));
}

// True if two of the ranges [begin, begin + len) share a row.
bool overlap(const std::vector<AttnSeg>& segs, bool keys) {
    std::vector<std::pair<uint64_t, uint64_t>> r;
    for (const AttnSeg& s : segs) {
        const uint64_t at = keys ? s.k_begin : s.q_begin, len = keys ? s.k_len : s.q_len;
        if (len) r.emplace_back(at, at + len);
    }
    std::sort(r.begin(), r.end());
    for (size_t i = 1; i < r.size(); ++i)
        if (r[i].first < r[i - 1].second) return true;
    return false;
}

int upload(gatgpu_ctx* c, DevBuf& b, const void* p, size_t bytes) {
    HIPCHECK(c, b.ensure(bytes));
    if (bytes) HIPCHECK(c, hipMemcpyAsync(b.p, p, bytes, hipMemcpyHostToDevice, c->stream));
    return GATGPU_OK;
}

// Long tiles first: the last blocks to start are then short ones.
void longest_first(std::vector<AttnTask>& t) {
    std::stable_sort(t.begin(), t.end(), [](const AttnTask& x, const AttnTask& y) { return x.hi - x.lo > y.hi - y.lo; });
}

// Cuts tasks into equal ranges (multiples of 64) of `chunk` and less, or (whole) of `chunk` and more; tiles: what
// launch_attention_join takes.  False where none was longer.
bool split_tasks(std::vector<AttnTask>& tasks, std::vector<AttnTask>& tiles, uint64_t chunk, bool whole) {
    std::vector<AttnTask> cut;
    for (const AttnTask& t : tasks) {
        const uint32_t first = uint32_t(cut.size());
        const uint64_t len = t.hi - std::min(t.lo, t.hi), n = std::max<uint64_t>(1, whole ? len / chunk : (len + chunk - 1) / chunk), size = ((len + n - 1) / n + 63) / 64 * 64;
        uint64_t lo = t.lo;
        do {
            const uint64_t hi = n == 1 ? t.hi : std::min<uint64_t>(t.hi, lo + size);
            cut.push_back({t.seg, t.at, uint32_t(lo), uint32_t(hi)});
            lo = hi;
        } while (lo < t.hi);
        tiles.push_back({t.seg, t.at, first, uint32_t(cut.size()) - first});
    }
    if (cut.size() == tasks.size()) {
        tiles.clear();
        return false;
    }
    tasks.swap(cut);
    return true;
}

int build(gatgpu_attention* P) {
    gatgpu_ctx* c = P->ctx;
    const gatgpu_attention_shape& sh = P->shape;
    const uint64_t group = uint64_t(sh.heads / sh.kv_heads), kvh = uint64_t(sh.kv_heads), cus = uint64_t(c->cus);
    // Short segments go to the kernels that hold all their keys (their bias gradients are summed
    // by lanes, so the query heads of a key/value head must divide 32).
    const bool bf16 = sh.precision == GATGPU_BF16;
    const int width = attention_width(sh.dim);
    const bool holds = bf16 ? attention_small_width<uint16_t>(width) : attention_small_width<float>(width);
    // Forward, us with and without that kernel, 8 heads, table: 23 / 28 (1500 segments of up to 30 keys, 8 x 32 in
    // bf16), 37 / 46 (in FP32); of 33 to 64 keys 94 / 129 (1500 segments, 8 x 64 in bf16), but 29 / 23 where a
    // head's two tiles in turn leave the chip few waves (300 segments), and 126 / 110 in FP32.
    uint64_t half = 0;  // segments of 33 to 64 keys
    for (const AttnSeg& s : P->segs) half += s.k_len > 32 && s.k_len <= 64;
    const uint32_t held = !holds ? 0 : bf16 && half * kvh >= 12 * cus ? 64 : 32;
    const auto small = [&](const AttnSeg& s) { return s.k_len > 0 && s.k_len <= held; };
    // Backward, the same: 53 / 122 (1500 of up to 30 keys, 8 x 32 in bf16), 167 / 249 (60), 533 / 558 (120); 8 x 64:
    // 113 / 229, 303 / 472, but 1152 / 952 (120): four waves with a table, but one block a CU.
    uint32_t most = 0;  // keys
    for (uint32_t w = 1; w <= 4 && 32 % group == 0; w *= 2)
        if ((bf16 ? attention_small_backward_lds_bf16 : attention_small_backward_lds_fp32)(sh.dim, int(w), sh.bias, int(group), sh.buckets) <=
            (w == 4 && sh.bias == GATGPU_BIAS_TABLE ? kAttnLds / 2 : kAttnLds))
            most = 32 * w;
    P->own_delta = most;
    const auto small_bwd = [&](const AttnSeg& s) { return s.k_len > 0 && s.k_len <= most; };
    std::vector<AttnTask> sf[2], sb[3];
    const auto waves_of = [](const AttnSeg& s) { return s.k_len <= 32 ? 0 : s.k_len <= 64 ? 1 : 2; };  // log2
    uint64_t count_f[2] = {}, count_b[3] = {};
    for (const AttnSeg& s : P->segs) {
        if (small(s)) ++count_f[s.k_len > 32];
        if (small_bwd(s)) ++count_b[waves_of(s)];
    }
    // Heads a block: as many as leave 8 waves a SIMD, since each of them starts with a trip to memory.
    const auto run = [&](uint64_t count, uint64_t waves) {
        return std::max<uint64_t>(1, std::min(kvh, count * waves * kvh / (32 * cus)));
    };
    for (size_t s = 0; s < P->segs.size(); ++s) {
        const AttnSeg& g = P->segs[s];
        const auto add = [&](std::vector<AttnTask>& to, uint64_t heads) {
            for (uint64_t h = 0; h < kvh; h += heads)
                to.push_back({uint32_t(s), uint32_t(P->small_parts), uint32_t(h), uint32_t(std::min(kvh, h + heads))});
        };
        if (small(g) && g.q_len) add(sf[g.k_len > 32], run(count_f[g.k_len > 32], 1));
        if (small_bwd(g)) {
            const int w = waves_of(g);
            add(sb[w], run(count_b[w], uint64_t(1) << w));
            ++P->small_parts;
        }
    }
    // What the general kernels take: blocks of four waves by rows and by keys, rows, keys.
    uint64_t f4 = 0, q4 = 0, k4 = 0, frows = 0, brows = 0, keys = 0, longest = 0;
    for (const AttnSeg& s : P->segs) {
        const uint64_t rows = s.q_len * group;
        if (!small(s)) {
            f4 += (rows + 127) / 128;
            frows += rows;
            if (s.q_len) longest = std::max<uint64_t>(longest, s.k_len);
        }
        if (!small_bwd(s)) {
            q4 += (rows + 127) / 128;
            k4 += (uint64_t(s.k_len) + 63) / 64;
            brows += rows;
            keys += s.k_len;
        }
    }
    // Four waves a block share their tiles' keys (rows) where three of four have rows (keys).  Backward, us by
    // four waves and by one: 35 / 37 (one segment of 600, 8 x 64), 100 / 133 (two of 2000), 22 / 23 (one of 300).
    // Forward only where that leaves no units idle, since single waves can be cut further: 16 / 20 (four of 600,
    // 160 blocks), 39 / 28 (one of 2000, 128 blocks); 32 columns 36 / 30 (256 blocks), 18.7 / 19.6 (320).
    // (A launch must take their threads too: blocks that are not full have more than the single waves have.)
    const auto full = [&](uint64_t total, uint64_t tiles, uint64_t tile) {
        return tiles && total >= tiles * tile * 3 / 4 && tiles * kvh * 256 <= kMaxThreads;
    };
    P->wfwd = full(frows, f4, 128) && f4 * kvh * 2 > (width < 64 ? 2 * cus : cus) ? 4 : 1;
    P->wbwd_q = full(brows, q4, 128) ? 4 : 1;
    P->wbwd_kv = full(keys, k4, 64) ? 4 : 1;  // (two pairs of waves with 32 keys each, or one)
    // Wide tables for many shared heads leave no room for four waves' tiles.
    const auto lds = bf16 ? attention_backward_lds_bf16 : attention_backward_lds_fp32;
    if (lds(kAttnBackwardQ, sh.dim, P->wbwd_q, sh.bias, int(group), sh.buckets) > kAttnLds) P->wbwd_q = 1;
    if (lds(kAttnBackwardKv, sh.dim, P->wbwd_kv, sh.bias, int(group), sh.buckets) > kAttnLds) P->wbwd_kv = 1;

    std::vector<AttnTask> fwd, bq, bk, join;
    const auto q_tiles = [&](std::vector<AttnTask>& out, uint32_t tile, const auto& skip) {
        for (size_t s = 0; s < P->segs.size(); ++s) {
            const AttnSeg& g = P->segs[s];
            if (skip(g)) continue;
            const uint64_t n = g.q_len * group;
            for (uint64_t r = 0; r < n; r += tile) {
                const uint64_t last = std::min<uint64_t>(n, r + tile) - 1;
                out.push_back({uint32_t(s), uint32_t(r), 0, seen(sh, g, int64_t(last / group))});
            }
        }
    };
    q_tiles(fwd, 32u * uint32_t(P->wfwd), small);
    q_tiles(bq, 32u * uint32_t(P->wbwd_q), small_bwd);
    // Few tiles: the keys of each are cut into ranges, so that more waves take part.  Those of at most
    // `chunk` keys are tasks of their own, which another launch joins; 4, 6, 8 and 12 of them a unit and head
    // took 200, 197, 197 and 210 us over 48 sequences of up to 24K keys: more ranges even out the last
    // ones and cost more sums to join.  The waves of one block cut the keys instead (and join them in LDS)
    // where that leaves each of them not much more.  One token over n keys, 8 x 64, bf16, us by
    // blocks and by tasks: 5.5 / 8.1 (n = 400), 7.5 / 8.5 (900), 11.4 / 9.4 (1800); 16 of them: 13.4 / 19.5
    // (1800); FP32 products take 8 times as long: 8.4 / 11.8 (400), 13.5 / 12.0 (900; 8 x 32).  Where blocks of
    // one wave fill the chip, short rows stay with them: 64 tokens over 200 keys 9.2 by blocks, 8.6 so.
    const uint64_t blocks = fwd.size() * kvh;
    if (P->wfwd == 1 && blocks && blocks < 4 * cus && (longest > 256 || blocks <= cus)) {
        uint64_t work = 0;
        for (const AttnTask& t : fwd) work += t.hi;
        const uint64_t want = std::max<uint64_t>(1, 6 * cus / kvh);  // tasks
        const uint64_t chunk = std::max<uint64_t>(128, (work / want + 31) / 32 * 32);
        const uint64_t cuts = uint64_t(bf16 ? attention_cuts<uint16_t>(width) : attention_cuts<float>(width));
        P->cut = longest * 4 <= cuts * chunk * (bf16 ? 6 : 3) &&
                 (bf16 ? attention_forward_cut_lds_bf16 : attention_forward_cut_lds_fp32)(sh.dim, sh.bias, int(group)) <= kAttnLds;
        if (!P->cut) P->split = split_tasks(fwd, join, chunk, false);
        for (const AttnTask& t : join)
            P->join_rows = std::max<uint32_t>(P->join_rows, std::min<uint32_t>(32, uint32_t(P->segs[t.seg].q_len * group) - t.at));
    }
    for (size_t s = 0; s < P->segs.size(); ++s) {
        const AttnSeg& g = P->segs[s];
        if (small_bwd(g)) continue;
        const uint32_t n = uint32_t(g.q_len * group);
        for (uint64_t k = 0; k < g.k_len; k += P->wbwd_kv == 1 ? 32 : 64) {
            uint32_t lo = 0;  // first row that sees key k
            if (sh.mask != GATGPU_MASK_FULL && k >= g.prefix) {
                const int64_t first = int64_t(k) - (int64_t(g.k_len) - int64_t(g.q_len));
                lo = uint32_t(std::min<int64_t>(g.q_len, std::max<int64_t>(0, first)) * int64_t(group)) / 64 * 64;  // (of whole tiles)
            }
            bk.push_back({uint32_t(s), uint32_t(k), lo, n});
        }
    }
    // Backward passes with few blocks: the same, keys of query tiles and rows of key tiles, into about two ranges a
    // unit.  The joined sums are as large as several outputs, so ranges are long, and none are cut from as many
    // blocks as units (two segments of 2000, 8 x 64: 101 us so, 107 cut).  us without and with: one segment of
    // 2000 91 / 85 (8 x 64, bf16), 398 / 297 (FP32), of 1000 108 / 43 (8 heads on 2), of 3000 579 / 109 (8 on 1, causal).
    std::vector<AttnTask> join_q, join_kv;
    const auto spread_out = [&](std::vector<AttnTask>& tasks, std::vector<AttnTask>& tiles) {
        const uint64_t blocks = tasks.size() * kvh, want = std::max<uint64_t>(1, 2 * cus / kvh);
        uint64_t work = 0;
        for (const AttnTask& t : tasks) work += t.hi - std::min(t.lo, t.hi);
        if (blocks == 0 || blocks >= cus) return;
        const uint64_t least = bf16 ? (blocks * 4 <= cus ? 256 : 512) : (blocks * 2 <= cus ? 96 : 512);
        (void)split_tasks(tasks, tiles, std::max(least, work / want), true);
    };
    spread_out(bq, join_q);
    spread_out(bk, join_kv);
    if (!P->split) longest_first(fwd);
    if (join_q.empty()) longest_first(bq);
    if (join_kv.empty()) longest_first(bk);
    // A task's heads go to different XCDs, whose L2s then keep few heads' keys each, or to the same one, which
    // then has whole lines of narrow rows.  Forward and backward in bf16, us: 24 graphs of 650 to 1300 rows, 8 x 64
    // 139 + 413 spread, 164 + 500 not; 500 of 60 to 120 69 + 310, 71 + 314; 8 x 32: 100 of 250 29 + 80, 27 + 65;
    // 24 of 1300 84 + 210, 92 + 218.
    P->spread = longest > 512 || sh.dim * (bf16 ? 2 : 4) >= 128;
    for (int i = 0; i < 2; ++i) {
        P->nsmall[i] = sf[i].size();
        if (int r = upload(c, P->dsmall[i], sf[i].data(), sf[i].size() * sizeof(AttnTask))) return r;
    }
    for (int i = 0; i < 3; ++i) {
        P->nsmall_bwd[i] = sb[i].size();
        if (int r = upload(c, P->dsmall_bwd[i], sb[i].data(), sb[i].size() * sizeof(AttnTask))) return r;
    }
    P->nfwd = fwd.size();
    P->nbwd_q = bq.size();
    P->nbwd_kv = bk.size();
    P->njoin = join.size();
    P->njoin_q = join_q.size();
    P->njoin_kv = join_kv.size();
    if (int r = upload(c, P->dsegs, P->segs.data(), P->segs.size() * sizeof(AttnSeg))) return r;
    if (int r = upload(c, P->dfwd, fwd.data(), fwd.size() * sizeof(AttnTask))) return r;
    if (int r = upload(c, P->dbwd_q, bq.data(), bq.size() * sizeof(AttnTask))) return r;
    if (int r = upload(c, P->dbwd_kv, bk.data(), bk.size() * sizeof(AttnTask))) return r;
    if (int r = upload(c, P->djoin, join.data(), join.size() * sizeof(AttnTask))) return r;
    if (int r = upload(c, P->djoin_q, join_q.data(), join_q.size() * sizeof(AttnTask))) return r;
    if (int r = upload(c, P->djoin_kv, join_kv.data(), join_kv.size() * sizeof(AttnTask))) return r;
    HIPCHECK(c, hipStreamSynchronize(c->stream));
    return GATGPU_OK;
}

uint64_t pad256(uint64_t b) { return (b + 255) / 256 * 256; }
uint64_t part_bytes(const gatgpu_attention* P) {
    return P->split ? pad256(P->nfwd * uint64_t(P->shape.kv_heads) * 32 * uint64_t(attention_width(P->shape.dim)) * 4) : 0;
}
uint64_t forward_bytes(const gatgpu_attention* P) {
    return P->split ? part_bytes(P) + P->nfwd * uint64_t(P->shape.kv_heads) * 32 * 8 : 0;
}
uint64_t delta_bytes(const gatgpu_attention* P) { return pad256(P->rows * uint64_t(P->shape.heads) * 4); }
uint64_t bias_bytes(const gatgpu_attention* P) {
    const gatgpu_attention_shape& sh = P->shape;
    return sh.bias == GATGPU_BIAS_TABLE ? pad256((P->small_parts + P->nbwd_q) * uint64_t(sh.heads) * uint64_t(sh.buckets) * 4) : 0;
}
// Rows of a task's tile in the backward passes.
uint32_t height_q(const gatgpu_attention* P) { return 32 * uint32_t(P->wbwd_q); }
uint32_t height_kv(const gatgpu_attention* P) { return P->wbwd_kv == 1 ? 32 : 64; }
uint64_t backward_bytes(const gatgpu_attention* P) {
    const uint64_t row = uint64_t(P->shape.kv_heads) * uint64_t(attention_width(P->shape.dim)) * 4;
    const uint64_t part = std::max(P->njoin_q ? P->nbwd_q * height_q(P) * row : 0, P->njoin_kv ? P->nbwd_kv * height_kv(P) * 2 * row : 0);
    return delta_bytes(P) + bias_bytes(P) + part;
}

// A matrix of rows: there, aligned, wide enough, on the device.  Of no rows: anything, since nothing reads or writes it
// (and an empty array may have no address).
int check_rows(gatgpu_ctx* c, const char* name, const void* p, uint64_t stride, uint64_t width, int size, uint64_t rows = 1) {
    if (!rows) return GATGPU_OK;
    if (!p) return fail(c, GATGPU_EINVAL, std::string("null ") + name);
    if (reinterpret_cast<uintptr_t>(p) % 16 || stride * uint64_t(size) % 16)
        return fail(c, GATGPU_EINVAL, std::string(name) + " and its stride must be 16-byte aligned");
    if (stride < width || stride > kMaxRow) return fail(c, GATGPU_EINVAL, std::string(name) + " has a bad row stride");
    return check_device_array(c, p, name);
}
int check_floats(gatgpu_ctx* c, const char* name, const void* p) {
    if (!p) return fail(c, GATGPU_EINVAL, std::string("null ") + name);
    if (reinterpret_cast<uintptr_t>(p) % 4) return fail(c, GATGPU_EINVAL, std::string(name) + " must be 4-byte aligned");
    return check_device_array(c, p, name);
}

int check_call(gatgpu_attention* P, const gatgpu_attention_io* io, void* ws, uint64_t bytes, uint64_t need) {
    gatgpu_ctx* c = P->ctx;
    if (!io) return fail(c, GATGPU_EINVAL, "null arrays");
    const gatgpu_attention_shape& sh = P->shape;
    const int size = sh.precision == GATGPU_BF16 ? 2 : 4;
    const uint64_t qw = uint64_t(sh.heads) * uint64_t(sh.dim), kw = uint64_t(sh.kv_heads) * uint64_t(sh.dim);
    if (int r = check_rows(c, "q", io->q, io->q_stride, qw, size, P->rows)) return r;
    if (int r = check_rows(c, "k", io->k, io->k_stride, kw, size, P->keys)) return r;
    if (int r = check_rows(c, "v", io->v, io->v_stride, kw, size, P->keys)) return r;
    if (int r = check_rows(c, "out", io->out, io->out_stride, qw, size, P->rows)) return r;
    if (sh.bias != GATGPU_BIAS_NONE)
        if (int r = check_floats(c, "bias", io->bias)) return r;
    if (sh.bias == GATGPU_BIAS_TABLE && P->dist_bytes)
        if (int r = check_rows(c, "dist", io->dist, 16, 16, 1)) return r;
    if (io->rest) {
        if (sh.precision != GATGPU_BF16) return fail(c, GATGPU_EINVAL, "rest belongs to bf16 outputs");
        if (int r = check_rows(c, "rest", io->rest, io->out_stride, qw, size, P->rows)) return r;
    }
    if (need) {
        if (bytes < need) return fail(c, GATGPU_EINVAL, "workspace of " + std::to_string(bytes) + " bytes, " + std::to_string(need) + " needed");
        if (int r = check_rows(c, "workspace", ws, 16, 16, 1)) return r;
    }
    return GATGPU_OK;
}

AttnArgs make_args(const gatgpu_attention* P, const gatgpu_attention_io* io) {
    const gatgpu_attention_shape& sh = P->shape;
    AttnArgs a;
    a.segs = P->dsegs.as<AttnSeg>();
    a.heads = sh.heads;
    a.kv_heads = sh.kv_heads;
    set_group(a, sh.heads / sh.kv_heads);
    a.dim = sh.dim;
    a.causal = sh.mask == GATGPU_MASK_PREFIX;
    a.bias_kind = sh.bias;
    a.buckets = sh.buckets;
    a.spread = P->spread;
    a.scale = sh.scale;
    a.cap = sh.cap;
    a.capped = P->capped;
    a.q = io->q;
    a.k = io->k;
    a.v = io->v;
    a.qs = io->q_stride;
    a.ks = io->k_stride;
    a.vs = io->v_stride;
    a.bias = sh.bias == GATGPU_BIAS_NONE ? nullptr : io->bias;
    a.dist = sh.bias == GATGPU_BIAS_TABLE ? io->dist : nullptr;
    a.out = io->out;
    a.rest = io->rest;
    a.os = io->out_stride;
    a.lse = io->lse;
    return a;
}

int create(gatgpu_ctx* c, const gatgpu_attention_shape* sh, uint64_t n, const uint64_t* q_begin, const uint32_t* q_len,
           const uint64_t* k_begin, const uint32_t* k_len, const uint32_t* prefix, gatgpu_attention** out) {
    if (!out) return fail(c, GATGPU_EINVAL, "null output pointer");
    *out = nullptr;
    if (!sh) return fail(c, GATGPU_EINVAL, "null shape");
    if (sh->precision != GATGPU_FP32 && sh->precision != GATGPU_BF16) return fail(c, GATGPU_EINVAL, "bad precision");
    if (sh->heads < 1 || sh->heads > 64 || sh->kv_heads < 1 || sh->heads % sh->kv_heads)
        return fail(c, GATGPU_EINVAL, "heads must be 1 to 64 and a multiple of kv_heads");
    if (sh->dim < 8 || sh->dim > kAttnMaxDim || sh->dim % 8) return fail(c, GATGPU_EINVAL, "dim must be a multiple of 8, at most 128");
    if (sh->mask != GATGPU_MASK_FULL && sh->mask != GATGPU_MASK_PREFIX) return fail(c, GATGPU_EINVAL, "bad mask");
    if (sh->bias < GATGPU_BIAS_NONE || sh->bias > GATGPU_BIAS_TABLE) return fail(c, GATGPU_EINVAL, "bad bias");
    if (sh->bias == GATGPU_BIAS_TABLE && (sh->buckets < 1 || sh->buckets > kAttnMaxBuckets))
        return fail(c, GATGPU_EINVAL, "a bias table has 1 to 64 buckets");
    if (!(sh->scale > 0.0f) || !std::isfinite(sh->scale)) return fail(c, GATGPU_EINVAL, "scale must be positive and finite");
    if (!(sh->cap >= 0.0f) || !std::isfinite(sh->cap)) return fail(c, GATGPU_EINVAL, "cap must be 0 or positive and finite");
    if (n && (!q_begin || !q_len || !k_begin || !k_len)) return fail(c, GATGPU_EINVAL, "null segment array");
    if (n > kMaxThreads / 64) return fail(c, GATGPU_EOVERFLOW, "too many segments");
    const uint64_t group = uint64_t(sh->heads / sh->kv_heads);
    std::unique_ptr<gatgpu_attention> P(new gatgpu_attention);
    P->ctx = c;
    P->shape = *sh;
    P->capped = attention_cap(sh->scale, sh->cap);
    if (sh->bias != GATGPU_BIAS_TABLE) P->shape.buckets = 0;
    P->segs.resize(n);
    uint64_t threads = 0;
    for (uint64_t s = 0; s < n; ++s) {
        AttnSeg& g = P->segs[s];
        g.q_begin = q_begin[s];
        g.k_begin = k_begin[s];
        g.q_len = q_len[s];
        g.k_len = k_len[s];
        g.prefix = prefix ? std::min(prefix[s], k_len[s]) : 0;
        g.dist_ld = (g.k_len + 15) / 16 * 16;
        if (g.q_len * group > kMaxLen || g.k_len > kMaxLen)
            return fail(c, GATGPU_EOVERFLOW, "segment " + std::to_string(s) + " is longer than 2^30 rows");
        if (g.q_begin > kMaxRow || g.k_begin > kMaxRow)
            return fail(c, GATGPU_EOVERFLOW, "segment " + std::to_string(s) + " begins beyond 2^44 rows");
        // A wave 32 packed rows, two waves 32 keys, of each key/value head.
        threads += std::max((g.q_len * group + 31) / 32, (uint64_t(g.k_len) + 31) / 32 * 2) * 64 * uint64_t(sh->kv_heads);
        if (threads > kMaxThreads) return fail(c, GATGPU_EOVERFLOW, "more tiles than a launch takes");
        g.base = P->rows;
        g.dist = P->dist_bytes;
        P->rows += g.q_len;
        P->keys += g.k_len;
        if (sh->bias == GATGPU_BIAS_TABLE) P->dist_bytes += uint64_t(g.q_len) * g.dist_ld;
    }
    if (overlap(P->segs, false)) return fail(c, GATGPU_EINVAL, "query rows of two segments overlap");
    P->shared_keys = overlap(P->segs, true);
    if (int r = build(P.get())) return r;
    *out = P.release();
    return GATGPU_OK;
}

}  // namespace

extern "C" {

int gatgpu_attention_create(gatgpu_ctx* c, const gatgpu_attention_shape* shape, uint64_t segments, const uint64_t* q_begin,
                            const uint32_t* q_len, const uint64_t* k_begin, const uint32_t* k_len, const uint32_t* prefix,
                            gatgpu_attention** out) {
    if (!c) return fail(nullptr, GATGPU_EINVAL, "null context");
    DeviceGuard on(c->device);
    if (!on.ok) return fail(c, GATGPU_EDEVICE, "cannot select the context's device");
    try {
        return create(c, shape, segments, q_begin, q_len, k_begin, k_len, prefix, out);
    } catch (const std::exception&) {
        return fail(c, GATGPU_ENOMEM, "host allocation failed");
    }
}

int gatgpu_attention_destroy(gatgpu_attention* P) {
    if (!P) return GATGPU_OK;
    DeviceGuard on(P->ctx->device);
    (void)hipStreamSynchronize(P->ctx->stream);
    delete P;
    return GATGPU_OK;
}

int gatgpu_attention_workspace(const gatgpu_attention* P, uint64_t* forward, uint64_t* backward) {
    if (!P) return fail(nullptr, GATGPU_EINVAL, "null plan");
    if (forward) *forward = forward_bytes(P);
    if (backward) *backward = backward_bytes(P);
    return GATGPU_OK;
}

int gatgpu_attention_distances(const gatgpu_attention* P, uint64_t* bytes, uint64_t* offset, uint32_t* ld) {
    if (!P) return fail(nullptr, GATGPU_EINVAL, "null plan");
    if (P->shape.bias != GATGPU_BIAS_TABLE) return fail(P->ctx, GATGPU_EINVAL, "the plan has no bias table");
    if (bytes) *bytes = P->dist_bytes;
    for (size_t s = 0; s < P->segs.size(); ++s) {
        if (offset) offset[s] = P->segs[s].dist;
        if (ld) ld[s] = P->segs[s].dist_ld;
    }
    return GATGPU_OK;
}

int gatgpu_attention_forward(gatgpu_attention* P, const gatgpu_attention_io* io, void* ws, uint64_t bytes) {
    if (!P) return fail(nullptr, GATGPU_EINVAL, "null plan");
    gatgpu_ctx* c = P->ctx;
    DeviceGuard on(c->device);
    if (!on.ok) return fail(c, GATGPU_EDEVICE, "cannot select the context's device");
    if (int r = check_call(P, io, ws, bytes, forward_bytes(P))) return r;
    if (io->lse && P->rows)
        if (int r = check_floats(c, "lse", io->lse)) return r;
    AttnArgs a = make_args(P, io);
    const bool bf16 = P->shape.precision == GATGPU_BF16;
    for (int i = 1; i >= 0; --i) {
        a.tasks = P->dsmall[i].as<AttnTask>();
        a.ntasks = P->nsmall[i];
        a.rest = P->own_delta >= uint32_t(32 * (i + 1)) ? nullptr : io->rest;
        if (a.ntasks) HIPCHECK(c, (bf16 ? launch_attention_small_forward_bf16 : launch_attention_small_forward_fp32)(a, i + 1, c->stream));
    }
    a.rest = io->rest;
    a.tasks = P->dfwd.as<AttnTask>();
    a.ntasks = P->nfwd;
    if (!a.ntasks) return GATGPU_OK;
    if (P->split) {
        a.part = static_cast<float*>(ws);
        a.stat = reinterpret_cast<float*>(static_cast<char*>(ws) + part_bytes(P));
    }
    if (P->cut) {
        HIPCHECK(c, (bf16 ? launch_attention_forward_cut_bf16 : launch_attention_forward_cut_fp32)(a, c->stream));
        return GATGPU_OK;
    }
    HIPCHECK(c, (bf16 ? launch_attention_forward_bf16 : launch_attention_forward_fp32)(a, P->wfwd, c->stream));
    if (P->split) HIPCHECK(c, launch_attention_join(a, bf16, P->djoin.as<AttnTask>(), P->njoin, P->join_rows, c->stream));
    return GATGPU_OK;
}

int gatgpu_attention_backward(gatgpu_attention* P, const gatgpu_attention_io* io, void* ws, uint64_t bytes) {
    if (!P) return fail(nullptr, GATGPU_EINVAL, "null plan");
    gatgpu_ctx* c = P->ctx;
    DeviceGuard on(c->device);
    if (!on.ok) return fail(c, GATGPU_EDEVICE, "cannot select the context's device");
    if (P->shared_keys) return fail(c, GATGPU_EINVAL, "key rows of two segments overlap: no backward pass");
    if (int r = check_call(P, io, ws, bytes, backward_bytes(P))) return r;
    const gatgpu_attention_shape& sh = P->shape;
    const bool bf16 = sh.precision == GATGPU_BF16;
    const int size = bf16 ? 2 : 4;
    const uint64_t qw = uint64_t(sh.heads) * uint64_t(sh.dim), kw = uint64_t(sh.kv_heads) * uint64_t(sh.dim);
    if (P->rows)
        if (int r = check_floats(c, "lse", io->lse)) return r;
    if (int r = check_rows(c, "dout", io->dout, io->dout_stride, qw, size, P->rows)) return r;
    if (int r = check_rows(c, "dq", io->dq, io->dq_stride, qw, size, P->rows)) return r;
    if (int r = check_rows(c, "dk", io->dk, io->dk_stride, kw, size, P->keys)) return r;
    if (int r = check_rows(c, "dv", io->dv, io->dv_stride, kw, size, P->keys)) return r;
    if (io->dbias) {
        if (sh.bias != GATGPU_BIAS_TABLE) return fail(c, GATGPU_EINVAL, "dbias without a bias table");
        if (bf16 && !io->rest && P->rows) return fail(c, GATGPU_EINVAL, "dbias of bf16 rows needs rest");
        if (int r = check_floats(c, "dbias", io->dbias)) return r;
    }
    AttnArgs a = make_args(P, io);
    a.dout = io->dout;
    a.dos = io->dout_stride;
    a.dq = io->dq;
    a.dk = io->dk;
    a.dv = io->dv;
    a.dqs = io->dq_stride;
    a.dks = io->dk_stride;
    a.dvs = io->dv_stride;
    a.delta = static_cast<float*>(ws);
    a.dbias = io->dbias ? reinterpret_cast<float*>(static_cast<char*>(ws) + delta_bytes(P)) : nullptr;
    for (int i = 2; i >= 0; --i) {
        a.tasks = P->dsmall_bwd[i].as<AttnTask>();
        a.ntasks = P->nsmall_bwd[i];
        if (a.ntasks)
            HIPCHECK(c, (bf16 ? launch_attention_small_backward_bf16 : launch_attention_small_backward_fp32)(a, 1 << i, c->stream));
    }
    a.first_part = P->small_parts;
    a.tasks = P->dbwd_q.as<AttnTask>();
    a.ntasks = P->nbwd_q;
    float* const part = reinterpret_cast<float*>(static_cast<char*>(ws) + delta_bytes(P) + bias_bytes(P));
    a.part = P->njoin_q ? part : nullptr;
    if (a.ntasks) HIPCHECK(c, (bf16 ? launch_attention_backward_q_bf16 : launch_attention_backward_q_fp32)(a, P->wbwd_q, c->stream));
    if (P->njoin_q)
        HIPCHECK(c, launch_attention_grad_join(a, bf16, false, P->djoin_q.as<AttnTask>(), P->njoin_q, height_q(P), c->stream));
    if (io->dbias) HIPCHECK(c, launch_attention_bias_sum(a, P->small_parts + P->nbwd_q, io->dbias, c->stream));
    a.tasks = P->dbwd_kv.as<AttnTask>();
    a.ntasks = P->nbwd_kv;
    a.part = P->njoin_kv ? part : nullptr;
    if (a.ntasks) HIPCHECK(c, (bf16 ? launch_attention_backward_kv_bf16 : launch_attention_backward_kv_fp32)(a, P->wbwd_kv, c->stream));
    if (P->njoin_kv)
        HIPCHECK(c, launch_attention_grad_join(a, bf16, true, P->djoin_kv.as<AttnTask>(), P->njoin_kv, height_kv(P), c->stream));
    return GATGPU_OK;
}

}  // extern "C"
