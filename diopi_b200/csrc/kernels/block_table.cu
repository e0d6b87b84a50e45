// Block tables and slot maps of a paged K/V cache, built on the device from the lengths of a batch
// (diopiBuildBlockTable). With c_i tokens cached, n_i new ones and blocks of bs tokens, request i holds
// have_i = ceil(c_i / bs) blocks and needs need_i = ceil((c_i + n_i) / bs) - have_i more, which are taken from the free
// list in request order: first_i = free_start + sum of need_r over r < i.
//
// Bound by latency: launch, lengths, block ids, stores. A decode step of 64 requests takes 3.0 us, 64 prompts of up to 8192 tokens
// 4.2, 1024 requests with the table of one slot for each token (16.8 MB) 14.5 (64-bit indexes: 2.9, 4.2, 16.9).
// One launch does everything: CTA (i, y) adds up need and n over the requests before i itself (B loads from L2, cheaper
// than a second kernel or a wait between CTAs for a thousand requests; the sums grow with B^2: a decode step of 2048
// requests takes 10 us, of 8192 61, and 13 and 120 with 64-bit lengths), then works on slice y of request i. Nothing
// it reads is written by another CTA: entries below have_i stay as they were, and the blocks behind them are read from
// the free list, not from the table.
#include "dev_util.cuh"

namespace b200 {
namespace k {
namespace {

constexpr int kTableThreads = 192;   // with 40 registers eight CTAs to an SM: 1024 requests are one wave
constexpr uint32_t kIds = 512;       // block ids held in shared memory
constexpr int kSliceTokens = 2048;   // positions of a request that one CTA of its row covers at least

__device__ __forceinline__ void store_index(const IndexArg& a, int64_t off, int64_t v) {
    if (a.is64)
        static_cast<int64_t*>(const_cast<void*>(a.ptr))[off] = v;
    else
        static_cast<int32_t*>(const_cast<void*>(a.ptr))[off] = static_cast<int32_t>(v);
}

// x / block_size for x < 2^31: a product and a shift. With l = ceil(log2 d) and m = ceil(2^(31 + l) / d), m * d exceeds
// 2^(31 + l) by less than d <= 2^l, so x * m / 2^(31 + l) exceeds x / d by less than 1 / d. (Every CTA divides for every
// request before its own.)
__device__ __forceinline__ uint32_t by_block(const BlockTableArgs& a, uint32_t x) {
    return static_cast<uint32_t>((static_cast<uint64_t>(x) * a.div_mul) >> a.div_shift);
}

struct RequestSpan {
    int64_t c, n, raw;   // cached tokens, new tokens that fit, new tokens asked for
    bool cut;
};

__device__ __forceinline__ RequestSpan span_of(const BlockTableArgs& a, int64_t c, int64_t n) {
    const int64_t cap = static_cast<int64_t>(a.cols) * a.block_size;
    RequestSpan s;
    s.cut = c < 0 || n < 0 || c > cap || n > cap - c;
    c = imin64(imax64(c, 0), cap);
    n = imin64(imax64(n, 0), 1ll << 31);
    s.raw = n;
    s.c = c;
    s.n = imin64(n, cap - c);
    return s;
}

__global__ void __launch_bounds__(kTableThreads, 8) block_table_kernel(const BlockTableArgs a) {
    __shared__ int64_t part[2][kTableThreads / 32];
    __shared__ int64_t ids[kIds];
    const int i = a.B - static_cast<int>(blockIdx.x), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;   // those with most to add up first
    const int bs = a.block_size;
    auto blocks = [&](int64_t tokens) -> uint32_t { return tokens == 0 ? 0u : by_block(a, static_cast<uint32_t>(tokens) - 1u) + 1u; };   // that hold them

    // What this CTA needs of its own request, asked for before the others' lengths are added up.
    const int own = min(i, a.B - 1);
    const int64_t own_c = own >= 0 ? load_index(a.cached, own) : 0, own_n = own >= 0 ? load_index(a.fresh, own) : 0;
    const int64_t start = imax64(load_index(a.free_start, 0), 0);
    int64_t before = 0, taken = 0;   // new tokens and blocks of the requests before i
    if (!a.cached.is64 && !a.fresh.is64 && a.cached.s0 == 1 && a.fresh.s0 == 1) {
        // The usual case in 32 bits: with 1024 requests half a million lengths are added up over all CTAs (18.5 us in 64 bits, 16.4).
        const int32_t *cp = static_cast<const int32_t*>(a.cached.ptr), *np = static_cast<const int32_t*>(a.fresh.ptr);
        const int32_t cap = static_cast<int32_t>(static_cast<int64_t>(a.cols) * bs);
        for (int r0 = tid; r0 < i; r0 += 4 * kTableThreads) {
            int32_t c[4], n[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int r = r0 + u * kTableThreads;
                c[u] = r < i ? cp[r] : 0;
                n[u] = r < i ? np[r] : 0;
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int32_t cc = min(max(c[u], 0), cap), raw = max(n[u], 0), nn = min(raw, cap - cc);
                before += raw;
                taken += blocks(cc + nn) - blocks(cc);
            }
        }
    } else {
        for (int r = tid; r < i; r += kTableThreads) {
            const RequestSpan s = span_of(a, load_index(a.cached, r), load_index(a.fresh, r));
            before += s.raw;
            taken += blocks(s.c + s.n) - blocks(s.c);
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        before += __shfl_xor_sync(0xffffffffu, before, o);
        taken += __shfl_xor_sync(0xffffffffu, taken, o);
    }
    if (lane == 0) {
        part[0][warp] = before;
        part[1][warp] = taken;
    }
    __syncthreads();
    before = taken = 0;
#pragma unroll
    for (int w = 0; w < kTableThreads / 32; ++w) {
        before += part[0][w];
        taken += part[1][w];
    }

    if (i == a.B) {   // one row of CTAs more than requests: the totals, and the slots that nobody got
        if (blockIdx.y == 0 && tid == 0) {
            store_index(a.new_start, static_cast<int64_t>(a.B) * a.new_start.s0, before);
            store_index(a.free_next, 0, imin64(start + taken, imax64(a.n_free, start)));
        }
        for (int64_t t = before + static_cast<int64_t>(blockIdx.y) * kTableThreads + tid; t < a.T; t += static_cast<int64_t>(gridDim.y) * kTableThreads)
            store_index(a.slot_map, t * a.slot_map.s0, kNoSlot);
        return;
    }

    const RequestSpan s = span_of(a, own_c, own_n);
    const uint32_t have = blocks(s.c);
    const uint32_t need = blocks(s.c + s.n) - have;
    const int64_t first = start + taken;
    bool bad = s.cut;
    bool ran_out = need > 0 && first + need > a.n_free;

    if (blockIdx.y == 0) {
        for (uint32_t j = tid; j < need; j += kTableThreads) {
            const int64_t f = first + j;
            const int64_t id = f < a.n_free ? load_index(a.free_blocks, f) : -1;
            store_index(a.table, static_cast<int64_t>(i) * a.table.s0 + static_cast<int64_t>(have + j) * a.table.s1, id);
        }
        if (tid == 0) {
            store_index(a.new_start, static_cast<int64_t>(i) * a.new_start.s0, before);
            store_index(a.seq_lens, static_cast<int64_t>(i) * a.seq_lens.s0, s.c + s.n);
        }
    }

    auto block_id = [&](uint32_t b) -> int64_t {
        if (b < have) return load_index(a.table, i, b);
        const int64_t f = first + (b - have);
        return f < a.n_free ? load_index(a.free_blocks, f) : -1;
    };
    // The slot at offset o of a block: kNoSlot where there is no block, or where the slot does not fit the tensor's type.
    auto slot_in = [&](int64_t id, uint32_t o, bool is64) -> int64_t {
        const int64_t slot = id * bs + o;
        if (id < 0 || (!is64 && slot > 0x7fffffffll)) {
            bad = true;
            return kNoSlot;
        }
        return slot;
    };
    const uint32_t stride = gridDim.y * kTableThreads, at = blockIdx.y * kTableThreads + tid;
    // The slots of positions pos .. pos + n - 1 to n elements of `to`, `step` apart from element `off` on. All threads of the
    // CTA call it with the same arguments: the ids of kIds blocks at a time are brought to shared memory first (asked for
    // one by one they cost a row of 8192 slots eleven memory latencies one after the other: 22 us instead of 18.6).
    auto write_slots = [&](const IndexArg& to, int64_t off, int64_t step, int64_t n, uint32_t pos) {
        if (n <= 0) return;
        if (n <= 2 * kTableThreads) {   // few enough for an id each
            for (int64_t k = at; k < n; k += stride) {
                const uint32_t p = pos + static_cast<uint32_t>(k), b = by_block(a, p);
                store_index(to, off + k * step, slot_in(block_id(b), p - b * static_cast<uint32_t>(bs), to.is64));
            }
            return;
        }
        const uint32_t last = by_block(a, pos + static_cast<uint32_t>(n) - 1);
        for (uint32_t b0 = by_block(a, pos); b0 <= last; b0 += kIds) {
            __syncthreads();
            for (uint32_t x = tid; x < kIds && b0 + x <= last; x += kTableThreads) ids[x] = block_id(b0 + x);
            __syncthreads();
            // elements [lo, hi) lie in these blocks
            const int64_t first_pos = static_cast<int64_t>(b0) * bs;
            const int64_t lo = imax64(first_pos - pos, 0), hi = imin64(first_pos + static_cast<int64_t>(kIds) * bs - pos, n);
            auto slot_at = [&](int64_t k, bool is64) {
                const uint32_t p = static_cast<uint32_t>(pos + k - first_pos), b = by_block(a, p);
                return slot_in(ids[b], p - b * static_cast<uint32_t>(bs), is64);
            };
            if (step == 1 && !to.is64) {   // four at a time
                int32_t* d = static_cast<int32_t*>(const_cast<void*>(to.ptr)) + off;
                const int64_t lead = static_cast<int64_t>(reinterpret_cast<uintptr_t>(d + lo) / 4 % 4);
                for (int64_t k = lo - lead + 4ll * at; k < hi; k += 4ll * stride) {
                    if (k >= lo && k + 4 <= hi) {
                        const uint32_t p = static_cast<uint32_t>(pos + k - first_pos);
                        uint32_t b = by_block(a, p), o = p - b * static_cast<uint32_t>(bs);
                        int32_t v[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            if (o == static_cast<uint32_t>(bs)) {
                                ++b;
                                o = 0;
                            }
                            v[e] = static_cast<int32_t>(slot_in(ids[b], o++, false));
                        }
                        *reinterpret_cast<int4*>(d + k) = make_int4(v[0], v[1], v[2], v[3]);
                    } else {
                        for (int64_t e = imax64(k, lo); e < imin64(k + 4, hi); ++e) d[e] = static_cast<int32_t>(slot_at(e, false));
                    }
                }
            } else {
                for (int64_t k = lo + at; k < hi; k += stride) store_index(to, off + k * step, slot_at(k, to.is64));
            }
        }
    };
    const int64_t room = imax64(imin64(s.raw, a.T - before), 0);   // new tokens that slot_map has entries for
    if (room < s.raw) bad = true;
    write_slots(a.slot_map, before * a.slot_map.s0, a.slot_map.s0, imin64(room, s.n), static_cast<uint32_t>(s.c));
    for (int64_t t = s.n + at; t < room; t += stride) store_index(a.slot_map, (before + t) * a.slot_map.s0, kNoSlot);
    if (a.wide.ptr != nullptr) {
        const int64_t L = s.c + s.n, skip = imax64(L - a.wide_cols, 0);   // only the last tokens of a request longer than the row
        if (skip > 0) bad = true;
        write_slots(a.wide, static_cast<int64_t>(i) * a.wide.s0 + (a.wide_cols - L + skip) * a.wide.s1, a.wide.s1, L - skip, static_cast<uint32_t>(skip));
    }
    if (bad || ran_out) report_status(a.status, 4);
}

}  // namespace

void launch_block_table(const BlockTableArgs& args, int sm_count, cudaStream_t st) {
    BlockTableArgs a = args;
    int l = 0;
    while ((1ll << l) < a.block_size) ++l;
    a.div_shift = 31 + l;
    a.div_mul = static_cast<uint32_t>(((1ull << (31 + l)) + a.block_size - 1) / a.block_size);
    // Slices of a row: enough CTAs for the SMs when the batch is small and its rows are long.
    const int64_t longest = std::max<int64_t>(a.wide.ptr ? a.wide_cols : 0, std::min<int64_t>(a.T, static_cast<int64_t>(a.cols) * a.block_size));
    int64_t y = (longest + kSliceTokens - 1) / kSliceTokens;
    y = std::min<int64_t>(y, std::max<int64_t>(1, static_cast<int64_t>(sm_count) * 8 / (a.B + 1)));
    dim3 grid(a.B + 1, static_cast<unsigned>(std::max<int64_t>(1, y)));
    block_table_kernel<<<grid, kTableThreads, 0, st>>>(a);
}

}  // namespace k
}  // namespace b200
