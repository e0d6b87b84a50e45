// Block tables and slot maps of a paged K/V cache, built on the device from the lengths of a batch
// (diopiBuildBlockTable). With c_i tokens cached, n_i new ones and blocks of bs tokens, request i holds
// have_i = ceil(c_i / bs) blocks and needs need_i = ceil((c_i + n_i) / bs) - have_i more, which are taken from the free
// list in request order: first_i = free_start + sum of need_r over r < i.
//
// Bound by launch latency (a decode step moves a few KB) or, with the table of one slot for each token, by its writes.
// One launch does everything: CTA (i, y) adds up need and n over the requests before i itself (B loads from L2, cheaper
// than a second kernel or a wait between CTAs for any B that a batch has), then works on slice y of request i. Nothing
// it reads is written by another CTA: entries below have_i stay as they were, and the blocks behind them are read from
// the free list, not from the table.
#include "dev_util.cuh"

namespace b200 {
namespace k {
namespace {

constexpr int kTableThreads = 256;
constexpr int kSliceTokens = 2048;   // positions of a request that one CTA of its row covers at least

__device__ __forceinline__ void store_index(const IndexArg& a, int64_t off, int64_t v) {
    if (a.is64)
        static_cast<int64_t*>(const_cast<void*>(a.ptr))[off] = v;
    else
        static_cast<int32_t*>(const_cast<void*>(a.ptr))[off] = static_cast<int32_t>(v);
}

struct RequestSpan {
    int64_t c, n, raw;   // cached tokens, new tokens that fit, new tokens asked for
    bool cut;
};

__device__ __forceinline__ RequestSpan span_of(const BlockTableArgs& a, int i) {
    const int64_t cap = static_cast<int64_t>(a.cols) * a.block_size;
    int64_t c = load_index(a.cached, i), n = load_index(a.fresh, i);
    RequestSpan s;
    s.cut = c < 0 || n < 0 || c > cap || n > cap - c;
    c = imin64(imax64(c, 0), cap);
    n = imin64(imax64(n, 0), 1ll << 31);
    s.raw = n;
    s.c = c;
    s.n = imin64(n, cap - c);
    return s;
}

__global__ void __launch_bounds__(kTableThreads, 6) block_table_kernel(const BlockTableArgs a) {
    __shared__ int64_t part[2][kTableThreads / 32];
    const int i = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int bs = a.block_size;
    auto blocks = [&](int64_t tokens) { return (static_cast<uint32_t>(tokens) + static_cast<uint32_t>(bs) - 1u) / static_cast<uint32_t>(bs); };

    int64_t before = 0, taken = 0;   // new tokens and blocks of the requests before i
    for (int r = tid; r < min(i, a.B); r += kTableThreads) {
        const RequestSpan s = span_of(a, r);
        before += s.raw;
        taken += blocks(s.c + s.n) - blocks(s.c);
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

    const int64_t start = imax64(load_index(a.free_start, 0), 0);
    if (i == a.B) {   // one row of CTAs behind the last request: the totals, and the slots that nobody got
        if (blockIdx.y == 0 && tid == 0) {
            store_index(a.new_start, static_cast<int64_t>(a.B) * a.new_start.s0, before);
            store_index(a.free_next, 0, imin64(start + taken, imax64(a.n_free, start)));
        }
        for (int64_t t = before + static_cast<int64_t>(blockIdx.y) * kTableThreads + tid; t < a.T; t += static_cast<int64_t>(gridDim.y) * kTableThreads)
            store_index(a.slot_map, t * a.slot_map.s0, kNoSlot);
        return;
    }

    const RequestSpan s = span_of(a, i);
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
    // The slots of positions pos .. pos + n - 1 to n elements of `to`, `step` apart from element `off` on.
    auto write_slots = [&](const IndexArg& to, int64_t off, int64_t step, int64_t n, uint32_t pos) {
        if (step == 1 && !to.is64) {
            // four at a time, one division and one block id for them unless a block ends among them
            int32_t* d = static_cast<int32_t*>(const_cast<void*>(to.ptr)) + off;
            const int lead = static_cast<int>(reinterpret_cast<uintptr_t>(d) / 4 % 4);   // elements of the first aligned four that are not ours
            for (int64_t k = 4ll * at - lead; k < n; k += 4ll * stride) {
                const int e0 = k < 0 ? static_cast<int>(-k) : 0, e1 = n - k < 4 ? static_cast<int>(n - k) : 4;
                const uint32_t p = pos + static_cast<uint32_t>(k + e0);
                uint32_t b = p / static_cast<uint32_t>(bs), o = p - b * static_cast<uint32_t>(bs);
                int64_t id = block_id(b);
                int32_t v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    v[e] = 0;
                    if (e < e0 || e >= e1) continue;
                    if (o == static_cast<uint32_t>(bs)) {
                        id = block_id(++b);
                        o = 0;
                    }
                    v[e] = static_cast<int32_t>(slot_in(id, o++, false));
                }
                if (e0 == 0 && e1 == 4) {
                    *reinterpret_cast<int4*>(d + k) = make_int4(v[0], v[1], v[2], v[3]);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (e >= e0 && e < e1) d[k + e] = v[e];
                }
            }
            return;
        }
        for (int64_t k = at; k < n; k += stride) {
            const uint32_t p = pos + static_cast<uint32_t>(k), b = p / static_cast<uint32_t>(bs);
            store_index(to, off + k * step, slot_in(block_id(b), p - b * static_cast<uint32_t>(bs), to.is64));
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

void launch_block_table(const BlockTableArgs& a, int sm_count, cudaStream_t st) {
    // Slices of a row: enough CTAs for the SMs when the batch is small and its rows are long.
    const int64_t longest = std::max<int64_t>(a.wide.ptr ? a.wide_cols : 0, std::min<int64_t>(a.T, static_cast<int64_t>(a.cols) * a.block_size));
    int64_t y = (longest + kSliceTokens - 1) / kSliceTokens;
    y = std::min<int64_t>(y, std::max<int64_t>(1, static_cast<int64_t>(sm_count) * 8 / (a.B + 1)));
    dim3 grid(a.B + 1, static_cast<unsigned>(std::max<int64_t>(1, y)));
    block_table_kernel<<<grid, kTableThreads, 0, st>>>(a);
}

}  // namespace k
}  // namespace b200
