// Attention of the newest tokens over a paged cache of 8-bit codes with one scale for each (block, K/V head)
// (diopiQuantizedPagedAttention). With K/V rows j of request i in block b_j, codes kc, vc and scales ks, vs:
//     x_j = softmax_scale * ks[b_j] * (q . kc_j),   out = sum_j softmax(x)_j * vs[b_j] * vc_j
// New token t of n sees the first L - (n - 1 - t) tokens; a row that sees none gives zeros.
//
// quant_split_kernel (head_dim a multiple of 16 up to 256, any block_size) is bound by the bytes of the codes. The
// query rows that share a K/V head (n * group of them) are the N extent of mma.sync m16n8k16 in fp16 with fp32
// accumulators: every code of either kind is an fp16 number, so nothing is lost by the conversion in registers, and the
// scales stay outside the products. A tile is up to 16 tokens of one K/V head, always inside one block, hence one ks and one vs:
//     S^T = Kc Q^T;  m = f max(S), f = ks * softmax_scale * log2 e;  P = 2^((S - max S) f + 15);  O^T += (2^(m - ref) vs) (Vc^T P^T)
// The weights are taken against the tile's own maximum, so that they fill fp16's range (2^15 down to 2^-24: what is lost is
// below 2^-40 of the tile's largest weight) whatever the other tiles hold, and the product of a tile is added in fp32 with
// its factor; ref is only raised when a tile exceeds it by 2^16, or by less where values are above 2^41 (value_lift).
// Queries are scaled by the power of two that brings their row's maximum to [1, 2) before they become fp16 (bf16 and fp32
// reach further than fp16 does); fp32 queries and their weights are split into two fp16 numbers each, with two products.
// What is rounded to fewer than 24 bits: a query element of bf16 or fp32 to 2^-25 of its row's largest where that is more than its
// own last bits; a weight of fp16 or bf16 queries to one fp16 number (2^-11 of it). Against 64 bits the fp16 results of the third case
// below are off by 2.7e-4 of their size on average, 2.1e-4 with weights in two parts, which is the rounding of the results
// themselves (bf16: 1.7e-3 either way); two parts cost 19 % (70 to 83 us on the first case: spills at 128 registers).
//
// Work split: the tiles of the batch are cut into equal ranges, one per team, a team being the warps of one K/V head (one warp for up
// to 8 * NT query rows, mt of them beyond). The teams of a CTA are hw neighbouring heads of the same range, which keeps their reads
// next to each other in memory, times tw ranges. A team has a ring of tiles of its own, filled by TMA (two loads, K and V, of 16 rows,
// swizzled: the reads below are free of bank conflicts), and its leader refills a slot as soon as it is read: no producer warp, and no
// barrier between teams. Block ids and scales of the next 32 tiles are held by the 32 lanes. Where a request falls into several
// ranges its parts are merged by quant_combine_kernel (a programmatic dependent launch); else it is written directly.
//
// Measured (calls one after the other in a graph, merge included): 64 query heads over 8 K/V heads, 64 requests of 512 to 4096
// tokens, bf16, e4m3: 70 us = 4350 GB/s; four requests of 30011 to 131072 tokens, fp16: 72 us; a K/V head for each of 32 query
// heads, fp16, int8: 209 to 233 us on different GPUs = 0.79 to 0.88 of the copy rate. While it streams the loop runs at the copy
// rate (the loads alone take as long); what is left is 5 us of start (lengths, block ids, first tiles), up to 9 us between the first SM's end and the last one's
// (some groups of SMs get a tenth less bandwidth), 5 us of merge. Tried and dropped: query rows as the M extent (half of
// the products on padding; 98 us); a producer warp beside 16 others (96 registers, spills: 124 us); the last eighth of each
// range given away through clusterlaunchcontrol (79 us; 82 with the next piece's tiles fetched ahead); two CTAs of
// eight warps an SM (the same time).
//
// The new-token form for e4m3 at head_dim 128 spills 4 to 12 bytes a thread, fp32 queries 24 to 88 at head_dim 128 and 256, the
// merge at 64 registers 68 to 72 (it asks for four parts at once; 32 warps an SM hide the rest).
//
// quant_plain_kernel: any width, strides and block size, and batches whose lengths the split kernel cannot hold (more than 4096);
// one CTA to a query row, a warp to every fourth token (the first case above: 9854 us; 4097 requests of up to 60 tokens, 32
// heads over 8: 4100 us, 4096 of them 170 on the split kernel).
#include <cuda.h>

#include <atomic>
#include <mutex>
#include <type_traits>

#include "decode_common.cuh"

namespace b200 {
namespace k {

namespace {

__device__ __forceinline__ float code_value(uint8_t c, bool e4m3) {
    if (!e4m3) return static_cast<float>(static_cast<int8_t>(c));
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(c)));
    return __half2float(__ushort_as_half(static_cast<uint16_t>(h & 0xffffu)));
}

// Tokens of request i, never negative and never more than its row of the table names.
__device__ __forceinline__ int quant_len(const QuantAttnArgs& a, int i) {
    const int64_t cap = static_cast<int64_t>(a.cols) * a.block_size;
    const int64_t L = load_index(a.lens, i);
    return static_cast<int>(imin64(imax64(L, 0), cap));
}

constexpr int kTile = 16;   // tokens of a tile
constexpr float kLowest = -3e38f;   // below every logit, and finite

// How far the reference of the weights has to be above a logit in a block of value scale s, so that a sum of weights times values
// stays finite wherever their mean is: s * 2^-lift < 2^(from + 1). 0 for the values that a model has; else differences of logits are
// taken at a distance of up to 86 from the reference, which rounds them to 2^-18.
__device__ __forceinline__ float value_lift(float s, int from) { return static_cast<float>(max(static_cast<int>(__float_as_uint(s) << 1 >> 24) - 127 - from, 0)); }
// What the reference of the split kernel may lag behind a tile's maximum. With a weight of 2^(15 + kLag - lift) at most the sum over
// 2^31 tokens of code * s stays below 2^(31 + 9 + 42 + 31) = 2^113, and l above 2^(15 - 86).
constexpr float kLag = 16.f;

// Tiles of L tokens: none reaches over the end of a block.
__device__ __forceinline__ int tiles_of(const QuantAttnArgs& a, int L) {
    if (a.block_size % kTile == 0) return (L + kTile - 1) / kTile;
    const int full = L / a.block_size, rest = L - full * a.block_size;
    return full * ((a.block_size + kTile - 1) / kTile) + (rest + kTile - 1) / kTile;
}

constexpr int kPlainWarps = 4;
constexpr int kPlainRegs = 16;   // head_dim <= 512

template <typename T>
__global__ void __launch_bounds__(32 * kPlainWarps) quant_plain_kernel(const QuantAttnArgs a) {
    __shared__ float s_ml[kPlainWarps][2];
    __shared__ float s_o[kPlainWarps][32 * kPlainRegs];
    const int i = blockIdx.x, hq = blockIdx.y % a.Hq, t = blockIdx.y / a.Hq;
    const int h = hq / (a.Hq / a.Hkv);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int L = quant_len(a, i) - (a.n - 1 - t);
    const T* q = static_cast<const T*>(a.q) + static_cast<int64_t>(i) * a.q_s0 + static_cast<int64_t>(t) * a.q_s1 + static_cast<int64_t>(hq) * a.q_s2;
    const uint8_t* kb = static_cast<const uint8_t*>(a.cache[0]) + static_cast<int64_t>(h) * a.c_s2[0];
    const uint8_t* vb = static_cast<const uint8_t*>(a.cache[1]) + static_cast<int64_t>(h) * a.c_s2[1];
    float qr[kPlainRegs], o[kPlainRegs];
#pragma unroll
    for (int r = 0; r < kPlainRegs; ++r) {
        const int d = lane + 32 * r;
        qr[r] = d < a.D ? Cvt<T>::to_f(q[d]) * a.softmax_scale * kLog2e : 0.f;
        o[r] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    for (int j = warp; j < L; j += kPlainWarps) {
        const int64_t b = load_index(a.table, i, j / a.block_size);
        if (b < 0 || b >= a.blocks) {
            if (lane == 0) report_status(a.status, 1);
            continue;
        }
        const int p = j % a.block_size;
        const float ks = a.scale[0][b * a.s_s0[0] + static_cast<int64_t>(h) * a.s_s1[0]], vs = a.scale[1][b * a.s_s0[1] + static_cast<int64_t>(h) * a.s_s1[1]];
        const uint8_t* kr = kb + b * a.c_s0[0] + static_cast<int64_t>(p) * a.c_s1[0];
        const uint8_t* vr = vb + b * a.c_s0[1] + static_cast<int64_t>(p) * a.c_s1[1];
        float x = 0.f;
#pragma unroll
        for (int r = 0; r < kPlainRegs; ++r) {
            const int d = lane + 32 * r;
            if (d < a.D) x = fmaf(qr[r], code_value(kr[d * a.c_s3[0]], a.e4m3), x);
        }
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) x += __shfl_xor_sync(0xffffffffu, x, s);
        x *= ks;
        const float mn = fmaxf(m, x + value_lift(vs, 64));   // a sum of 2^31 tokens ends below 2^(31 + 9 + 65)
        const float al = exp2f(m - mn), w = exp2f(x - mn);
        m = mn;
        l = fmaf(l, al, w);
#pragma unroll
        for (int r = 0; r < kPlainRegs; ++r) {
            const int d = lane + 32 * r;
            if (d < a.D) o[r] = fmaf(o[r], al, w * vs * code_value(vr[d * a.c_s3[1]], a.e4m3));
        }
    }
    if (lane == 0) {
        s_ml[warp][0] = m;
        s_ml[warp][1] = l;
    }
#pragma unroll
    for (int r = 0; r < kPlainRegs; ++r) s_o[warp][lane + 32 * r] = o[r];
    __syncthreads();
    float M = -INFINITY, Ls = 0.f, w[kPlainWarps];
#pragma unroll
    for (int k = 0; k < kPlainWarps; ++k) M = fmaxf(M, s_ml[k][0]);
#pragma unroll
    for (int k = 0; k < kPlainWarps; ++k) {
        w[k] = s_ml[k][0] == -INFINITY ? 0.f : exp2f(s_ml[k][0] - M);   // a warp that saw no token
        Ls = fmaf(s_ml[k][1], w[k], Ls);
    }
    const float inv = Ls == 0.f ? 0.f : 1.f / Ls;
    T* out = static_cast<T*>(a.out) + static_cast<int64_t>(i) * a.o_s0 + static_cast<int64_t>(t) * a.o_s1 + static_cast<int64_t>(hq) * a.o_s2;
    for (int d = threadIdx.x; d < a.D; d += 32 * kPlainWarps) {
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < kPlainWarps; ++k) v = fmaf(s_o[k][d], w[k], v);
        out[d] = Cvt<T>::from_f(v * inv);
    }
}

// ---------------------------------------------------------------------------------------------------
// The split kernel.
// ---------------------------------------------------------------------------------------------------
constexpr int kQMaxStages = 8;
constexpr int kQMaxB = 4096;
constexpr int kTilesPerRange = 4;               // at least, so that short batches are not cut into crumbs (2: the same times, twice the parts)

// Warps of a CTA: as many as the registers of a thread's queries and accumulators leave room for (a spilled register costs
// an L2 access here, as shared memory leaves no L1).
constexpr int split_warps(bool f32, int hd, int nt) { return hd * nt * (f32 ? 2 : 1) <= 128 ? 16 : hd == 128 && f32 ? 12 : 8; }

struct QuantPlan {
    int hd;           // 64, 128 or 256: head_dim rounded up
    int nt;           // N tiles of 8 query rows of a warp
    int mt;           // warps of a team
    int n_z;          // CTAs along the query rows of a K/V head
    int hw;           // K/V heads of a CTA: a divisor of Hkv
    int n_hg;         // CTAs along the K/V heads
    int tw;           // ranges of a CTA
    int block_tiles;  // tiles of a block
    bool ragged;      // the last of them is not full
    int stages;       // tiles of a team's ring
    int n_cta, n_range;
    int off_bars, off_pre, off_len, off_flag, smem_bytes;
    bool qvec;        // four elements of q can be loaded at once
};

__device__ __forceinline__ void tma_4d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// 8 x 8 transpose of 16-bit elements: lane 4 r + c holds columns 2c, 2c + 1 of row r, before and after.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// What two fp32 values lose as fp16, as fp16.
__device__ __forceinline__ uint32_t pack_rest(float lo, float hi, uint32_t packed) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&packed));
    return pack_f16(lo - f.x, hi - f.y);
}
// Four codes in one register -> two registers of two fp16 numbers, exactly. int8: the byte with its sign bit flipped is the
// low byte of the fp16 number 1024 + 128 + code.
template <bool E4M3>
__device__ __forceinline__ void codes_to_f16(uint32_t c, uint32_t& lo, uint32_t& hi) {
    if constexpr (E4M3) {
        asm("{\n.reg .b16 l, h;\nmov.b32 {l, h}, %2;\ncvt.rn.f16x2.e4m3x2 %0, l;\ncvt.rn.f16x2.e4m3x2 %1, h;\n}\n" : "=r"(lo), "=r"(hi) : "r"(c));
    } else {
        const uint32_t x = c ^ 0x80808080u;
        const uint32_t l = __byte_perm(x, 0x64646464u, 0x4140), h = __byte_perm(x, 0x64646464u, 0x4342);
        const __half2 bias = __half2half2(__ushort_as_half(0x6480));   // 1152
        const __half2 a = __hsub2(*reinterpret_cast<const __half2*>(&l), bias), b = __hsub2(*reinterpret_cast<const __half2*>(&h), bias);
        lo = *reinterpret_cast<const uint32_t*>(&a);
        hi = *reinterpret_cast<const uint32_t*>(&b);
    }
}

__device__ __forceinline__ int used_ranges(int total, int n_range) { return max(1, min(n_range, (total + kTilesPerRange - 1) / kTilesPerRange)); }

// MANY: more than one new token to a request, so that the rows of a tile may see different tokens. (Only the care for NaN
// goes by it: the masks written out for one token alone, the kernel for e4m3 at head_dim 128 spills and is 4 % slower.)
template <typename T, bool E4M3, int HD, int NT, bool MANY>
__global__ void __launch_bounds__(32 * split_warps(std::is_same<T, float>::value, HD, NT), 1)
    quant_split_kernel(const QuantAttnArgs a, const QuantPlan p, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                       float* __restrict__ ws_acc, float* __restrict__ ws_ml) {
    constexpr bool SPLIT = std::is_same<T, float>::value;   // two fp16 numbers for each fp32 one
    constexpr int RB = HD < 128 ? HD : 128;                 // bytes of a row of one TMA box
    constexpr int NH = HD / RB;                             // boxes side by side (head_dim 256: 2)
    constexpr int CH = HD / 16;                             // k steps of Kc Q^T: 16 bytes of codes each
    constexpr int VB = RB / 8;                              // bytes of a V row that a lane takes from each box
    constexpr int DM = HD / 16;                             // M tiles of Vc^T P^T
    constexpr int BOX = kTile * RB;                         // bytes of a box
    constexpr uint32_t STAGE = 2 * NH * BOX;                // K, then V
    constexpr int kThreads = 32 * split_warps(SPLIT, HD, NT);
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);   // the swizzle goes by address bits
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + p.off_bars);                      // [team][full, empty][stage]
    int* pre = reinterpret_cast<int*>(smem + p.off_pre);                                  // pre[i] = first tile of request i
    int* lens = reinterpret_cast<int*>(smem + p.off_len);
    volatile int* give_up = reinterpret_cast<volatile int*>(smem + p.off_flag);

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (threadIdx.x < 2)
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(threadIdx.x == 0 ? &map_k : &map_v)) : "memory");

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int group = a.Hq / a.Hkv;
    const int R = a.n * group;                 // query rows of a K/V head
    const int teams = p.hw * p.tw;

    if (tid < teams * p.stages) {
        uint64_t* b = bars + tid / p.stages * (2 * p.stages) + tid % p.stages;
        mbar_init(smem_u32(b), 1);
        mbar_init(smem_u32(b + p.stages), p.mt);
    }
    if (tid == 0) {
        *give_up = 0;
        pre[0] = 0;
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    for (int i = tid; i < a.B; i += kThreads) {
        const int L = quant_len(a, i);
        lens[i] = L;
        pre[i + 1] = tiles_of(a, L);
    }
    __syncthreads();
    if (warp == 0) {
        int carry = 0;
        for (int base = 0; base < a.B; base += 32) {
            const int idx = base + lane;
            int v = idx < a.B ? pre[idx + 1] : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, v, o);
                if (lane >= o) v += u;
            }
            if (idx < a.B) pre[idx + 1] = v + carry;
            carry += __shfl_sync(0xffffffffu, v, 31);
        }
    }
    __syncthreads();

    const int team = warp / p.mt, mtile = warp - team * p.mt;
    const int hl = team % p.hw, range = team / p.hw * p.n_cta + blockIdx.x;   // few ranges: spread over the SMs
    const int total = pre[a.B];
    const int used = used_ranges(total, p.n_range);
    if (team < teams && range < used && total > 0) {
        const int t0 = static_cast<int>(static_cast<int64_t>(total) * range / used);
        const int t1 = static_cast<int>(static_cast<int64_t>(total) * (range + 1) / used);
        const int hkv = blockIdx.y * p.hw + hl;
        const uint32_t ring0 = smem_u32(smem) + static_cast<uint32_t>(team * p.stages) * STAGE;
        const uint32_t full0 = smem_u32(bars + team * 2 * p.stages), empty0 = full0 + 8u * p.stages;

        // ---- what the lanes know of 32 tiles: lane k of tile base + k ----
        struct Ahead {
            int block, at;   // at = 32 * position in the block + tokens (0: leave the tile out)
            float ks, vs;
        } cur, nxt;
        auto request_of = [&](int t) {
            int lo = 0, hi = a.B;   // smallest i with pre[i + 1] > t
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (pre[mid + 1] > t)
                    hi = mid;
                else
                    lo = mid + 1;
            }
            return lo;
        };
        // First position of a request's tile, its block's column and its place in the block.
        auto place_of = [&](int tile, int& col, int& at) {
            col = tile / p.block_tiles;
            at = (tile - col * p.block_tiles) * kTile;
            return col * a.block_size + at;
        };
        // In two halves, so that what comes between them hides the load of the block ids.
        auto ask_ids = [&](Ahead& x, int from) -> int64_t {
            x.at = 0;
            const int t = from + lane;
            if (t >= t1) return 0;
            const int i = request_of(t);
            int col, at;
            const int pos = place_of(t - pre[i], col, at);
            x.at = at * 32 + min(min(kTile, a.block_size - at), lens[i] - pos);
            return load_index(a.table, i, col);
        };
        auto take_ids = [&](Ahead& x, int64_t id) {
            const bool ok = id >= 0 && id < a.blocks;
            if (!ok) report_status(a.status, 1);
            x.block = ok ? static_cast<int>(id) : 0;
            if (!ok) x.at = 0;
            x.ks = x.vs = 0.f;
        };
        auto load_scales = [&](Ahead& x) {
            if (x.at != 0) {
                x.ks = a.scale[0][x.block * a.s_s0[0] + hkv * a.s_s1[0]];
                x.vs = a.scale[1][x.block * a.s_s0[1] + hkv * a.s_s1[1]];
            }
        };
        auto fetch = [&](int slot, int block, int at) {   // one lane
            const uint32_t full = full0 + 8u * slot, dst = ring0 + slot * STAGE;
            if (at == 0) {
                mbar_arrive(full);
                return;
            }
            mbar_arrive_expect_tx(full, STAGE);
#pragma unroll
            for (int h = 0; h < NH; ++h) {
                tma_4d(dst + h * BOX, &map_k, h * RB, at >> 5, hkv, block, full);
                tma_4d(dst + (NH + h) * BOX, &map_v, h * RB, at >> 5, hkv, block, full);
            }
        };
        const int g = lane >> 2, c = lane & 3;
        const int rbase = (blockIdx.z * p.mt + mtile) * 8 * NT;   // first query row of this warp
        // K: lane l names row l & 7 of matrix l >> 3, matrix m being the 16 bytes 4 i + m of eight tokens. In each register the lane
        // then has four neighbouring codes of token g: k columns 2c, 2c + 1 and 2c + 8, 2c + 9 of a k step stand for d = 4c .. 4c + 3.
        // The swizzle moves the 16 bytes i of a row to i ^ (row & 7), or (row / 2) & 3 in rows of 64 bytes; tiles start at
        // multiples of 1024 bytes, so a change of i or of the row's parity is a change of address bits.
        const uint32_t k_lane = (lane & 7) * RB + (((lane >> 3) ^ (RB == 128 ? lane & 7 : (lane & 7) >> 1)) << 4);
        // V: the lane has VB neighbouring codes, at d = VB * g, of tokens 2c, 2c + 1, 2c + 8, 2c + 9: the k columns that its A
        // fragments want. Rows g and g + 8 of M tile j stand for d = VB * g + 2 j and the next one.
        const uint32_t v_lane = NH * BOX + 2 * c * RB + (RB == 128 ? (g ^ (2 * c)) << 4 : (((g >> 1) ^ c) << 4) + (g & 1) * 8);

        uint32_t qf[NT][CH][2], ql[NT][SPLIT ? CH : 1][2];
        float o[NT][DM][4];                             // rows 2c (elements 0, 2) and 2c + 1 (1, 3) of the N tile
        float ref[NT][2], l[NT][2], rs[NT][2];
        int req = request_of(t0) - 1, req_end = t0, part_first = 0, lim_min = 0, whole_end = 0;
        // The next request from tile t on: its query rows as they are in memory ...
        auto ask_request = [&](int t) {
            do ++req;
            while (pre[req + 1] <= t);
            req_end = min(pre[req + 1], t1);
            part_first = t - pre[req];
            lim_min = lens[req] - (a.n - 1);            // what the first new token sees
            // Full tiles before this one are seen by every row: with one new token all of them.
            whole_end = a.n == 1 ? t1 : pre[req] + (p.ragged ? 0 : max(lim_min, 0) / kTile);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                // ---- query row g of the N tile as a B fragment ----
                const int r = rbase + 8 * n + g, tq = r / group;
                const T* q = static_cast<const T*>(a.q) + static_cast<int64_t>(req) * a.q_s0 + static_cast<int64_t>(tq) * a.q_s1 +
                             static_cast<int64_t>(hkv * group + (r - tq * group)) * a.q_s2 + 4 * c;
                const int dmax = r < R ? a.D - 4 * c : 0;
                if constexpr (SPLIT) {
#pragma unroll
                    for (int i = 0; i < CH; ++i) {
                        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                        if (16 * i < dmax) v = p.qvec ? *reinterpret_cast<const float4*>(q + 16 * i) : make_float4(q[16 * i], q[16 * i + 1], q[16 * i + 2], q[16 * i + 3]);
                        qf[n][i][0] = __float_as_uint(v.x);
                        qf[n][i][1] = __float_as_uint(v.y);
                        ql[n][i][0] = __float_as_uint(v.z);
                        ql[n][i][1] = __float_as_uint(v.w);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < CH; ++i) {
                        uint2 v = make_uint2(0u, 0u);
                        if (16 * i < dmax) {
                            const unsigned short* e = reinterpret_cast<const unsigned short*>(q + 16 * i);
                            if (p.qvec)
                                v = *reinterpret_cast<const uint2*>(e);
                            else
                                v = make_uint2(e[0] | (static_cast<uint32_t>(e[1]) << 16), e[2] | (static_cast<uint32_t>(e[3]) << 16));
                        }
                        qf[n][i][0] = v.x;
                        qf[n][i][1] = v.y;
                    }
                }
            }
        };
        // ... and as B fragments: row g of each N tile.
        auto take_request = [&] {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float scale = 1.f, back = 1.f;
                bool infinite;   // logits of this row can only be infinite or NaN, so its result is NaN: also where all of them are -inf
                if constexpr (std::is_same<T, __half>::value) {
                    __half2 top = __float2half2_rn(0.f);
#pragma unroll
                    for (int i = 0; i < CH; ++i)
#pragma unroll
                        for (int h = 0; h < 2; ++h) top = __hmax2(top, __habs2(*reinterpret_cast<const __half2*>(&qf[n][i][h])));
                    const uint32_t lanes = __ballot_sync(0xffffffffu, __half2float(__hmax(top.x, top.y)) == INFINITY);
                    infinite = (lanes >> (lane & 28) & 15u) != 0;
                } else {   // 2^-e with the row's maximum in [2^e, 2^(e + 1))
                    float amax = 0.f;
#pragma unroll
                    for (int i = 0; i < CH; ++i)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const uint32_t u = qf[n][i][h];
                            if constexpr (SPLIT)
                                amax = fmaxf(amax, fmaxf(fabsf(__uint_as_float(u)), fabsf(__uint_as_float(ql[n][i][h]))));
                            else
                                amax = fmaxf(amax, fmaxf(fabsf(__uint_as_float(u << 16)), fabsf(__uint_as_float(u & 0xffff0000u))));
                        }
                    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
                    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
                    infinite = amax == INFINITY;
                    const uint32_t e = min(max(__float_as_uint(amax) >> 23, 1u), 253u);
                    scale = __uint_as_float((254u - e) << 23);
                    back = __uint_as_float(e << 23);
#pragma unroll
                    for (int i = 0; i < CH; ++i) {
                        if constexpr (SPLIT) {
                            const float x0 = __uint_as_float(qf[n][i][0]) * scale, x1 = __uint_as_float(qf[n][i][1]) * scale;
                            const float x2 = __uint_as_float(ql[n][i][0]) * scale, x3 = __uint_as_float(ql[n][i][1]) * scale;
                            qf[n][i][0] = pack_f16(x0, x1);
                            qf[n][i][1] = pack_f16(x2, x3);
                            ql[n][i][0] = pack_rest(x0, x1, qf[n][i][0]);
                            ql[n][i][1] = pack_rest(x2, x3, qf[n][i][1]);
                        } else {
#pragma unroll
                            for (int h = 0; h < 2; ++h)
                                qf[n][i][h] = pack_f16(__uint_as_float(qf[n][i][h] << 16) * scale, __uint_as_float(qf[n][i][h] & 0xffff0000u) * scale);
                        }
                    }
                }
                back = infinite ? __int_as_float(0x7fffffff) : back * (a.softmax_scale * kLog2e);
                rs[n][0] = __shfl_sync(0xffffffffu, back, 8 * c);       // of row 2c
                rs[n][1] = __shfl_sync(0xffffffffu, back, 8 * c + 4);   // of row 2c + 1
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    ref[n][e] = -INFINITY;
                    l[n][e] = 0.f;
                }
#pragma unroll
                for (int j = 0; j < DM; ++j) o[n][j][0] = o[n][j][1] = o[n][j][2] = o[n][j][3] = 0.f;
            }
        };

        int base = t0;
        const int64_t ids = ask_ids(cur, base);
        ask_request(t0);
        take_ids(cur, ids);
        load_scales(cur);
        if (mtile == 0) {
            for (int k = 0; k < min(p.stages, t1 - t0); ++k)
                if (lane == k) fetch(k, cur.block, cur.at);
        }
        __syncwarp();
        take_ids(nxt, ask_ids(nxt, base + 32));
        take_request();

        int slot = 0;
        uint32_t phase = 0;
        for (int t = t0; t < t1; ++t) {
            int k = t - base;
            if (k == 32) {
                cur = nxt;
                base += 32;
                k = 0;
                take_ids(nxt, ask_ids(nxt, base + 32));
            }
            if (k == 16) load_scales(nxt);
            if (t == req_end) {
                ask_request(t);
                take_request();
            }
            const int valid = __shfl_sync(0xffffffffu, cur.at, k) & 31;
            const float ks = __shfl_sync(0xffffffffu, cur.ks, k), vs = __shfl_sync(0xffffffffu, cur.vs, k);
            if (!__all_sync(0xffffffffu, mbar_wait(full0 + 8u * slot, phase, give_up) ? 1 : 0)) break;
            if (valid > 0) {
                const uint32_t kt = ring0 + slot * STAGE;
                // ---- S^T = Kc Q^T: 16 tokens by 8 query rows ----
                float s[NT][4], s2[NT][4];   // every other k step: two chains of products side by side
#pragma unroll
                for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = s2[n][0] = s2[n][1] = s2[n][2] = s2[n][3] = 0.f;
#pragma unroll
                for (int i = 0; i < CH; i += 4) {
                    const uint32_t at = ((kt + k_lane) ^ (i % (RB / 16) * 16)) + (i * 16 / RB) * BOX;
                    uint32_t b[4], d[4];
                    ldmatrix4(at, b);            // tokens 0-7
                    ldmatrix4(at + 8 * RB, d);   // tokens 8-15
#pragma unroll
                    for (int m = 0; m < 4; ++m) {
                        uint32_t f[4];
                        codes_to_f16<E4M3>(b[m], f[0], f[2]);
                        codes_to_f16<E4M3>(d[m], f[1], f[3]);
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            float (&to)[4] = NT == 1 && (m & 1) ? s2[n] : s[n];
                            mma_f16(to, f, qf[n][i + m][0], qf[n][i + m][1]);
                            if constexpr (SPLIT) mma_f16(to, f, ql[n][i + m][0], ql[n][i + m][1]);
                        }
                    }
                }
                if constexpr (NT == 1) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[0][e] += s2[0][e];
                }
                // ---- the codes of V, on their way while the weights are made ----
                uint32_t v[NH][4][VB / 4];   // tokens 2c, 2c + 1, 2c + 8, 2c + 9
#pragma unroll
                for (int h = 0; h < NH; ++h) {
                    const uint32_t vb = kt + v_lane;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t trow = (i & 1) * RB + (i >> 1) * 8 * RB + h * BOX;
                        if constexpr (RB == 128) {
                            const uint32_t at = (vb ^ ((i & 1) << 4)) + trow;
                            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                                         : "=r"(v[h][i][0]), "=r"(v[h][i][1]), "=r"(v[h][i][2]), "=r"(v[h][i][3])
                                         : "r"(at)
                                         : "memory");
                        } else {
                            const uint32_t at = vb + trow;
                            asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v[h][i][0]), "=r"(v[h][i][1]) : "r"(at) : "memory");
                        }
                    }
                }
                // Codes of tokens that do not exist are whatever the block holds, NaN perhaps: their weight is 0, so are they.
                if (valid < kTile) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (2 * c + (i & 1) + (i >> 1) * 8 >= valid) {
#pragma unroll
                            for (int h = 0; h < NH; ++h)
#pragma unroll
                                for (int w = 0; w < VB / 4; ++w) v[h][i][w] = 0u;
                        }
                }
                // ---- weights against the tile's own maximum ----
                // s[0], s[1]: token g, rows 2c, 2c + 1; s[2], s[3]: token g + 8
                const bool whole = valid == kTile && t < whole_end;
                int pos = 0;
                if (!whole) {
                    int col, at;
                    pos = place_of(t - pre[req], col, at);
                }
                uint32_t pb[NT][2], pl[NT][2];
                float gain[NT][2];
                const float lift = value_lift(vs, 41);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float f0 = ks * rs[n][0], f1 = ks * rs[n][1];
                    if (!whole) {
                        const int r = rbase + 8 * n + 2 * c;
                        const int n0 = min(valid, lim_min + (a.n > 1 ? r / group : 0) - pos), n1 = min(valid, lim_min + (a.n > 1 ? (r + 1) / group : 0) - pos);
                        s[n][0] = g < n0 ? s[n][0] * f0 : -INFINITY;
                        s[n][1] = g < n1 ? s[n][1] * f1 : -INFINITY;
                        s[n][2] = g + 8 < n0 ? s[n][2] * f0 : -INFINITY;
                        s[n][3] = g + 8 < n1 ? s[n][3] * f1 : -INFINITY;
                        f0 = f1 = 1.f;
                    }
                    float m0 = fmaxf(s[n][0], s[n][2]), m1 = fmaxf(s[n][1], s[n][3]);
#pragma unroll
                    for (int x = 4; x < 32; x *= 2) {
                        m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, x));
                        m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, x));
                    }
                    m0 = fmaxf(m0, kLowest);   // a row that sees nothing of the tile: every weight 2^-inf
                    m1 = fmaxf(m1, kLowest);
                    // Differences of the sums first: the exponents end at 15 exactly. (2^(S f - m) against the rounded m = max f - 15 is
                    // 2^16, infinite in fp16, from logits of 2^24 on.)
                    const float p0 = ex2_fast(fmaf(s[n][0] - m0, f0, 15.f)), p1 = ex2_fast(fmaf(s[n][1] - m1, f1, 15.f));
                    const float p2 = ex2_fast(fmaf(s[n][2] - m0, f0, 15.f)), p3 = ex2_fast(fmaf(s[n][3] - m1, f1, 15.f));
                    m0 = fmaxf(m0 * f0, kLowest);
                    m1 = fmaxf(m1 * f1, kLowest);
                    const float r0 = m0 + lift, r1 = m1 + lift;
                    if (__any_sync(0xffffffffu, r0 > ref[n][0] + kLag || r1 > ref[n][1] + kLag)) {
                        const float u0 = fmaxf(ref[n][0], r0), u1 = fmaxf(ref[n][1], r1);
                        const float a0 = ex2_fast(ref[n][0] - u0), a1 = ex2_fast(ref[n][1] - u1);
                        ref[n][0] = u0;
                        ref[n][1] = u1;
                        l[n][0] *= a0;
                        l[n][1] *= a1;
#pragma unroll
                        for (int j = 0; j < DM; ++j) {
                            o[n][j][0] *= a0;
                            o[n][j][1] *= a1;
                            o[n][j][2] *= a0;
                            o[n][j][3] *= a1;
                        }
                    }
                    const float w0 = ex2_fast(m0 - ref[n][0]), w1 = ex2_fast(m1 - ref[n][1]);
                    l[n][0] = fmaf(p0 + p2, w0, l[n][0]);   // of tokens g and g + 8: the lanes are added up at the end
                    l[n][1] = fmaf(p1 + p3, w1, l[n][1]);
                    gain[n][0] = w0 * vs;
                    gain[n][1] = w1 * vs;
                    // P^T as a B fragment: row g, tokens 2c, 2c + 1 and 2c + 8, 2c + 9
                    const uint32_t h0 = pack_f16(p0, p1), h1 = pack_f16(p2, p3);
                    pb[n][0] = transpose8(h0);
                    pb[n][1] = transpose8(h1);
                    if constexpr (SPLIT) {
                        pl[n][0] = transpose8(pack_rest(p0, p1, h0));
                        pl[n][1] = transpose8(pack_rest(p2, p3, h1));
                    }
                }
                // A weight of 0 does not keep a NaN code out of a sum. Where some rows see a token and others do not (the new
                // tokens among themselves), NaN codes are taken out of the tile and handed to the rows that see them.
                if constexpr (E4M3 && MANY) {
                    if (!whole) {
                        uint32_t found = 0;   // bit 7 of every byte that is 0x7f or 0xff
#pragma unroll
                        for (int h = 0; h < NH; ++h)
#pragma unroll
                            for (int i = 0; i < 4; ++i)
#pragma unroll
                                for (int w = 0; w < VB / 4; ++w) found |= (v[h][i][w] & 0x7f7f7f7fu) + 0x01010101u;
                        if (__any_sync(0xffffffffu, (found & 0x80808080u) != 0)) {
                            uint32_t sees[NT][2];   // bit k: the row sees token k of the tile
#pragma unroll
                            for (int n = 0; n < NT; ++n)
#pragma unroll
                                for (int e = 0; e < 2; ++e)
                                    sees[n][e] = (1u << max(min(valid, lim_min + (rbase + 8 * n + 2 * c + e) / group - pos), 0)) - 1u;
#pragma unroll
                            for (int h = 0; h < NH; ++h)
#pragma unroll
                                for (int j = 0; j < VB; ++j) {
                                    const uint32_t byte = 0xffu << (8 * (j & 3));
                                    uint32_t tokens = 0;   // those whose code at this place is NaN
#pragma unroll
                                    for (int i = 0; i < 4; ++i)
                                        if ((~v[h][i][j / 4] & byte & 0x7f7f7f7fu) == 0) {
                                            tokens |= 1u << (2 * c + (i & 1) + (i >> 1) * 8);
                                            v[h][i][j / 4] &= ~byte;
                                        }
                                    tokens |= __shfl_xor_sync(0xffffffffu, tokens, 1);
                                    tokens |= __shfl_xor_sync(0xffffffffu, tokens, 2);
#pragma unroll
                                    for (int n = 0; n < NT; ++n)
#pragma unroll
                                        for (int e = 0; e < 2; ++e)
                                            if (tokens & sees[n][e]) o[n][h * (VB / 2) + j / 2][2 * (j & 1) + e] = __int_as_float(0x7fffffff);
                                }
                        }
                    }
                }
                // ---- O^T += (w vs) (Vc^T P^T) ----
#pragma unroll
                for (int h = 0; h < NH; ++h) {
#pragma unroll
                    for (int w = 0; w < VB / 4; ++w) {
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const uint32_t sel = i == 0 ? 0x5140 : 0x7362;
                            uint32_t f[4];
                            codes_to_f16<E4M3>(__byte_perm(v[h][0][w], v[h][1][w], sel), f[0], f[1]);
                            codes_to_f16<E4M3>(__byte_perm(v[h][2][w], v[h][3][w], sel), f[2], f[3]);
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                float (&oj)[4] = o[n][h * (VB / 2) + w * 2 + i];
                                float tmp[4] = {0.f, 0.f, 0.f, 0.f};
                                mma_f16(tmp, f, pb[n][0], pb[n][1]);
                                if constexpr (SPLIT) mma_f16(tmp, f, pl[n][0], pl[n][1]);
                                oj[0] = fmaf(tmp[0], gain[n][0], oj[0]);
                                oj[1] = fmaf(tmp[1], gain[n][1], oj[1]);
                                oj[2] = fmaf(tmp[2], gain[n][0], oj[2]);
                                oj[3] = fmaf(tmp[3], gain[n][1], oj[3]);
                            }
                        }
                    }
                }
            }

            __syncwarp();
            // ---- refill: the slot just read, or, where other warps read it too, the one before it ----
            if (p.mt > 1 && lane == 0) mbar_arrive(empty0 + 8u * slot);
            if (mtile == 0) {
                const int lag = p.mt > 1 ? 1 : 0;
                const int u = t - lag + p.stages;   // the tile to fetch
                if (t - lag >= t0 && u < t1) {
                    const int ku = u - base;
                    const int to = slot >= lag ? slot - lag : p.stages - 1;
                    if (lane == (ku & 31)) {   // the lane that knows the tile
                        const uint32_t ph = to > slot ? phase ^ 1u : phase;   // the slot before slot 0 was read in the round before
                        if (lag == 0 || mbar_wait(empty0 + 8u * to, ph, give_up)) fetch(to, ku < 32 ? cur.block : nxt.block, ku < 32 ? cur.at : nxt.at);
                    }
                    __syncwarp();
                }
            }
            if (++slot == p.stages) {
                slot = 0;
                phase ^= 1u;
            }
            if (t + 1 != req_end) continue;

            // ---- the request's part in this range is done: written directly when it is all of it ----
            const bool alone = part_first == 0 && t + 1 == pre[req + 1];
            const int64_t part = (static_cast<int64_t>(range) + req) * a.n * a.Hq;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int x = 4; x < 32; x *= 2) {
                    l[n][0] += __shfl_xor_sync(0xffffffffu, l[n][0], x);
                    l[n][1] += __shfl_xor_sync(0xffffffffu, l[n][1], x);
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int r = rbase + 8 * n + 2 * c + e;
                    if (r >= R) continue;
                    const int tq = r / group, hq = hkv * group + (r - tq * group);
                    const float inv = l[n][e] == 0.f ? 0.f : 1.f / l[n][e];
                    T* out = static_cast<T*>(a.out) + static_cast<int64_t>(req) * a.o_s0 + static_cast<int64_t>(tq) * a.o_s1 + static_cast<int64_t>(hq) * a.o_s2;
                    const bool vec = aligned16(out);
                    const int64_t row = part + static_cast<int64_t>(tq) * a.Hq + hq;
#pragma unroll
                    for (int h = 0; h < NH; ++h) {
                        const int d = h * RB + g * VB;
                        if (d >= a.D) continue;
                        float f[VB];
#pragma unroll
                        for (int j = 0; j < VB; ++j) f[j] = o[n][h * (VB / 2) + j / 2][2 * (j & 1) + e];
                        if (!alone) {
#pragma unroll
                            for (int j = 0; j < VB; j += 4) *reinterpret_cast<float4*>(ws_acc + row * a.D + d + j) = make_float4(f[j], f[j + 1], f[j + 2], f[j + 3]);
                            continue;
                        }
                        constexpr int VN = Vec16<T>::N;
#pragma unroll
                        for (int j = 0; j < VB; j += VN) {
                            float x[VN];
#pragma unroll
                            for (int i = 0; i < VN; ++i) x[i] = f[j + i] * inv;
                            if (vec) {
                                *reinterpret_cast<uint4*>(out + d + j) = pack16<T>(x);
                            } else {
#pragma unroll
                                for (int i = 0; i < VN; ++i) out[d + j + i] = Cvt<T>::from_f(x[i]);
                            }
                        }
                    }
                    if (!alone && g == 0) *reinterpret_cast<float2*>(ws_ml + row * 2) = make_float2(ref[n][e], l[n][e]);
                }
            }
        }
    }

    // A thread that gave up a wait reports it; copies that might still be in flight get time to land before the shared
    // memory of the CTA is released.
    if (*give_up) {
        if (lane == 0) report_status(a.status, 3);
        const unsigned long long t_begin = global_ns();
        while (global_ns() - t_begin < 2000000ull) __nanosleep(1000);
    }
}

// Merges the parts of a request that several ranges had, and writes zeros for an empty one. `wpr` warps share a query row: the
// launch gives a row as many as it has parts for on average, as the parts of one long request are too many for one warp to
// read one after the other (four requests of 30011 to 131072 tokens: 145 us with one warp to a row, 6 with eight that ask for
// eight parts at a time).
constexpr int kMergeWarps = 8;

// HD: head_dim rounded up to 64 (two parts of a row side by side in a warp), 128 or 256. U: parts that a warp asks for at once.
template <typename T, int HD, int U>
__global__ void __launch_bounds__(32 * kMergeWarps, U > 4 ? 1 : HD > 128 ? 3 : 4) quant_combine_kernel(const QuantAttnArgs a, int n_range, int wpr, const float* __restrict__ ws_acc,
                                                                         const float* __restrict__ ws_ml) {
    __shared__ int s_part[kMergeWarps][2];
    constexpr bool WIDE = HD > 128;
    constexpr int NV = WIDE ? 8 : 4, SIDE = HD == 64 ? 2 : 1, LANES = 32 / SIDE;
    __shared__ float s_acc[kMergeWarps][32 * NV + 1];
    const int i = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int before = 0, all = 0;
    for (int r = threadIdx.x; r < a.B; r += 32 * kMergeWarps) {
        const int n = tiles_of(a, quant_len(a, r));
        all += n;
        if (r < i) before += n;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        before += __shfl_xor_sync(0xffffffffu, before, o);
        all += __shfl_xor_sync(0xffffffffu, all, o);
    }
    if (lane == 0) {
        s_part[warp][0] = before;
        s_part[warp][1] = all;
    }
    __syncthreads();
    before = all = 0;
#pragma unroll
    for (int w = 0; w < kMergeWarps; ++w) {
        before += s_part[w][0];
        all += s_part[w][1];
    }
    const int tiles = tiles_of(a, quant_len(a, i));
    const int used = used_ranges(all, n_range);
    // Range c has the tiles [all * c / used, all * (c + 1) / used): every one of the used ranges has some.
    int c_first = 0, parts = 0;
    if (tiles > 0) {
        auto range_of = [&](int t) {
            const int64_t c = ((static_cast<int64_t>(t) + 1) * used - 1) / all;
            return static_cast<int>(c < used - 1 ? c : used - 1);
        };
        c_first = range_of(before);
        parts = range_of(before + tiles - 1) - c_first + 1;
    }
    // Also where there is nothing to merge: this grid must not be done before the one that it depends on.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (parts == 1) return;   // written by that range
    const int row = blockIdx.y * (kMergeWarps / wpr) + warp / wpr, sub = warp % wpr;
    const bool here = row < a.n * a.Hq;
    const int64_t rows = static_cast<int64_t>(a.n) * a.Hq;
    const float* ml = ws_ml + ((static_cast<int64_t>(c_first) + i) * rows + row) * 2;
    const float* acc = ws_acc + ((static_cast<int64_t>(c_first) + i) * rows + row) * a.D;
    const int dl = 4 * (lane % LANES);
    float v[NV];   // d = dl .. + 3, and 128 further
#pragma unroll
    for (int e = 0; e < NV; ++e) v[e] = 0.f;
    float L = 0.f;
    if (here) {
        float M = kLowest;
        for (int c = lane; c < parts; c += 32) M = fmaxf(M, ml[c * rows * 2]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
        const bool d0 = dl < a.D, d1 = dl + 128 < a.D;
        const int by = wpr * SIDE;
        for (int c = sub * SIDE + lane / LANES; c < parts; c += U * by) {
            float2 x[U];
            float4 y[U], z[WIDE ? U : 1];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t at = (c + u * by) * rows;
                const bool in = c + u * by < parts;
                x[u] = in ? *reinterpret_cast<const float2*>(ml + at * 2) : make_float2(-INFINITY, 0.f);
                y[u] = in && d0 ? *reinterpret_cast<const float4*>(acc + at * a.D + dl) : make_float4(0.f, 0.f, 0.f, 0.f);
                if constexpr (WIDE) z[u] = in && d1 ? *reinterpret_cast<const float4*>(acc + at * a.D + dl + 128) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float w = exp2f(x[u].x - M);
                L = fmaf(x[u].y, w, L);
                v[0] = fmaf(y[u].x, w, v[0]);
                v[1] = fmaf(y[u].y, w, v[1]);
                v[2] = fmaf(y[u].z, w, v[2]);
                v[3] = fmaf(y[u].w, w, v[3]);
                if constexpr (WIDE) {
                    v[4] = fmaf(z[u].x, w, v[4]);
                    v[5] = fmaf(z[u].y, w, v[5]);
                    v[6] = fmaf(z[u].z, w, v[6]);
                    v[7] = fmaf(z[u].w, w, v[7]);
                }
            }
        }
    }
    if constexpr (SIDE == 2) {
        L += __shfl_xor_sync(0xffffffffu, L, 16);
#pragma unroll
        for (int e = 0; e < NV; ++e) v[e] += __shfl_xor_sync(0xffffffffu, v[e], 16);
    }
    if (wpr > 1) {
#pragma unroll
        for (int e = 0; e < NV; ++e) s_acc[warp][e * 32 + lane] = v[e];
        if (lane == 0) s_acc[warp][32 * NV] = L;
        __syncthreads();
        if (sub != 0) return;
        for (int w = 1; w < wpr; ++w) {
#pragma unroll
            for (int e = 0; e < NV; ++e) v[e] += s_acc[warp + w][e * 32 + lane];
            L += s_acc[warp + w][32 * NV];
        }
    }
    if (!here) return;
    const float inv = L == 0.f ? 0.f : 1.f / L;
    const int t = row / a.Hq, h = row - t * a.Hq;
    T* out = static_cast<T*>(a.out) + static_cast<int64_t>(i) * a.o_s0 + static_cast<int64_t>(t) * a.o_s1 + static_cast<int64_t>(h) * a.o_s2;
#pragma unroll
    for (int e = 0; e < NV; ++e) {
        const int d = dl + (e & 3) + (e >> 2) * 128;
        if (d < a.D && lane < LANES) out[d] = Cvt<T>::from_f(v[e] * inv);
    }
}

// ---------------------------------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------------------------------
using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                              const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encode_fn() {
    static EncodeFn fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult qres;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &qres) == cudaSuccess && qres == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeFn>(ptr);
    });
    return fn;
}

// [head_dim, position, head, block] of one cache whatever its strides; a box is 16 positions of a head. Bytes of a row
// beyond head_dim and rows beyond the block arrive as zeros.
bool encode_map(const QuantAttnArgs& a, const QuantPlan& p, int m, CUtensorMap* map) {
    EncodeFn fn = encode_fn();
    if (!fn) return false;
    const int rb = p.hd < 128 ? p.hd : 128;
    auto stride = [](int64_t s, int64_t extent) { return static_cast<cuuint64_t>(extent > 1 ? s : 16); };
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(a.D), static_cast<cuuint64_t>(a.block_size), static_cast<cuuint64_t>(a.Hkv), static_cast<cuuint64_t>(a.blocks)};
    const cuuint64_t strides[3] = {stride(a.c_s1[m], a.block_size), stride(a.c_s2[m], a.Hkv), stride(a.c_s0[m], a.blocks)};
    const cuuint32_t box[4] = {static_cast<cuuint32_t>(rb), kTile, 1, 1};
    const cuuint32_t ones[4] = {1, 1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(a.cache[m]), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
              rb == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Whether the split kernel takes these arguments, and how it cuts them.
bool make_quant_plan(const QuantAttnArgs& a, int sm_count, int max_smem, QuantPlan& p) {
    if (a.force_plain || a.D % 16 != 0 || a.block_size >= (1 << 25) || a.blocks <= 0 || a.cols <= 0) return false;
    if (a.D > 256) return false;
    const int64_t block_tiles = (a.block_size + kTile - 1) / kTile;
    if (a.B > kQMaxB || static_cast<int64_t>(a.B) * a.cols * block_tiles >= (1ll << 30) || a.blocks >= (1ll << 31)) return false;
    for (int m = 0; m < 2; ++m) {
        auto ok = [](int64_t s, int64_t extent) { return extent <= 1 || (s > 0 && s % 16 == 0 && s < (1ll << 40)); };
        if (a.c_s3[m] != 1 || !ok(a.c_s0[m], a.blocks) || !ok(a.c_s1[m], a.block_size) || !ok(a.c_s2[m], a.Hkv) ||
            reinterpret_cast<uintptr_t>(a.cache[m]) % 16 != 0)
            return false;
    }
    p = QuantPlan{};
    p.block_tiles = static_cast<int>(block_tiles);
    p.ragged = a.block_size % kTile != 0;
    p.hd = a.D <= 64 ? 64 : a.D <= 128 ? 128 : 256;
    const int R = a.n * (a.Hq / a.Hkv);
    const bool f32 = a.dt == Dt::F32;
    p.nt = R > 8 && p.hd <= 128 && !f32 ? 2 : 1;
    const int warps = split_warps(f32, p.hd, p.nt);
    p.mt = std::min((R + 8 * p.nt - 1) / (8 * p.nt), warps);
    p.n_z = (R + p.mt * 8 * p.nt - 1) / (p.mt * 8 * p.nt);
    // Heads of a CTA: the divisor of Hkv that keeps most warps busy, the largest of those.
    int busy = 0;
    for (int h = 1; h <= warps / p.mt; ++h) {
        const int b = h * (warps / p.mt / h);
        if (a.Hkv % h == 0 && h <= 8 && b >= busy) {
            busy = b;
            p.hw = h;
        }
    }
    p.n_hg = a.Hkv / p.hw;
    p.tw = warps / p.mt / p.hw;
    const int teams = p.hw * p.tw, stage = 2 * kTile * p.hd;
    const int fixed = 1024 + teams * 2 * kQMaxStages * 8 + (2 * a.B + 1) * 4 + 64;
    p.stages = std::min((max_smem - fixed) / (teams * stage), kQMaxStages);
    if (p.stages < 2) return false;
    int off = teams * p.stages * stage;
    auto take = [&](int bytes) {
        const int at = off;
        off += (bytes + 15) / 16 * 16;
        return at;
    };
    p.off_bars = take(teams * 2 * p.stages * 8);
    p.off_pre = take((a.B + 1) * 4);
    p.off_len = take(a.B * 4);
    p.off_flag = take(4);
    p.smem_bytes = off + 1024;
    if (p.smem_bytes > max_smem) return false;
    const int64_t most = static_cast<int64_t>(a.B) * a.cols * block_tiles;
    const int64_t ranges = std::max<int64_t>(1, (most + kTilesPerRange - 1) / kTilesPerRange);
    p.n_cta = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(sm_count / (p.n_hg * p.n_z), (ranges + p.tw - 1) / p.tw)));
    p.n_range = p.n_cta * p.tw;
    const int64_t el = a.dt == Dt::F32 ? 4 : 2;
    p.qvec = reinterpret_cast<uintptr_t>(a.q) % (4 * el) == 0 && a.q_s0 % 4 == 0 && a.q_s1 % 4 == 0 && a.q_s2 % 4 == 0;
    return true;
}

int64_t part_rows(const QuantAttnArgs& a, const QuantPlan& p) { return (static_cast<int64_t>(p.n_range) + a.B) * a.n * a.Hq; }

template <typename T, bool E4M3, int HD, int NT, bool MANY>
void launch_split(const QuantAttnArgs& a, const QuantPlan& p, const CUtensorMap& mk, const CUtensorMap& mv, float* acc, float* ml, int max_smem, cudaStream_t st) {
    auto kern = quant_split_kernel<T, E4M3, HD, NT, MANY>;
    constexpr int threads = 32 * split_warps(std::is_same<T, float>::value, HD, NT);
    // once per kernel and device: the call is not free, and the limit may as well be the device's
    static std::atomic<uint64_t> done{0};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 64 || !(done.load(std::memory_order_acquire) >> dev & 1)) {
        cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, max_smem);
        if (dev < 64) done.fetch_or(1ull << dev, std::memory_order_release);
    }
    kern<<<dim3(p.n_cta, p.n_hg, p.n_z), threads, p.smem_bytes, st>>>(a, p, mk, mv, acc, ml);
    int wpr = 1;
    while (wpr < kMergeWarps && wpr * (HD == 64 ? 16 : 8) * a.B < p.n_range) wpr *= 2;   // eight parts to a warp on average
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.B, (a.n * a.Hq + kMergeWarps / wpr - 1) / (kMergeWarps / wpr), 1);
    cfg.blockDim = dim3(32 * kMergeWarps);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, wpr == kMergeWarps ? quant_combine_kernel<T, HD, 8> : quant_combine_kernel<T, HD, 4>, a, p.n_range, wpr, static_cast<const float*>(acc), static_cast<const float*>(ml));
}

template <typename T>
void launch_split_t(const QuantAttnArgs& a, const QuantPlan& p, const CUtensorMap& mk, const CUtensorMap& mv, float* acc, float* ml, int max_smem, cudaStream_t st) {
    auto go = [&](auto e4m3, auto hd) {
        auto rows = [&](auto nt) {
            if constexpr (e4m3.value) {   // int8 has no NaN
                if (a.n > 1) return launch_split<T, true, hd.value, nt.value, true>(a, p, mk, mv, acc, ml, max_smem, st);
            }
            launch_split<T, e4m3.value, hd.value, nt.value, false>(a, p, mk, mv, acc, ml, max_smem, st);
        };
        if constexpr (!std::is_same<T, float>::value && hd.value <= 128) {
            if (p.nt == 2) return rows(std::integral_constant<int, 2>{});
        }
        rows(std::integral_constant<int, 1>{});
    };
    auto widths = [&](auto e4m3) {
        if (p.hd == 64)
            go(e4m3, std::integral_constant<int, 64>{});
        else if (p.hd == 128)
            go(e4m3, std::integral_constant<int, 128>{});
        else
            go(e4m3, std::integral_constant<int, 256>{});
    };
    a.e4m3 ? widths(std::true_type{}) : widths(std::false_type{});
}

}  // namespace

int64_t quantized_attention_workspace_bytes(const QuantAttnArgs& a, int sm_count, int max_smem) {
    QuantPlan p;
    if (!make_quant_plan(a, sm_count, max_smem, p)) return 0;
    return part_rows(a, p) * (a.D + 2) * 4 + 256;
}

const char* launch_quantized_attention(const QuantAttnArgs& a, void* ws, int sm_count, int max_smem, cudaStream_t st) {
    QuantPlan p;
    CUtensorMap mk, mv;
    if (ws != nullptr && make_quant_plan(a, sm_count, max_smem, p) && encode_map(a, p, 0, &mk) && encode_map(a, p, 1, &mv)) {
        const uintptr_t base = (reinterpret_cast<uintptr_t>(ws) + 255) & ~static_cast<uintptr_t>(255);
        float* acc = reinterpret_cast<float*>(base);
        float* ml = acc + part_rows(a, p) * a.D;
        if (a.dt == Dt::F16)
            launch_split_t<__half>(a, p, mk, mv, acc, ml, max_smem, st);
        else if (a.dt == Dt::BF16)
            launch_split_t<__nv_bfloat16>(a, p, mk, mv, acc, ml, max_smem, st);
        else
            launch_split_t<float>(a, p, mk, mv, acc, ml, max_smem, st);
        return "split";
    }
    const dim3 grid(a.B, a.n * a.Hq);
    if (a.dt == Dt::F16)
        quant_plain_kernel<__half><<<grid, 32 * kPlainWarps, 0, st>>>(a);
    else if (a.dt == Dt::BF16)
        quant_plain_kernel<__nv_bfloat16><<<grid, 32 * kPlainWarps, 0, st>>>(a);
    else
        quant_plain_kernel<float><<<grid, 32 * kPlainWarps, 0, st>>>(a);
    return "plain";
}

}  // namespace k
}  // namespace b200
