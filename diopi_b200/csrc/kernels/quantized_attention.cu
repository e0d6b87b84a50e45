// Attention of the newest tokens over a paged cache of 8-bit codes with one scale for each (block, K/V head)
// (diopiQuantizedPagedAttention). With K/V rows j of request i in block b_j, codes kc, vc and scales ks, vs:
//     x_j = softmax_scale * ks[b_j] * (q . kc_j),   out = sum_j softmax(x)_j * vs[b_j] * vc_j
// New token t of n sees the first L - (n - 1 - t) tokens; a row that sees none gives zeros.
//
// quant_split_kernel (block_size and head_dim multiples of 16, head_dim up to 256) is bound by the bytes of the codes. The
// query rows that share a K/V head (n * group of them) are the M extent of mma.sync m16n8k16 in fp16 with fp32
// accumulators, as in token_decode_gqa.cu: every code of either kind is an fp16 number, so nothing is lost by the
// conversion in registers, and the scales stay outside the products. A tile is 16 tokens of one K/V head, always inside one
// block, hence one ks and one vs:
//     S = Q Kc^T;  m = max(S * f), f = ks * softmax_scale * log2 e;  P = 2^(S f - m + 15);  O += (2^(m - ref) vs) (P Vc)
// The weights are taken against the tile's own maximum, so that they fill fp16's range (2^15 down to 2^-24: what is lost is
// below 2^-40 of the tile's largest weight) whatever the other tiles hold, and the
// product of a tile is added in fp32 with its factor; ref is only raised when a tile exceeds it by 2^40. Queries are scaled
// by the power of two that brings their row's maximum to [1, 2) before they become fp16 (bf16 and fp32 reach further than
// fp16 does); fp32 queries and their weights are split into two fp16 numbers each, with two products.
//
// Work split: a step is TT tokens of hw K/V heads; the steps of the batch are cut into equal ranges, one per CTA, and the parts of a
// request that fell to several CTAs are merged by quant_combine_kernel (a programmatic dependent launch). A request that
// one CTA has whole is written by it directly. Eight consumer warps are (token tile, M tile, K/V head); one producer warp
// looks up the blocks two batches of steps ahead and their scales one ahead, and fetches a tile of hw heads with one TMA
// load each for K and V ([head][token][128 bytes], swizzled: the reads below are free of bank conflicts whatever the layout of
// the cache in memory).
//
// quant_plain_kernel: any width, strides and block size; one CTA to a query row, a warp to every fourth token.
#include <cuda.h>

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
        const float mn = fmaxf(m, x);
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
constexpr int kQWarps = 8;                      // consumer warps
constexpr int kQThreads = 32 * (kQWarps + 1);
constexpr int kQMaxStages = 16;
constexpr int kQMaxB = 4096;
constexpr int kTile = 16;                       // tokens of a tile
constexpr int kStepsPerCta = 2;                 // a CTA gets this many steps at least, so that short batches are not cut into crumbs

struct QuantPlan {
    int hd;           // 64, 128 or 256: head_dim rounded up
    int hw;           // K/V heads of a CTA: a divisor of Hkv
    int n_hg;         // CTAs along the K/V heads
    int mt;           // M tiles of 16 query rows of a CTA
    int n_z;          // CTAs along the query rows of a K/V head (more than 128 of them)
    int tw;           // token tiles that the warps work on side by side
    int ts;           // token tiles that a warp works through in one step
    int tt;           // tokens of a step: 16 * tw * ts
    int items;        // (tile, head) pairs of a step: hw * tw * ts, at most 16
    int stage_bytes, nstages, n_cta;
    int off_meta, off_bars, off_pre, off_len, off_red, off_flag, smem_bytes;
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

// Steps [t, t1) of the flattened (request, step) pairs.
struct QuantWalk {
    const int* pre;   // pre[i] = first step of request i
    int t, t1, i;
    __device__ void init(const int* pre_, int B, int t0_, int t1_) {
        pre = pre_;
        t = t0_;
        t1 = t1_;
        int lo = 0, hi = B;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (pre[mid + 1] > t)
                hi = mid;
            else
                lo = mid + 1;
        }
        i = lo;
    }
    __device__ bool next(int& req, int& step, bool& last) {
        if (t >= t1) return false;
        while (pre[i + 1] <= t) ++i;
        req = i;
        step = t - pre[i];
        ++t;
        last = t == t1 || t == pre[i + 1];
        return true;
    }
};

__device__ __forceinline__ int used_ctas(int total, int n_cta) { return max(1, min(n_cta, (total + kStepsPerCta - 1) / kStepsPerCta)); }

template <typename T, bool E4M3, int HD>
__global__ void __launch_bounds__(kQThreads, 1)
    quant_split_kernel(const QuantAttnArgs a, const QuantPlan p, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                       float* __restrict__ ws_acc, float* __restrict__ ws_ml) {
    constexpr bool SPLIT = std::is_same<T, float>::value;   // two fp16 numbers for each fp32 one
    constexpr int RB = HD < 128 ? HD : 128;                 // bytes of a row of one TMA box
    constexpr int NH = HD / RB;                             // boxes side by side (head_dim 256: 2)
    constexpr int CH = HD / 16;                             // k steps of Q K^T: 16 bytes of codes each
    constexpr int VB = RB / 8;                              // bytes of a V row that a lane takes from each box
    constexpr int DN = HD / 8;                              // n tiles of P V
    constexpr int HEAD_TILE = kTile * RB;                   // bytes of one head's tile in a box
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);   // the swizzle goes by address bits
    float4* meta = reinterpret_cast<float4*>(smem + p.off_meta);                          // [stage][item]: ks, vs, tokens
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + p.off_bars);                      // full[nstages], empty[nstages], merge[2]
    int* pre = reinterpret_cast<int*>(smem + p.off_pre);
    int* lens = reinterpret_cast<int*>(smem + p.off_len);
    float* red = reinterpret_cast<float*>(smem + p.off_red);
    volatile int* give_up = reinterpret_cast<volatile int*>(smem + p.off_flag);

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int group = a.Hq / a.Hkv;
    const int R = a.n * group;                 // query rows of a K/V head
    const int hg0 = blockIdx.y * p.hw;
    const int active = p.hw * p.mt * p.tw;     // consumer warps with work

    if (tid == 0) {
        for (int s = 0; s < p.nstages; ++s) {
            mbar_init(smem_u32(&bars[s]), 1);
            mbar_init(smem_u32(&bars[p.nstages + s]), active);
        }
        mbar_init(smem_u32(&bars[2 * p.nstages]), active);
        mbar_init(smem_u32(&bars[2 * p.nstages + 1]), active);
        *give_up = 0;
        pre[0] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    for (int i = tid; i < a.B; i += kQThreads) {
        const int L = quant_len(a, i);
        lens[i] = L;
        pre[i + 1] = (L + p.tt - 1) / p.tt;
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

    const int total = pre[a.B];
    const int used = used_ctas(total, p.n_cta), cta = blockIdx.x;
    if (cta >= used) return;
    const int t0 = static_cast<int>(static_cast<int64_t>(total) * cta / used);
    const int t1 = static_cast<int>(static_cast<int64_t>(total) * (cta + 1) / used);
    const uint32_t ring0 = smem_u32(smem);
    const uint32_t box_bytes = static_cast<uint32_t>(p.hw) * HEAD_TILE;
    const uint32_t tiles = static_cast<uint32_t>(p.tw * p.ts);
    const uint32_t v_off = tiles * NH * box_bytes;

    if (warp == kQWarps) {
        // =========================== producer warp ===============================
        // A lane is one (token tile, head) pair of one of the next 32 / items steps. Three batches of steps are on their way:
        // the block ids of one are being loaded, the scales of the one before, and the one before that is issued.
        const int per_batch = 32 / p.items;
        const int sb = lane / p.items, item = lane - sb * p.items;
        const int tile = item / p.hw, hl = item - tile * p.hw;
        struct Batch {
            int n = 0, valid = 0, at = 0;
            int64_t block = -1;
            float ks = 0.f, vs = 0.f;
        } cur, nxt, far;
        QuantWalk walk;
        walk.init(pre, a.B, t0, t1);
        auto load_ids = [&](Batch& b) {
            int req = 0, step = 0, my_req = -1, my_step = 0;
            bool last;
            b.n = 0;
            for (; b.n < per_batch; ++b.n) {
                if (!walk.next(req, step, last)) break;
                if (b.n == sb) {
                    my_req = req;
                    my_step = step;
                }
            }
            b.valid = 0;
            if (my_req >= 0) {
                const int pos = my_step * p.tt + tile * kTile;
                b.valid = max(0, min(kTile, lens[my_req] - pos));
                if (b.valid > 0) {
                    const int col = pos / a.block_size;
                    b.at = pos - col * a.block_size;
                    b.block = load_index(a.table, my_req, col);
                }
            }
        };
        auto load_scales = [&](Batch& b) {
            if (b.valid > 0) {
                if (b.block < 0 || b.block >= a.blocks) {
                    report_status(a.status, 1);
                    b.valid = 0;
                } else {
                    b.ks = a.scale[0][b.block * a.s_s0[0] + static_cast<int64_t>(hg0 + hl) * a.s_s1[0]];
                    b.vs = a.scale[1][b.block * a.s_s0[1] + static_cast<int64_t>(hg0 + hl) * a.s_s1[1]];
                }
            }
        };
        load_ids(nxt);
        load_ids(far);
        load_scales(nxt);
        int ring = 0;
        uint32_t phase = 0;
        bool ok = true;
        while (ok && nxt.n > 0) {
            cur = nxt;
            nxt = far;
            load_ids(far);
            load_scales(nxt);
            for (int s = 0; s < cur.n; ++s) {
                const uint32_t full = smem_u32(&bars[ring]);
                const bool mine = sb == s, load = mine && hl == 0 && cur.valid > 0;
                const uint32_t n_load = __popc(__ballot_sync(0xffffffffu, load));
                if (lane == 0) ok = mbar_wait(smem_u32(&bars[p.nstages + ring]), phase ^ 1u, give_up);
                ok = __all_sync(0xffffffffu, ok ? 1 : 0) != 0;
                if (!ok) break;
                if (mine) meta[ring * p.items + item] = make_float4(cur.ks, cur.vs, static_cast<float>(cur.valid), 0.f);
                __syncwarp();
                if (lane == 0) mbar_arrive_expect_tx(full, n_load * 2u * NH * box_bytes);
                __syncwarp();
                if (load) {
                    const uint32_t dst = ring0 + static_cast<uint32_t>(ring) * p.stage_bytes + static_cast<uint32_t>(tile) * NH * box_bytes;
#pragma unroll
                    for (int h = 0; h < NH; ++h) {
                        tma_4d(dst + h * box_bytes, &map_k, h * RB, cur.at, hg0, static_cast<int>(cur.block), full);
                        tma_4d(dst + v_off + h * box_bytes, &map_v, h * RB, cur.at, hg0, static_cast<int>(cur.block), full);
                    }
                }
                if (++ring == p.nstages) {
                    ring = 0;
                    phase ^= 1u;
                }
            }
        }
    } else if (warp < active) {
        // =========================== consumer warps ==============================
        const int hl = warp % p.hw, mtile = (warp / p.hw) % p.mt, tok = warp / (p.hw * p.mt);
        const int hkv = hg0 + hl;
        const int g = lane >> 2, c = lane & 3;
        const int r0 = (blockIdx.z * p.mt + mtile) * 16 + g, r1 = r0 + 8;   // the two query rows of this thread's accumulators
        const int tq0 = r0 / group, tq1 = r1 / group;                       // their new tokens
        const int64_t row0 = static_cast<int64_t>(tq0) * a.Hq + hkv * group + (r0 - tq0 * group);
        const int64_t row1 = static_cast<int64_t>(tq1) * a.Hq + hkv * group + (r1 - tq1 * group);
        // K: lane l names row l & 7 of matrix l >> 3, matrix m being the 16 bytes 4 i + m of eight tokens. In each register the lane
        // then has four neighbouring codes of token g: k columns 2c, 2c + 1 and 2c + 8, 2c + 9 of a k step stand for d = 4c .. 4c + 3.
        const int krow = lane & 7, ksw = RB == 128 ? krow : (krow >> 1);
        // V: the lane has VB neighbouring codes, at d = VB * g, of tokens 2c, 2c + 1, 2c + 8, 2c + 9: the k rows that its B fragments
        // want. Column g of n tile j stands for d = VB * g + j.
        const uint32_t v_lane = RB == 128 ? static_cast<uint32_t>(2 * c * 128) : static_cast<uint32_t>(2 * c * 64);

        uint32_t qf[CH][4], ql[SPLIT ? CH : 1][4];
        float o[DN][4];
        float ref0 = -INFINITY, ref1 = -INFINITY, l0 = 0.f, l1 = 0.f, rs0 = 0.f, rs1 = 0.f;
        int cur_req = -1, part_first = 0, lim0 = 0, lim1 = 0, lim_min = 0;
        uint32_t merge_phase = 0;

        QuantWalk walk;
        walk.init(pre, a.B, t0, t1);
        int req, step;
        bool last;
        int ring = 0;
        uint32_t phase = 0;
        while (walk.next(req, step, last)) {
            if (req != cur_req) {
                cur_req = req;
                part_first = step;
                ref0 = ref1 = -INFINITY;
                l0 = l1 = 0.f;
#pragma unroll
                for (int j = 0; j < DN; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
                const int L = lens[req];
                lim_min = L - (a.n - 1);            // what the first new token sees
                lim0 = lim_min + tq0;
                lim1 = lim_min + tq1;
                // ---- the query rows as A fragments ----
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int r = half ? r1 : r0;
                    const int tq = half ? tq1 : tq0;
                    const T* q = static_cast<const T*>(a.q) + static_cast<int64_t>(req) * a.q_s0 + static_cast<int64_t>(tq) * a.q_s1 +
                                 static_cast<int64_t>(hkv * group + (r - tq * group)) * a.q_s2;
                    float amax = 0.f, scale = 1.f, back = 1.f;
                    float x[CH][4];
#pragma unroll
                    for (int k = 0; k < CH; ++k) {
                        const int d = 16 * k + 4 * c;
                        x[k][0] = x[k][1] = x[k][2] = x[k][3] = 0.f;
                        if (r < R && d < a.D) {
                            if (p.qvec) {
                                if constexpr (SPLIT) {
                                    const float4 v = *reinterpret_cast<const float4*>(q + d);
                                    x[k][0] = v.x;
                                    x[k][1] = v.y;
                                    x[k][2] = v.z;
                                    x[k][3] = v.w;
                                } else {
                                    const uint2 v = *reinterpret_cast<const uint2*>(q + d);
                                    const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
                                    for (int i = 0; i < 4; ++i) x[k][i] = Cvt<T>::to_f(e[i]);
                                }
                            } else {
#pragma unroll
                                for (int i = 0; i < 4; ++i) x[k][i] = Cvt<T>::to_f(q[d + i]);
                            }
                        }
#pragma unroll
                        for (int i = 0; i < 4; ++i) amax = fmaxf(amax, fabsf(x[k][i]));
                    }
                    if constexpr (!std::is_same<T, __half>::value) {   // 2^-e with the row's maximum in [2^e, 2^(e + 1))
                        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
                        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
                        const uint32_t e = min(max(__float_as_uint(amax) >> 23, 1u), 253u);
                        scale = __uint_as_float((254u - e) << 23);
                        back = __uint_as_float(e << 23);
                    }
#pragma unroll
                    for (int k = 0; k < CH; ++k) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) x[k][i] *= scale;
                        qf[k][half] = pack_f16(x[k][0], x[k][1]);
                        qf[k][half + 2] = pack_f16(x[k][2], x[k][3]);
                        if constexpr (SPLIT) {
                            ql[k][half] = pack_rest(x[k][0], x[k][1], qf[k][half]);
                            ql[k][half + 2] = pack_rest(x[k][2], x[k][3], qf[k][half + 2]);
                        }
                    }
                    (half ? rs1 : rs0) = back * (a.softmax_scale * kLog2e);
                }
            }
            const bool ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&bars[ring]), phase, give_up) ? 1 : 0) != 0;
            if (!ok) break;
            const uint32_t stage = ring0 + static_cast<uint32_t>(ring) * p.stage_bytes;
            for (int ts = 0; ts < p.ts; ++ts) {
                const int tile = ts * p.tw + tok;
                const float4 mt = meta[ring * p.items + tile * p.hw + hl];
                const int valid = static_cast<int>(mt.z);
                if (valid == 0) continue;
                const uint32_t kt = stage + static_cast<uint32_t>(tile) * NH * box_bytes + static_cast<uint32_t>(hl) * HEAD_TILE;
                const uint32_t vt = kt + v_off;
                // ---- S = Q Kc^T: tokens 0-7 and 8-15 ----
                float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < CH; k += 4) {
                    const int cc = (k % (RB / 16)) + (lane >> 3);
                    const uint32_t at = kt + (k * 16 / RB) * box_bytes + krow * RB + ((cc ^ ksw) << 4);
                    uint32_t b[4], d[4];
                    ldmatrix4(at, b);
                    ldmatrix4(at + 8 * RB, d);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t lo, hi;
                        codes_to_f16<E4M3>(b[i], lo, hi);
                        mma_f16(s0, qf[k + i], lo, hi);
                        if constexpr (SPLIT) mma_f16(s0, ql[k + i], lo, hi);
                        codes_to_f16<E4M3>(d[i], lo, hi);
                        mma_f16(s1, qf[k + i], lo, hi);
                        if constexpr (SPLIT) mma_f16(s1, ql[k + i], lo, hi);
                    }
                }
                // ---- weights against the tile's own maximum ----
                // s0[0], s0[1]: row r0, tokens 2c, 2c + 1; s0[2], s0[3]: row r1; s1: the tokens eight further
                float f0 = mt.x * rs0, f1 = mt.x * rs1;
                const int pos = step * p.tt + tile * kTile;
                const bool whole = valid == kTile && pos + kTile <= lim_min;
                if (!whole) {
                    const int n0 = min(valid, lim0 - pos), n1 = min(valid, lim1 - pos);
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        s0[i] = 2 * c + i < n0 ? s0[i] * f0 : -INFINITY;
                        s1[i] = 2 * c + i + 8 < n0 ? s1[i] * f0 : -INFINITY;
                        s0[i + 2] = 2 * c + i < n1 ? s0[i + 2] * f1 : -INFINITY;
                        s1[i + 2] = 2 * c + i + 8 < n1 ? s1[i + 2] * f1 : -INFINITY;
                    }
                    f0 = f1 = 1.f;
                }
                float m0 = fmaxf(fmaxf(s0[0], s0[1]), fmaxf(s1[0], s1[1]));
                float m1 = fmaxf(fmaxf(s0[2], s0[3]), fmaxf(s1[2], s1[3]));
                m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, 1));
                m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, 1));
                m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, 2));
                m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, 2));
                m0 = fmaxf(fmaf(m0, f0, -15.f), -1e30f);   // a row that sees nothing of the tile: every weight 2^-inf
                m1 = fmaxf(fmaf(m1, f1, -15.f), -1e30f);
                float p0[4], p1[4];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    p0[i] = ex2_fast(fmaf(s0[i], f0, -m0));
                    p1[i] = ex2_fast(fmaf(s1[i], f0, -m0));
                    p0[i + 2] = ex2_fast(fmaf(s0[i + 2], f1, -m1));
                    p1[i + 2] = ex2_fast(fmaf(s1[i + 2], f1, -m1));
                }
                if (__any_sync(0xffffffffu, m0 > ref0 + 40.f || m1 > ref1 + 40.f)) {
                    const float n0 = fmaxf(ref0, m0), n1 = fmaxf(ref1, m1);
                    const float a0 = ex2_fast(ref0 - n0), a1 = ex2_fast(ref1 - n1);
                    ref0 = n0;
                    ref1 = n1;
                    l0 *= a0;
                    l1 *= a1;
#pragma unroll
                    for (int j = 0; j < DN; ++j) {
                        o[j][0] *= a0;
                        o[j][1] *= a0;
                        o[j][2] *= a1;
                        o[j][3] *= a1;
                    }
                }
                const float w0 = ex2_fast(m0 - ref0), w1 = ex2_fast(m1 - ref1);
                l0 = fmaf((p0[0] + p0[1]) + (p1[0] + p1[1]), w0, l0);
                l1 = fmaf((p0[2] + p0[3]) + (p1[2] + p1[3]), w1, l1);
                const float g0 = w0 * mt.y, g1 = w1 * mt.y;
                uint32_t pa[4], pl[4];
                pa[0] = pack_f16(p0[0], p0[1]);
                pa[1] = pack_f16(p0[2], p0[3]);
                pa[2] = pack_f16(p1[0], p1[1]);
                pa[3] = pack_f16(p1[2], p1[3]);
                if constexpr (SPLIT) {
                    pl[0] = pack_rest(p0[0], p0[1], pa[0]);
                    pl[1] = pack_rest(p0[2], p0[3], pa[1]);
                    pl[2] = pack_rest(p1[0], p1[1], pa[2]);
                    pl[3] = pack_rest(p1[2], p1[3], pa[3]);
                }
                // ---- O += (w vs) (P Vc) ----
                // Codes of tokens that do not exist are whatever the block holds, NaN perhaps: their weight is 0, so are they.
                uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;
                if (valid < kTile) {
                    keep0 = (2 * c < valid ? 0x00ff00ffu : 0u) | (2 * c + 1 < valid ? 0xff00ff00u : 0u);
                    keep1 = (2 * c + 8 < valid ? 0x00ff00ffu : 0u) | (2 * c + 9 < valid ? 0xff00ff00u : 0u);
                }
#pragma unroll
                for (int h = 0; h < NH; ++h) {
                    uint32_t v[4][VB / 4];   // tokens 2c, 2c + 1, 2c + 8, 2c + 9
                    const uint32_t vb = vt + h * box_bytes + v_lane;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t trow = (i & 1) * RB + (i >> 1) * 8 * RB;
                        if constexpr (RB == 128) {
                            const uint32_t at = vb + trow + ((g ^ (2 * c + (i & 1))) << 4);
                            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v[i][0]), "=r"(v[i][1]), "=r"(v[i][2]), "=r"(v[i][3]) : "r"(at) : "memory");
                        } else {
                            const uint32_t at = vb + trow + (((g >> 1) ^ c) << 4) + (g & 1) * 8;
                            asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v[i][0]), "=r"(v[i][1]) : "r"(at) : "memory");
                        }
                    }
#pragma unroll
                    for (int w = 0; w < VB / 4; ++w) {
                        uint32_t b0[4], b1[4];
                        codes_to_f16<E4M3>(__byte_perm(v[0][w], v[1][w], 0x5140) & keep0, b0[0], b0[1]);
                        codes_to_f16<E4M3>(__byte_perm(v[0][w], v[1][w], 0x7362) & keep0, b0[2], b0[3]);
                        codes_to_f16<E4M3>(__byte_perm(v[2][w], v[3][w], 0x5140) & keep1, b1[0], b1[1]);
                        codes_to_f16<E4M3>(__byte_perm(v[2][w], v[3][w], 0x7362) & keep1, b1[2], b1[3]);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            float (&oj)[4] = o[h * VB + w * 4 + i];
                            float tmp[4] = {0.f, 0.f, 0.f, 0.f};
                            mma_f16(tmp, pa, b0[i], b1[i]);
                            if constexpr (SPLIT) mma_f16(tmp, pl, b0[i], b1[i]);
                            oj[0] = fmaf(tmp[0], g0, oj[0]);
                            oj[1] = fmaf(tmp[1], g0, oj[1]);
                            oj[2] = fmaf(tmp[2], g1, oj[2]);
                            oj[3] = fmaf(tmp[3], g1, oj[3]);
                        }
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&bars[p.nstages + ring]));
            if (++ring == p.nstages) {
                ring = 0;
                phase ^= 1u;
            }
            if (!last) continue;

            // ---- the request's part in this CTA is done ----
            l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
            l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
            l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
            l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
            bool fine = true;
            // The warps of the same head and rows but other token tiles: the upper half hands its state over, until one is left.
            constexpr int STATE = 4 * DN + 4;
            for (int half = p.tw >> 1; half > 0 && fine; half >>= 1) {
                float* box = red + static_cast<size_t>(((tok & (half - 1)) * p.mt + mtile) * p.hw + hl) * (STATE * 32) + lane;
                if (tok >= half && tok < 2 * half) {
#pragma unroll
                    for (int j = 0; j < DN; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) box[(4 * j + e) * 32] = o[j][e];
                    box[(4 * DN) * 32] = ref0;
                    box[(4 * DN + 1) * 32] = ref1;
                    box[(4 * DN + 2) * 32] = l0;
                    box[(4 * DN + 3) * 32] = l1;
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&bars[2 * p.nstages]));
                fine = __all_sync(0xffffffffu, mbar_wait(smem_u32(&bars[2 * p.nstages]), merge_phase, give_up) ? 1 : 0) != 0;
                if (!fine) break;
                if (tok < half) {
                    const float u0 = box[(4 * DN) * 32], u1 = box[(4 * DN + 1) * 32];
                    const float n0 = fmaxf(fmaxf(ref0, u0), -1e30f), n1 = fmaxf(fmaxf(ref1, u1), -1e30f);
                    const float a0 = ex2_fast(ref0 - n0), a1 = ex2_fast(ref1 - n1), b0 = ex2_fast(u0 - n0), b1 = ex2_fast(u1 - n1);
                    ref0 = n0;
                    ref1 = n1;
                    l0 = fmaf(l0, a0, box[(4 * DN + 2) * 32] * b0);
                    l1 = fmaf(l1, a1, box[(4 * DN + 3) * 32] * b1);
#pragma unroll
                    for (int j = 0; j < DN; ++j) {
                        o[j][0] = fmaf(o[j][0], a0, box[(4 * j) * 32] * b0);
                        o[j][1] = fmaf(o[j][1], a0, box[(4 * j + 1) * 32] * b0);
                        o[j][2] = fmaf(o[j][2], a1, box[(4 * j + 2) * 32] * b1);
                        o[j][3] = fmaf(o[j][3], a1, box[(4 * j + 3) * 32] * b1);
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&bars[2 * p.nstages + 1]));
                fine = __all_sync(0xffffffffu, mbar_wait(smem_u32(&bars[2 * p.nstages + 1]), merge_phase, give_up) ? 1 : 0) != 0;
                merge_phase ^= 1u;
            }
            if (!fine) break;
            if (tok > 0) continue;
            // A request that this CTA has seen from its first step to its last one is finished here.
            const bool alone = part_first == 0 && step + 1 == pre[req + 1] - pre[req];
            const int64_t part = (static_cast<int64_t>(cta) + req) * a.n * a.Hq;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int r = half ? r1 : r0;
                if (r >= R) continue;
                const int64_t row = half ? row1 : row0;
                const float l = half ? l1 : l0;
                if (alone) {
                    const float inv = l == 0.f ? 0.f : 1.f / l;
                    const int tq = half ? tq1 : tq0;
                    T* out = static_cast<T*>(a.out) + static_cast<int64_t>(req) * a.o_s0 + static_cast<int64_t>(tq) * a.o_s1 +
                             static_cast<int64_t>(hkv * group + (r - tq * group)) * a.o_s2;
                    const bool vec = aligned16(out);
#pragma unroll
                    for (int h = 0; h < NH; ++h)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int d = h * RB + (2 * c + e) * VB;
                            if (d >= a.D) continue;
                            constexpr int VN = Vec16<T>::N;
#pragma unroll
                            for (int j = 0; j < VB; j += VN) {
                                float f[VN];
#pragma unroll
                                for (int i = 0; i < VN; ++i) f[i] = o[h * VB + j + i][2 * half + e] * inv;
                                if (vec) {
                                    *reinterpret_cast<uint4*>(out + d + j) = pack16<T>(f);
                                } else {
#pragma unroll
                                    for (int i = 0; i < VN; ++i) out[d + j + i] = Cvt<T>::from_f(f[i]);
                                }
                            }
                        }
                } else {
                    float* acc = ws_acc + (part + row) * a.D;
#pragma unroll
                    for (int h = 0; h < NH; ++h)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int d = h * RB + (2 * c + e) * VB;
                            if (d >= a.D) continue;
#pragma unroll
                            for (int j = 0; j < VB; j += 4)
                                *reinterpret_cast<float4*>(acc + d + j) = make_float4(o[h * VB + j][2 * half + e], o[h * VB + j + 1][2 * half + e],
                                                                                      o[h * VB + j + 2][2 * half + e], o[h * VB + j + 3][2 * half + e]);
                        }
                    if (c == 0) *reinterpret_cast<float2*>(ws_ml + (part + row) * 2) = make_float2(half ? ref1 : ref0, l);
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

// Merges the parts of a request that several CTAs had, and writes zeros for an empty one. One warp to a query row.
template <typename T>
__global__ void __launch_bounds__(128) quant_combine_kernel(const QuantAttnArgs a, int tt, int n_cta, const float* __restrict__ ws_acc,
                                                            const float* __restrict__ ws_ml) {
    __shared__ int s_part[4][2];
    const int i = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int before = 0, all = 0;
    for (int r = threadIdx.x; r < a.B; r += blockDim.x) {
        const int n = (quant_len(a, r) + tt - 1) / tt;
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
    before = s_part[0][0] + s_part[1][0] + s_part[2][0] + s_part[3][0];
    all = s_part[0][1] + s_part[1][1] + s_part[2][1] + s_part[3][1];
    const int steps = (quant_len(a, i) + tt - 1) / tt;
    const int used = used_ctas(all, n_cta);
    // CTA c has the steps [all * c / used, all * (c + 1) / used): every one of the used CTAs has some.
    int c_first = 0, c_last = -1;
    if (steps > 0) {
        auto cta_of = [&](int t) {
            const int64_t c = ((static_cast<int64_t>(t) + 1) * used - 1) / all;
            return static_cast<int>(c < used - 1 ? c : used - 1);
        };
        c_first = cta_of(before);
        c_last = cta_of(before + steps - 1);
        if (c_first == c_last) return;   // written by that CTA
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int row = blockIdx.y * 4 + warp;
    if (row >= a.n * a.Hq) return;
    constexpr int RG = 8;   // head_dim <= 256
    float acc[RG];
#pragma unroll
    for (int r = 0; r < RG; ++r) acc[r] = 0.f;
    const int64_t rows = static_cast<int64_t>(a.n) * a.Hq;
    float M = -INFINITY, L = 0.f;
    for (int c = c_first; c <= c_last; ++c) M = fmaxf(M, ws_ml[((static_cast<int64_t>(c) + i) * rows + row) * 2]);
    M = fmaxf(M, -1e30f);
    for (int c = c_first; c <= c_last; ++c) {
        const int64_t at = (static_cast<int64_t>(c) + i) * rows + row;
        const float2 ml = *reinterpret_cast<const float2*>(ws_ml + at * 2);
        const float w = exp2f(ml.x - M);
        L = fmaf(ml.y, w, L);
#pragma unroll
        for (int r = 0; r < RG; ++r) {
            const int d = lane + 32 * r;
            if (d < a.D) acc[r] = fmaf(ws_acc[at * a.D + d], w, acc[r]);
        }
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    const int t = row / a.Hq, h = row - t * a.Hq;
    T* out = static_cast<T*>(a.out) + static_cast<int64_t>(i) * a.o_s0 + static_cast<int64_t>(t) * a.o_s1 + static_cast<int64_t>(h) * a.o_s2;
#pragma unroll
    for (int r = 0; r < RG; ++r) {
        const int d = lane + 32 * r;
        if (d < a.D) out[d] = Cvt<T>::from_f(acc[r] * inv);
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

// [head_dim, position, head, block] of one cache whatever its strides; a box is 16 positions of hw heads. Bytes of a row
// beyond head_dim arrive as zeros.
bool encode_map(const QuantAttnArgs& a, const QuantPlan& p, int m, CUtensorMap* map) {
    EncodeFn fn = encode_fn();
    if (!fn) return false;
    const int rb = p.hd < 128 ? p.hd : 128;
    auto stride = [](int64_t s, int64_t extent) { return static_cast<cuuint64_t>(extent > 1 ? s : 16); };
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(a.D), static_cast<cuuint64_t>(a.block_size), static_cast<cuuint64_t>(a.Hkv), static_cast<cuuint64_t>(a.blocks)};
    const cuuint64_t strides[3] = {stride(a.c_s1[m], a.block_size), stride(a.c_s2[m], a.Hkv), stride(a.c_s0[m], a.blocks)};
    const cuuint32_t box[4] = {static_cast<cuuint32_t>(rb), kTile, static_cast<cuuint32_t>(p.hw), 1};
    const cuuint32_t ones[4] = {1, 1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(a.cache[m]), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
              rb == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Whether the split kernel takes these arguments, and how it cuts them.
bool make_quant_plan(const QuantAttnArgs& a, int sm_count, int max_smem, QuantPlan& p) {
    if (a.force_plain || a.D % 16 != 0 || a.block_size % kTile != 0 || a.blocks <= 0 || a.cols <= 0) return false;
    // head_dim 256 in fp32 would need 128 registers of query fragments beside 128 of accumulators
    if (a.D > 256 || (a.dt == Dt::F32 && a.D > 128)) return false;
    if (a.B > kQMaxB || static_cast<int64_t>(a.B) * a.cols * a.block_size / kTile >= (1ll << 30) || a.blocks >= (1ll << 31)) return false;
    for (int m = 0; m < 2; ++m) {
        auto ok = [](int64_t s, int64_t extent) { return extent <= 1 || (s > 0 && s % 16 == 0 && s < (1ll << 40)); };
        if (a.c_s3[m] != 1 || !ok(a.c_s0[m], a.blocks) || !ok(a.c_s1[m], a.block_size) || !ok(a.c_s2[m], a.Hkv) ||
            reinterpret_cast<uintptr_t>(a.cache[m]) % 16 != 0)
            return false;
    }
    p = QuantPlan{};
    p.hd = a.D <= 64 ? 64 : a.D <= 128 ? 128 : 256;
    const int R = a.n * (a.Hq / a.Hkv);
    p.mt = 1;
    while (p.mt < kQWarps && p.mt * 16 < R) p.mt *= 2;
    p.n_z = (R + p.mt * 16 - 1) / (p.mt * 16);
    p.hw = 1;
    for (int h = 2; h <= kQWarps / p.mt; ++h)
        if (a.Hkv % h == 0) p.hw = h;
    p.n_hg = a.Hkv / p.hw;
    p.tw = 1;
    while (p.hw * p.mt * p.tw * 2 <= kQWarps) p.tw *= 2;
    // A step of about 32 KB: enough bytes to pay for its hand-over, and still six of them in flight.
    const int pair = 2 * kTile * p.hd;   // K and V of a tile
    p.ts = 1;
    while (p.hw * p.tw * p.ts * 2 * pair <= 32768 && p.hw * p.tw * p.ts * 2 <= 16) p.ts *= 2;
    p.tt = kTile * p.tw * p.ts;
    p.items = p.hw * p.tw * p.ts;
    p.stage_bytes = p.items * pair;
    const int state = (4 * (p.hd / 8) + 4) * 32 * 4;
    const int red_bytes = p.tw > 1 ? p.tw / 2 * p.mt * p.hw * state : 0;
    const int fixed = 1024 + kQMaxStages * p.items * 16 + (2 * kQMaxStages + 2) * 8 + (2 * a.B + 1) * 4 + red_bytes + 64;
    p.nstages = std::min((max_smem - fixed) / p.stage_bytes, kQMaxStages);
    if (p.nstages < 2) return false;
    int off = p.nstages * p.stage_bytes;
    auto take = [&](int bytes) {
        const int at = off;
        off += (bytes + 15) / 16 * 16;
        return at;
    };
    p.off_meta = take(p.nstages * p.items * 16);
    p.off_bars = take((2 * p.nstages + 2) * 8);
    p.off_red = take(red_bytes);
    p.off_pre = take((a.B + 1) * 4);
    p.off_len = take(a.B * 4);
    p.off_flag = take(4);
    p.smem_bytes = off + 1024;
    if (p.smem_bytes > max_smem) return false;
    const int64_t most = static_cast<int64_t>(a.B) * ((static_cast<int64_t>(a.cols) * a.block_size + p.tt - 1) / p.tt);
    p.n_cta = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(sm_count / (p.n_hg * p.n_z), (most + kStepsPerCta - 1) / kStepsPerCta)));
    const int64_t el = a.dt == Dt::F32 ? 4 : 2;
    p.qvec = reinterpret_cast<uintptr_t>(a.q) % (4 * el) == 0 && a.q_s0 % 4 == 0 && a.q_s1 % 4 == 0 && a.q_s2 % 4 == 0;
    return true;
}

int64_t part_rows(const QuantAttnArgs& a, const QuantPlan& p) { return (static_cast<int64_t>(p.n_cta) + a.B) * a.n * a.Hq; }

template <typename T, bool E4M3, int HD>
void launch_split(const QuantAttnArgs& a, const QuantPlan& p, const CUtensorMap& mk, const CUtensorMap& mv, float* acc, float* ml, cudaStream_t st) {
    auto kern = quant_split_kernel<T, E4M3, HD>;
    cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, p.smem_bytes);
    kern<<<dim3(p.n_cta, p.n_hg, p.n_z), kQThreads, p.smem_bytes, st>>>(a, p, mk, mv, acc, ml);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.B, (a.n * a.Hq + 3) / 4, 1);
    cfg.blockDim = dim3(128);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, quant_combine_kernel<T>, a, p.tt, p.n_cta, static_cast<const float*>(acc), static_cast<const float*>(ml));
}

template <typename T>
void launch_split_t(const QuantAttnArgs& a, const QuantPlan& p, const CUtensorMap& mk, const CUtensorMap& mv, float* acc, float* ml, cudaStream_t st) {
    if (p.hd == 64) {
        a.e4m3 ? launch_split<T, true, 64>(a, p, mk, mv, acc, ml, st) : launch_split<T, false, 64>(a, p, mk, mv, acc, ml, st);
    } else if (p.hd == 128) {
        a.e4m3 ? launch_split<T, true, 128>(a, p, mk, mv, acc, ml, st) : launch_split<T, false, 128>(a, p, mk, mv, acc, ml, st);
    } else if constexpr (!std::is_same<T, float>::value) {
        a.e4m3 ? launch_split<T, true, 256>(a, p, mk, mv, acc, ml, st) : launch_split<T, false, 256>(a, p, mk, mv, acc, ml, st);
    }
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
            launch_split_t<__half>(a, p, mk, mv, acc, ml, st);
        else if (a.dt == Dt::BF16)
            launch_split_t<__nv_bfloat16>(a, p, mk, mv, acc, ml, st);
        else
            launch_split_t<float>(a, p, mk, mv, acc, ml, st);
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
