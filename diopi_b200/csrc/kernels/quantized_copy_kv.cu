// New K and V rows into a paged cache of 8-bit codes with one scale for each (block, head) (diopiQuantizedCopyKV).
//
// A block whose first position is written by the call begins anew: with amax the largest magnitude of the call's rows in it
//     int8:  s = max(amax * fp32(1 / 127), 2^-126)         e4m3:  s = 2^k, the smallest k >= -126 with amax <= 448 * 2^k
// (s = 0 when amax = 0). A block that an earlier call began keeps its tokens: its scale becomes s' = s * 2^k with the
// smallest k >= 0 that covers the new rows, and the codes in front of them become rne(code * 2^-k). Growth by powers of two
// keeps that exact where the format can hold the result, so that a block filled token by token does not drift. A new code is
// the correctly rounded quotient x / s, ties to even; all of it is a function of the values alone, so that any order of
// the work gives the same bits. NaN and infinities do not count into amax: they saturate (int8 NaN: 0, e4m3 NaN: NaN).
//
// Bytes: T * H * D * (e + 1) for each of K and V. One pass: the rows of a block stay in registers between the maximum and
// the codes. A unit is one (request, block, head) of one matrix; 16 (8) rows of it belong to a warp, with 16 elements of a row to
// a lane, and up to 8 warps share a unit through shared memory. Blocks of more rows than that are read twice (the second time from
// L1/L2). Bound by memory latency over 24 warps an SM, then by its rate: 36864 tokens x 32 heads x 128, fp16 to int8: 165 us =
// 5500 GB/s = 0.84 of the copy rate; 124971 tokens x 8 heads, fp16 to e4m3: 128 us, 0.92. With fewer than 8 heads some warps of a
// CTA have none (4 heads 99 us, 2: 91, 1: 86). On the way there: vectors side by side in a lane instead of whole lines, 394 us;
// calls for the rare cases inside the loop, 231; the element-wise rows inside the loop, 171. Up to 40 bytes a thread are still
// spilled at 80 and 64 registers (head_dim to 128); more registers leave an SM fewer CTAs.
#include <cuda_fp8.h>

#include <type_traits>

#include "dev_util.cuh"

namespace b200 {
namespace k {
namespace {

constexpr int kCopyThreads = 256;
constexpr int kCopyWarps = kCopyThreads / 32;
constexpr float kFltMin = 1.17549435e-38f;   // 2^-126

// The scale of a block that begins anew.
__device__ __forceinline__ float fresh_scale(float amax, bool e4m3) {
    if (!(amax > 0.f)) return 0.f;
    if (!e4m3) return fmaxf(__fmul_rn(amax, 1.f / 127.f), kFltMin);
    const uint32_t u = __float_as_uint(amax);
    const int e = static_cast<int>(u >> 23);                       // biased; 0 for subnormals
    int k = e - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);         // 448 = 1.75 * 2^8
    k = e == 0 ? 1 : max(k, 1);                                    // 2^-126 at least
    return __uint_as_float(static_cast<uint32_t>(k) << 23);
}

// Smallest k >= 0 with old * 2^k >= need. The quotient of two fp32 values is further from any power of two than the
// rounding of a double, unless it is one.
__device__ __forceinline__ int growth_steps(float old, float need) {
    if (!(need > old)) return 0;
    const double r = static_cast<double>(need) / static_cast<double>(old);
    const int hi = __double2hiint(r), lo = __double2loint(r);
    return ((hi >> 20) & 0x7ff) - 1023 + (((hi & 0xfffff) | lo) != 0 ? 1 : 0);
}

__device__ __forceinline__ float pow2f(int k) { return k < -149 ? 0.f : exp2f(static_cast<float>(k)); }

// One value, any input: the definition itself in double (a quotient of two fp32 values is never close enough to a tie of
// an 8-bit format, without being one, for the rounding to double to matter; a rounding to fp32 between the two would).
template <bool E4M3>
__device__ __noinline__ uint32_t encode_slow(float x, float s) {
    if (E4M3) {
        if (isnan(x)) return 0x7fu;
        if (s == 0.f) return 0u;
        const double q = static_cast<double>(x) / static_cast<double>(s);
        const float y = __double2float_rz(q);   // to odd: the code's rounding then sees all of q
        return __nv_cvt_float_to_fp8(__uint_as_float(__float_as_uint(y) | (static_cast<double>(y) != q ? 1u : 0u)), __NV_SATFINITE, __NV_E4M3);
    }
    if (isnan(x) || s == 0.f) return 0u;
    double y = rint(static_cast<double>(x) / static_cast<double>(s));
    y = y > 127. ? 127. : (y < -127. ? -127. : y);
    return static_cast<uint32_t>(static_cast<int>(y)) & 0xffu;
}

__device__ __forceinline__ uint32_t e4m3_pair(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

// Four codes. e4m3: s is a power of two here, hence 1 / s, so x * lo is exact (hi is not used). int8: adding 1.5 * 2^23 rounds x * inv to an
// integer, which sits in the low byte. `lo` and `hi` hold 1 / s between them (the approximate reciprocal is off by one unit
// in the last place at most), so where both give one code the quotient has it; `split` collects the bits in which they differ.
struct Inverse {
    float lo, hi;
};
template <bool E4M3>
__device__ __forceinline__ Inverse inverse_of(float s) {
    Inverse v;
    if constexpr (E4M3) {
        v.lo = v.hi = s > 0.f ? __uint_as_float(0x7f000000u - __float_as_uint(s)) : 0.f;   // 2^-k of 2^k
    } else {
        float r;
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
        v.lo = s > 0.f ? __uint_as_float(__float_as_uint(r) - 2) : 0.f;
        v.hi = s > 0.f ? __uint_as_float(__float_as_uint(r) + 2) : 0.f;
    }
    return v;
}
constexpr float kMagic = 12582912.f;
template <bool E4M3>
__device__ __forceinline__ uint32_t encode4(const float* x, Inverse inv, uint32_t& split) {
    if constexpr (E4M3) {
        return e4m3_pair(x[0] * inv.lo, x[1] * inv.lo) | (e4m3_pair(x[2] * inv.lo, x[3] * inv.lo) << 16);
    } else {
        uint32_t b[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            b[i] = __float_as_uint(fmaf(x[i], inv.lo, kMagic));
            split |= b[i] ^ __float_as_uint(fmaf(x[i], inv.hi, kMagic));
        }
        return __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    }
}
// The nearest integer to x / s, ties to even, for finite |x / s| <= 127.5: the remainder of a candidate that is off by one at
// most is exact in one fma.
__device__ __forceinline__ uint32_t encode_near(float x, float s, float inv) {
    float q = fmaf(x, inv, kMagic) - kMagic;
    const float r = fmaf(-q, s, x), two = 2.f * fabsf(r);
    if (two > s || (two == s && (static_cast<int>(q) & 1))) q += r > 0.f ? 1.f : -1.f;
    return static_cast<uint32_t>(static_cast<int>(q)) & 0xffu;
}

// A code in a scale that has grown by 2^k; f = 2^-k.
__device__ __forceinline__ uint32_t shrink_code(uint32_t c, float f, bool e4m3) {
    if (e4m3) {
        __half_raw h = __nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(c), __NV_E4M3);
        return __nv_cvt_float_to_fp8(__half2float(__half(h)) * f, __NV_SATFINITE, __NV_E4M3);
    }
    return static_cast<uint32_t>(static_cast<int>(rintf(static_cast<float>(static_cast<int8_t>(c)) * f))) & 0xffu;
}

struct CopyUnit {
    int64_t row0;        // first row of the call in this block
    int64_t block;       // block id, -1: nothing to do
    int p0, p1;          // positions written
};

// Finds unit u of the batch: the requests' touched blocks, one after the other. All threads of the CTA take part.
__device__ __forceinline__ CopyUnit find_unit(const QuantCopyArgs& a, int u) {
    __shared__ int warp_sum[kCopyWarps];
    __shared__ int s_req, s_j;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t cap = static_cast<int64_t>(a.cols) * a.block_size;
    if (tid == 0) s_req = -1;
    int carry = 0;
    CopyUnit un{0, -1, 0, 0};
    for (int base = 0; base < a.B; base += kCopyThreads) {
        const int r = base + tid;
        int cnt = 0;
        if (r < a.B) {
            const int64_t c = load_index(a.cached, r);
            const int64_t n = imin64(load_index(a.new_start, r + 1), a.T) - load_index(a.new_start, r);
            if (u == 0 && n > 0 && (c < 0 || n > cap - c)) report_status(a.status, 1);   // the tokens that the table has no column for
            if (n > 0 && c >= 0 && c < cap) cnt = static_cast<int>((c % a.block_size + imin64(n, cap - c) + a.block_size - 1) / a.block_size);
        }
        int v = cnt;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int w = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += w;
        }
        if (lane == 31) warp_sum[warp] = v;
        __syncthreads();
        int total = 0, below = 0;
#pragma unroll
        for (int w = 0; w < kCopyWarps; ++w) {
            below += w < warp ? warp_sum[w] : 0;
            total += warp_sum[w];
        }
        const int first = carry + below + v - cnt;
        if (u >= first && u < first + cnt) {
            s_req = r;
            s_j = u - first;
        }
        carry += total;
        __syncthreads();
        if (u > 0 && u < carry) break;
    }
    __syncthreads();
    const int req = s_req;
    if (req < 0) return un;
    const int j = s_j;
    const int64_t c = load_index(a.cached, req), t0 = load_index(a.new_start, req);
    const int64_t n = imin64(imin64(load_index(a.new_start, req + 1), a.T) - t0, cap - c);
    const int64_t b = c / a.block_size + j, lo = imax64(c, b * a.block_size), hi = imin64(c + n, (b + 1) * a.block_size);
    const int64_t id = load_index(a.table, req, b);
    if (id < 0 || id >= a.blocks || t0 < 0) {
        if (tid == 0) report_status(a.status, 1);
        return un;
    }
    un.row0 = t0 + (lo - c);
    un.block = id;
    un.p0 = static_cast<int>(lo - b * a.block_size);
    un.p1 = static_cast<int>(hi - b * a.block_size);
    return un;
}

// The bits of the largest magnitude of a 16-byte vector as fp32: above those of infinity if there is a NaN, equal if there is
// an infinity.
template <typename T>
__device__ __forceinline__ uint32_t top_of(const uint4& v) {
    if constexpr (sizeof(T) == 2) {
        using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
        const T2* w = reinterpret_cast<const T2*>(&v);
        const T2 u = __hmax2_nan(__hmax2_nan(__habs2(w[0]), __habs2(w[1])), __hmax2_nan(__habs2(w[2]), __habs2(w[3])));
        return __float_as_uint(Cvt<T>::to_f(__hmax_nan(u.x, u.y))) & 0x7fffffffu;
    } else {
        return max(max(v.x & 0x7fffffffu, v.y & 0x7fffffffu), max(v.z & 0x7fffffffu, v.w & 0x7fffffffu));
    }
}
template <typename T>
__device__ __forceinline__ float finite_top_of(const uint4& v) {
    float f[Vec16<T>::N], m = 0.f;
    unpack16<T>(v, f);
#pragma unroll
    for (int j = 0; j < Vec16<T>::N; ++j) m = fmaxf(m, isfinite(f[j]) ? fabsf(f[j]) : 0.f);
    return m;
}

constexpr uint32_t kInfBits = 0x7f800000u;

// Rows of a warp: 16, or 8 where 16 of them would take 64 registers of every lane in fp32 (19 requests of up to 517 tokens, 5
// heads x 80: 12.7 us; 13.7 with 16).
template <typename T>
constexpr int warp_rows(int lpr) { return sizeof(T) == 4 && lpr >= 8 ? 8 : 16; }
// CTAs of an SM that the registers are to leave room for: the rows are held between the two passes.
template <typename T>
constexpr int copy_ctas(int lpr) {
    const int held = warp_rows<T>(lpr) * lpr / 32 * 4 * static_cast<int>(sizeof(T));   // registers of a lane
    return held <= 16 ? 4 : held <= 32 ? 3 : held <= 64 ? 2 : 1;
}

// One row of a unit that encode4 is not for (a NaN or an infinity in it, a scale of another kind); the lanes of a row share it.
template <typename T, bool E4M3>
__device__ __noinline__ void encode_row_slow(const T* x, uint8_t* to, int D, int first, int step, float s) {
    for (int d = first; d < D; d += step) to[d] = static_cast<uint8_t>(encode_slow<E4M3>(Cvt<T>::to_f(x[d]), s));
}

// What earlier calls left in a block, in a scale grown by 2^steps: rows p, p + by, ... below p0, 16 codes of each.
template <bool E4M3>
__device__ __noinline__ void shrink_rows(uint8_t* dst, int64_t pitch, int p, int p0, int by, int steps) {
    const float f = pow2f(-steps);
    for (; p < p0; p += by) {
        uint4* at = reinterpret_cast<uint4*>(dst + static_cast<int64_t>(p) * pitch);
        uint4 v = *at;
        uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            uint32_t o = 0;
#pragma unroll
            for (int b = 0; b < 4; ++b) o |= shrink_code((w[e] >> (8 * b)) & 0xffu, f, E4M3) << (8 * b);
            w[e] = o;
        }
        *at = v;
    }
}

// Lanes of a row LPR, with 16 elements each: vectors of 16 bytes, LPR lanes apart, so that a load covers whole lines (where the
// row is shorter some vectors are left out). W warps to a unit.
template <typename T, bool E4M3, int LPR, int W, bool REREAD>
__global__ void __launch_bounds__(kCopyThreads, copy_ctas<T>(LPR)) quantized_copy_kernel(const QuantCopyArgs a) {
    constexpr int E = Vec16<T>::N;             // elements of a vector
    constexpr int N = 16 / E;                  // vectors of a lane's row
    constexpr int RPP = 32 / LPR;              // rows of a warp's pass
    constexpr int kWarpRows = warp_rows<T>(LPR);
    constexpr int PASSES = kWarpRows / RPP;
    constexpr int UPC = kCopyWarps / W;        // heads of a CTA
    __shared__ uint32_t s_top[2][kCopyWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const CopyUnit un = find_unit(a, blockIdx.x);
    if (un.block < 0) return;                  // the same for the whole CTA
    const int h = blockIdx.y * UPC + warp / W, wu = warp % W;
    const bool here = h < a.H;
    const int rl = lane / LPR, cl = lane % LPR;
    const bool full_width = a.D == 16 * LPR;

    // K and V one after the other, or (two CTAs along z) one of them. (The rows of both asked for before either is stored: 128
    // registers, two CTAs an SM, 220 us on the prompts above when this form took 171.)
#pragma unroll 1
    for (int m = blockIdx.z; m < 2; m += gridDim.z) {
        const int64_t pitch = a.src_s0[m];
        // row of position 0 of this block, in front of the first row when the call does not write it: not read there
        const T* src = static_cast<const T*>(a.src[m]) + (un.row0 - un.p0) * pitch + static_cast<int64_t>(h) * a.src_s1[m];
        uint8_t* dst = static_cast<uint8_t*>(a.cache[m]) + un.block * a.c_s0[m] + static_cast<int64_t>(h) * a.c_s2[m];
        float* scale = a.scale[m] + un.block * a.s_s0[m] + static_cast<int64_t>(h) * a.s_s1[m];

        const int chunks = REREAD ? (un.p1 + W * kWarpRows - 1) / (W * kWarpRows) : 1;
        uint4 r[PASSES][N];
        // The rows of chunk q that belong to the call; a unit whose every row does, at full width, needs no looking.
        auto load_rows = [&](int q) {
            const int p = (q * W + wu) * kWarpRows + rl;
            const T* from = src + p * pitch + cl * E;
            const bool whole = full_width && here && p - rl >= un.p0 && p - rl + kWarpRows <= un.p1;
            if (whole) {
#pragma unroll
                for (int i = 0; i < PASSES; ++i) {
#pragma unroll
                    for (int n = 0; n < N; ++n) r[i][n] = __ldg(reinterpret_cast<const uint4*>(from + n * LPR * E));
                    from += RPP * pitch;
                }
            } else {
#pragma unroll
                for (int i = 0; i < PASSES; ++i) {
                    const bool in = here && p + i * RPP >= un.p0 && p + i * RPP < un.p1;
#pragma unroll
                    for (int n = 0; n < N; ++n)
                        r[i][n] = in && (n * LPR + cl) * E < a.D ? __ldg(reinterpret_cast<const uint4*>(from + n * LPR * E)) : make_uint4(0, 0, 0, 0);
                    from += RPP * pitch;
                }
            }
        };
        const float old = here && un.p0 > 0 ? *scale : 0.f;   // read by every lane before the barrier below, written after it

        uint32_t top = 0;
        for (int q = 0; q < chunks; ++q) {
            load_rows(q);
#pragma unroll
            for (int i = 0; i < PASSES; ++i)
#pragma unroll
                for (int n = 0; n < N; ++n) top = max(top, top_of<T>(r[i][n]));
        }
        auto over_unit = [&](uint32_t x, int buf) {   // the largest of a unit
            x = __reduce_max_sync(0xffffffffu, x);
            if constexpr (W > 1) {
                if (lane == 0) s_top[buf][warp] = x;
                __syncthreads();
#pragma unroll
                for (int w = 0; w < W; ++w) x = max(x, s_top[buf][warp / W * W + w]);
            }
            return x;
        };
        top = over_unit(top, 0);
        const bool odd = top >= kInfBits;   // a NaN or an infinity in the unit: it does not count
        if (W > 1 ? __syncthreads_or(odd) != 0 : odd) {
            uint32_t f = 0;
            for (int q = 0; q < chunks; ++q) {
                if (REREAD) load_rows(q);
#pragma unroll
                for (int i = 0; i < PASSES; ++i)
#pragma unroll
                    for (int n = 0; n < N; ++n) f = max(f, __float_as_uint(finite_top_of<T>(r[i][n])));
            }
            top = over_unit(f, 1);
        }

        float s = fresh_scale(__uint_as_float(top), E4M3);
        if (here && un.p0 > 0 && old > 0.f) {
            const int steps = growth_steps(old, s);
            s = steps > 0 ? static_cast<float>(scalbn(static_cast<double>(old), steps)) : old;
            if (steps > 0 && cl * 16 < a.D) shrink_rows<E4M3>(dst + cl * 16, a.c_s1[m], wu * RPP + rl, un.p0, W * RPP, steps);
        }
        if (here && wu == 0 && lane == 0) *scale = s;

        // Of this file's own scales none: a block that someone else began, with a scale that has no reciprocal among the normal numbers, or
        // that is no power of two where the codes are e4m3.
        const bool by_element = odd || s > 0x1p126f || (E4M3 && (__float_as_uint(s) & 0x7fffffu) != 0);
        if (by_element) {   // the same for the whole unit; apart from the loop below, whose rows would be spilled around the call
            for (int p = un.p0 + wu * RPP + rl; here && p < un.p1; p += W * RPP)
                encode_row_slow<T, E4M3>(src + p * pitch, dst + p * a.c_s1[m], a.D, cl, LPR, s);
        } else {
            const Inverse inv = inverse_of<E4M3>(s);
            const uint32_t nonzero = E4M3 && s == 0.f ? 0u : 0xffffffffu;   // a block of zeros has codes 0: no -0 (0x80) for a -0
            for (int q = 0; q < chunks; ++q) {
                if (REREAD) load_rows(q);
                const int p = (q * W + wu) * kWarpRows + rl;
                uint8_t* to = dst + p * a.c_s1[m] + cl * E;
#pragma unroll
                for (int i = 0; i < PASSES; ++i) {
                    if (here && p + i * RPP >= un.p0 && p + i * RPP < un.p1) {
#pragma unroll
                        for (int n = 0; n < N; ++n) {
                            if (!full_width && (n * LPR + cl) * E >= a.D) continue;
                            float f[E];
                            unpack16<T>(r[i][n], f);
                            uint32_t w[E / 4], split = 0;
#pragma unroll
                            for (int e = 0; e < E / 4; ++e) w[e] = encode4<E4M3>(f + 4 * e, inv, split) & nonzero;
                            if (!E4M3 && split != 0) {
#pragma unroll
                                for (int e = 0; e < E / 4; ++e)
                                    w[e] = encode_near(f[4 * e], s, inv.lo) | (encode_near(f[4 * e + 1], s, inv.lo) << 8) | (encode_near(f[4 * e + 2], s, inv.lo) << 16) |
                                           (encode_near(f[4 * e + 3], s, inv.lo) << 24);
                            }
                            if constexpr (E == 8)
                                *reinterpret_cast<uint2*>(to + n * LPR * E) = make_uint2(w[0], w[1]);
                            else
                                *reinterpret_cast<uint32_t*>(to + n * LPR * E) = w[0];
                        }
                    }
                    to += RPP * a.c_s1[m];
                }
            }
        }
        if constexpr (W > 1) __syncthreads();   // s_top is written again
    }
}

// Any width, strides and alignment: one CTA to a unit, element by element.
template <typename T>
__global__ void __launch_bounds__(kCopyThreads) quantized_copy_any_kernel(const QuantCopyArgs a) {
    __shared__ float s_amax[kCopyWarps];
    const int m = blockIdx.z, h = blockIdx.y, tid = threadIdx.x;
    const CopyUnit un = find_unit(a, blockIdx.x);
    if (un.block < 0) return;
    const T* src = static_cast<const T*>(a.src[m]) + un.row0 * a.src_s0[m] + static_cast<int64_t>(h) * a.src_s1[m];
    uint8_t* dst = static_cast<uint8_t*>(a.cache[m]) + un.block * a.c_s0[m] + static_cast<int64_t>(h) * a.c_s2[m];
    float* scale = a.scale[m] + un.block * a.s_s0[m] + static_cast<int64_t>(h) * a.s_s1[m];
    const float old = un.p0 > 0 ? *scale : 0.f;
    const int64_t n = static_cast<int64_t>(un.p1 - un.p0) * a.D;
    float amax = 0.f;
    for (int64_t i = tid; i < n; i += kCopyThreads) {
        const float x = Cvt<T>::to_f(src[i / a.D * a.src_s0[m] + i % a.D * a.src_s2[m]]);
        amax = fmaxf(amax, isfinite(x) ? fabsf(x) : 0.f);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if ((tid & 31) == 0) s_amax[tid >> 5] = amax;
    __syncthreads();
    for (int w = 0; w < kCopyWarps; ++w) amax = fmaxf(amax, s_amax[w]);
    float s = fresh_scale(amax, a.e4m3);
    if (un.p0 > 0 && old > 0.f) {
        const int steps = growth_steps(old, s);
        s = steps > 0 ? static_cast<float>(scalbn(static_cast<double>(old), steps)) : old;
        if (steps > 0) {
            const float f = pow2f(-steps);
            for (int64_t i = tid; i < static_cast<int64_t>(un.p0) * a.D; i += kCopyThreads) {
                uint8_t* at = dst + i / a.D * a.c_s1[m] + i % a.D * a.c_s3[m];
                *at = static_cast<uint8_t>(shrink_code(*at, f, a.e4m3));
            }
        }
    }
    if (tid == 0) *scale = s;
    for (int64_t i = tid; i < n; i += kCopyThreads) {
        const float x = Cvt<T>::to_f(src[i / a.D * a.src_s0[m] + i % a.D * a.src_s2[m]]);
        dst[(un.p0 + i / a.D) * a.c_s1[m] + i % a.D * a.c_s3[m]] = static_cast<uint8_t>(a.e4m3 ? encode_slow<true>(x, s) : encode_slow<false>(x, s));
    }
}

template <typename T, bool E4M3, int LPR>
void launch_rows(const QuantCopyArgs& a, int units, int sm_count, cudaStream_t st) {
    auto go = [&](auto kern, int w) {
        const int upc = kCopyWarps / w;
        const int y = (a.H + upc - 1) / upc;
        // Few CTAs: K and V side by side (64 requests of one token: 3.7 us, 4.8 one after the other); many: one look-up for both
        // (the prompts above: 198 us side by side when this form took 171).
        kern<<<dim3(units, y, static_cast<int64_t>(units) * y < 8 * sm_count ? 2 : 1), kCopyThreads, 0, st>>>(a);
    };
    constexpr int rows = warp_rows<T>(LPR);
    if (a.block_size <= rows) go(quantized_copy_kernel<T, E4M3, LPR, 1, false>, 1);
    else if (a.block_size <= 2 * rows) go(quantized_copy_kernel<T, E4M3, LPR, 2, false>, 2);
    else if (a.block_size <= 4 * rows) go(quantized_copy_kernel<T, E4M3, LPR, 4, false>, 4);
    else if (a.block_size <= 8 * rows) go(quantized_copy_kernel<T, E4M3, LPR, 8, false>, 8);
    else go(quantized_copy_kernel<T, E4M3, LPR, 8, true>, 8);
}

template <typename T, int LPR>
void launch_kind(const QuantCopyArgs& a, int units, int sm_count, cudaStream_t st) {
    a.e4m3 ? launch_rows<T, true, LPR>(a, units, sm_count, st) : launch_rows<T, false, LPR>(a, units, sm_count, st);
}

template <typename T>
void launch_t(const QuantCopyArgs& a, int units, int sm_count, cudaStream_t st) {
    bool rows = a.D % 16 == 0 && a.D <= 256;
    for (int m = 0; m < 2; ++m) {
        rows = rows && a.src_s2[m] == 1 && (a.src_s0[m] * sizeof(T)) % 16 == 0 && (a.src_s1[m] * sizeof(T)) % 16 == 0 &&
               reinterpret_cast<uintptr_t>(a.src[m]) % 16 == 0;
        rows = rows && a.c_s3[m] == 1 && a.c_s0[m] % 16 == 0 && a.c_s1[m] % 16 == 0 && a.c_s2[m] % 16 == 0 &&
               reinterpret_cast<uintptr_t>(a.cache[m]) % 16 == 0;
    }
    if (!rows)
        quantized_copy_any_kernel<T><<<dim3(units, a.H, 2), kCopyThreads, 0, st>>>(a);
    else if (a.D <= 64)
        launch_kind<T, 4>(a, units, sm_count, st);
    else if (a.D <= 128)
        launch_kind<T, 8>(a, units, sm_count, st);
    else
        launch_kind<T, 16>(a, units, sm_count, st);
}

}  // namespace

void launch_quantized_copy_kv(const QuantCopyArgs& a, int sm_count, cudaStream_t st) {
    // Touched blocks of a request of n tokens: n at most, and n / block_size + 2 at most.
    const int64_t units = std::min<int64_t>(a.T, a.T / a.block_size + 2ll * a.B);
    if (units <= 0) return;
    if (a.dt == Dt::F16)
        launch_t<__half>(a, static_cast<int>(units), sm_count, st);
    else if (a.dt == Dt::BF16)
        launch_t<__nv_bfloat16>(a, static_cast<int>(units), sm_count, st);
    else
        launch_t<float>(a, static_cast<int>(units), sm_count, st);
}

}  // namespace k
}  // namespace b200
