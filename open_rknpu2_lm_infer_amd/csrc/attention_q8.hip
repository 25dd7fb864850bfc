// The 8-bit KV cache: its C ABI (include/rk_npu_attention_q8.h), bookkeeping,
// and the kernels that write and read it. The attention over it:
// attention_q8.hpp, which also gives the layout.

#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cstring>
#include <mutex>
#include <new>
#include <shared_mutex>

#include "attention.hpp"
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Wunused-function"  // (the headers' other kernels)
#include "attention_q8.hpp"
#pragma clang diagnostic pop
#include "launch.hpp"

namespace hm {

constexpr uint32_t MAGIC_Q8_CACHE = 0x38514841u;

// ---------------------------------------------------------------------------
// Places within the layout, in values (codes: bytes; fp16 rows: halves).
// ---------------------------------------------------------------------------
// code of (key j of its unit, dim d)
__device__ __forceinline__ int q8_k_at(int D, int j, int d) {
    return (((j >> 4) * (D >> 6) + (d >> 6)) * 64 + ((d >> 3) & 3) * 16 + (j & 15)) * 16 + ((d >> 5) & 1) * 8 + (d & 7);
}
__device__ __forceinline__ int q8_v_at(int j, int d) {
    return ((d >> 5) * 64 + ((j >> 2) & 3) * 16 + (d & 15)) * 16 + ((d >> 4) & 1) * 8 + (j >> 4) * 4 + (j & 3);
}
// fp16 row value
__device__ __forceinline__ int q8_kt_at(int D, int j, int d) {
    return (((j >> 4) * (D >> 5) + (d >> 5)) * 64 + ((d >> 3) & 3) * 16 + (j & 15)) * 8 + (d & 7);
}
__device__ __forceinline__ int q8_vt_at(int j, int d) {
    return ((d >> 4) * 64 + ((j >> 2) & 3) * 16 + (d & 15)) * 8 + (j >> 4) * 4 + (j & 3);
}

struct Q8WriteParams {
    HeadsView src[2];  // K, V: the appended rows
    uint8_t* codes[2];
    float4* sc;
    const __half* old_rows[2];  // the open block's fp16 rows, or nullptr: its rows are codes
    __half* open_rows[2];       // where the new open block's rows go (nullptr: none)
    __half* last_rows[2];       // where the last complete block's rows are kept (nullptr: none completes)
    size_t head_bytes;
    int blocks;
    int length, rows;  // before, and appended
};

typedef unsigned q8_u4a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef float q8_f4a4 __attribute__((ext_vector_type(4), aligned(4)));

// The value of a stored code.
__device__ __forceinline__ float q8_value(unsigned code, int fmt) {
    return fmt == RK_NPU_HIP_KV_I8 ? (float)((int)code - 128) : __builtin_amdgcn_cvt_f32_fp8((int)code, 0);
}
__device__ __forceinline__ float q8_scale(const float4& s, int which) {
    return which ? ldexpf(s.y, __float_as_int(s.z)) : s.x;
}
// A block's quantisation: quotients most x / a, correctly rounded, and 4 of them
// as stored codes. The quotient: an approximation, then its exact remainder over a,
// which with a correctly rounded 1 / a gives the nearest f32 (Markstein's
// division). most x is exact (7 or 3 bits and fp16's 11), and a border of two codes
// lies further from any quotient that is not on it than f32 rounds (both are
// multiples of 1 / (2 a'), a' below 2^11, in the code's binade), so the codes are
// the definition's. i8: adding 1.5 2^23 + 128 rounds half to even and leaves code
// + 128 in the low byte.
struct Q8Quantiser {
    float a, inv, most;
    bool poison;
    template <int FMT>
    __device__ __forceinline__ unsigned codes4(const _Float16 (&x)[4]) const {
        float q[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float t = (float)x[i] * most, q0 = t * inv;
            q[i] = __builtin_fmaf(__builtin_fmaf(-q0, a, t), inv, q0);
        }
        if constexpr (FMT == RK_NPU_HIP_KV_I8) {
            unsigned w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(q[i] + 12583040.0f);
            const unsigned lo = __builtin_amdgcn_perm(w[1], w[0], 0x0C0C0400u);
            const unsigned hi = __builtin_amdgcn_perm(w[3], w[2], 0x04000C0Cu);
            return poison ? 0x80808080u : lo | hi;
        } else {
            const int w = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
            return poison ? 0u : (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], w, true);
        }
    }
};

// Threads for a block of B x D values: 16 values each, within 256 and 1024.
constexpr int q8_write_threads(int D, int B) { return B * D <= 4096 ? 256 : B * D >= 16384 ? 1024 : B * D / 16; }

// Writes appended rows. Block: one token block of one KV head, K (blockIdx.z 0) or
// V. Its rows come as fp16 into registers, every load before the first use, the old
// ones of a block that completes from the kept rows (or, after a deep truncation, from
// the block's codes). An open block's go straight to where they are kept. A complete
// block's meet in LDS, where the largest magnitude is known after one barrier and V is
// read transposed (ds_read_b64_tr_b16 hands lane l of 16 dim l of 4 keys).
//
// Measured: 131072 rows of 8 heads of 128, fp16, 138.5 us: 5.8 TB/s read and written.
// 37 rows that complete a block of 64 of 256 dims 5.8 us, one that completes 32 of 128
// 4.3 (8.8 and 5.2 with the old rows taken in row order, V's value by value): the
// launch, a memory round trip, the chain of one block.
template <int D, int B, int FMT>
__global__ __launch_bounds__(q8_write_threads(D, B)) void q8_write_kernel(Q8WriteParams P) {
    typedef short s4 __attribute__((ext_vector_type(4)));
    typedef _Float16 h4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s4 lds_s4;
    constexpr int NT = q8_write_threads(D, B), PT = B * D / 8 / NT;  // 8-value pieces per thread
    constexpr int pitch = D + 8, pieces = D / 8;                     // of a row in LDS, pieces of a row
    __shared__ __attribute__((aligned(16))) _Float16 rows[B * pitch];
    __shared__ unsigned red[NT / 64];
    const int which = blockIdx.z, g = blockIdx.y;
    const int b = P.length / B + blockIdx.x, tid = threadIdx.x;
    const int first = b * B, end = P.length + P.rows;
    const int have = min(end - first, B);  // rows of the block after the call
    const int old = max(0, min(P.length - first, B));
    const bool complete = have == B;
    const HeadsView src = which ? P.src[1] : P.src[0];
    uint8_t* codes = (which ? P.codes[1] : P.codes[0]) + (size_t)g * P.head_bytes + (size_t)first * D;
    float4* sc = P.sc + (size_t)g * P.blocks + b;
    const __half* from = which ? P.old_rows[1] : P.old_rows[0];
    const size_t kept = (size_t)g * B * D;
    const int lane = tid & 63, lo = lane & 15, hi = lane >> 4;
    // The old rows of a block that completes come in the order they are kept in, 8
    // values a thread and piece: K's of one key, V's of one dim. (In an open block the
    // kept rows stay where they are. From codes: row by row, below.)
    const bool ordered = complete && from;
    const int begin = from ? old : 0;
    v4u held[PT], raw[PT][2];
#pragma unroll
    for (int t = 0; t < PT; ++t) {
        const int i = t * NT + tid;
        held[t] = v4u{0u, 0u, 0u, 0u};
        if (ordered && i / (4 * D) * 32 < old) held[t] = *reinterpret_cast<const v4u*>(from + kept + (size_t)i * 8);
    }
#pragma unroll
    for (int t = 0; t < PT; ++t) {
        const int i = t * NT + tid, j = i / pieces, d = i % pieces * 8, unit = j >> 5, ju = j & 31;
        raw[t][0] = raw[t][1] = v4u{0u, 0u, 0u, 0u};
        if (j >= have || j < begin) continue;
        if (j >= old) {
            const long long at = g * src.head + (long long)(first + j - P.length) * src.row + d;
            if (src.f32) {
                const float* p = static_cast<const float*>(src.data) + at;
                raw[t][0] = __builtin_bit_cast(v4u, q8_f4(*reinterpret_cast<const q8_f4a4*>(p)));
                raw[t][1] = __builtin_bit_cast(v4u, q8_f4(*reinterpret_cast<const q8_f4a4*>(p + 4)));
            } else {
                raw[t][0] = v4u(*reinterpret_cast<const q8_u4a2*>(static_cast<const __half*>(src.data) + at));
            }
        } else {
            const uint8_t* p = codes + (size_t)unit * 32 * D;
            const float s = q8_scale(*sc, which);
            q8_h8 h;
#pragma unroll
            for (int k = 0; k < 8; ++k)
                h[k] = (_Float16)(q8_value(p[which ? q8_v_at(ju, d + k) : q8_k_at(D, ju, d + k)], FMT) * s);
            raw[t][0] = __builtin_bit_cast(v4u, h);
        }
    }
    unsigned big = 0;
#pragma unroll
    for (int t = 0; t < PT; ++t) {
        const int i = t * NT + tid, unit = i / (4 * D), step = (i >> 6) % (D / 16);
        if (!ordered || unit * 32 >= old) continue;  // (whole waves)
        if (which == 0) {
            const int j = unit * 32 + step / (D / 32) * 16 + lo;
            if (j >= old) held[t] = v4u{0u, 0u, 0u, 0u};
            if (j < old) *reinterpret_cast<v4u*>(rows + j * pitch + step % (D / 32) * 32 + 8 * hi) = held[t];
        } else {
            const q8_h8 h = __builtin_bit_cast(q8_h8, held[t]);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int j = unit * 32 + (k >> 2) * 16 + 4 * hi + (k & 3);
                if (j < old)
                    rows[j * pitch + 16 * step + lo] = h[k];
                else
                    held[t][k >> 1] &= k & 1 ? 0xFFFFu : 0xFFFF0000u;
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) big = max(big, max(held[t][k] & 0x7FFFu, (held[t][k] >> 16) & 0x7FFFu));
    }
#pragma unroll
    for (int t = 0; t < PT; ++t) {
        const int i = t * NT + tid, j = i / pieces, d = i % pieces * 8;
        if (j >= have || j < begin) continue;
        if (src.f32 && j >= old) {
            const q8_f4 x = __builtin_bit_cast(q8_f4, raw[t][0]), y = __builtin_bit_cast(q8_f4, raw[t][1]);
            q8_h8 h;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                h[k] = (_Float16)x[k];
                h[4 + k] = (_Float16)y[k];
            }
            raw[t][0] = __builtin_bit_cast(v4u, h);
        }
        if (complete) {
            *reinterpret_cast<v4u*>(rows + j * pitch + d) = raw[t][0];
#pragma unroll
            for (int k = 0; k < 4; ++k)
                big = max(big, max(raw[t][0][k] & 0x7FFFu, (raw[t][0][k] >> 16) & 0x7FFFu));
        } else {
            __half* p = (which ? P.open_rows[1] : P.open_rows[0]) + kept + (size_t)(j >> 5) * 32 * D;
            if (which == 0) {
                *reinterpret_cast<v4u*>(p + q8_kt_at(D, j & 31, d)) = raw[t][0];
            } else {
                unsigned short* u = reinterpret_cast<unsigned short*>(p);
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    u[q8_vt_at(j & 31, d + k)] = (unsigned short)(raw[t][0][k >> 1] >> (16 * (k & 1)));
            }
        }
    }
    if (!complete) return;  // (block-uniform)
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) big = max(big, (unsigned)__shfl_xor((int)big, i));
    if ((tid & 63) == 0) red[tid >> 6] = big;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) big = max(big, red[i]);
    // (zeros only: the smallest scale there is, which lifts no row's maximum)
    big = max(big, 1u);

    Q8Quantiser Q;
    Q.most = FMT == RK_NPU_HIP_KV_I8 ? 127.0f : 448.0f;
    Q.poison = big >= 0x7C00u;
    const float a = __half2float(__ushort_as_half((unsigned short)big));
    Q.a = Q.poison ? 1.0f : a;
    Q.inv = 1.0f / Q.a;
    if (tid == 0) {
        const float s = Q.poison ? NAN : a / Q.most;
        if (which == 0) {
            sc->x = s;
        } else {
            // (a / most is a normal number: a >= 2^-24)
            const int bits = __float_as_int(s), e = Q.poison ? 0 : ((bits >> 23) & 255) - 127;
            sc->y = Q.poison ? NAN : __int_as_float((bits & 0x7FFFFF) | 0x3F800000);
            sc->z = __int_as_float(e);
            sc->w = 1.0f / s;
        }
    }
    // lane (lo, hi)'s dim 16 n + lo of keys 4 hi..+3 of 16 keys from row j0
    auto transposed = [&](int j0, int n) {
        const _Float16* p = rows + (j0 + 4 * hi + (lo >> 2)) * pitch + 16 * n + 4 * (lo & 3);
        return __builtin_bit_cast(h4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)p));
    };
    // the last complete block's fp16 rows are kept too
    __half* keep = which ? P.last_rows[1] : P.last_rows[0];
    if (keep && first + 2 * B > end) {
#pragma unroll
        for (int t = 0; t < PT; ++t) {
            const int i = t * NT + tid, unit = i / (4 * D), step = (i >> 6) % (D / 16);
            q8_h8 h;
            if (which == 0) {
                const int at = step % (D / 32) * 32 + 8 * hi, j = unit * 32 + step / (D / 32) * 16 + lo;
                h = *reinterpret_cast<const q8_h8*>(rows + j * pitch + at);
            } else {
                const h4 x = transposed(unit * 32, step), y = transposed(unit * 32 + 16, step);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    h[k] = x[k];
                    h[4 + k] = y[k];
                }
            }
            *reinterpret_cast<q8_h8*>(keep + kept + (size_t)i * 8) = h;
        }
    }
    // the codes, in the order they lie in
#pragma unroll
    for (int t = 0; t < (PT + 1) / 2; ++t) {
        const int i = t * NT + tid, unit = i / (2 * D), step = (i >> 6) % (D / 32);
        if (PT == 1 && i >= B * D / 16) break;  // (whole waves)
        v4u w;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            _Float16 x[4], y[4];
            if (which == 0) {  // step: [16-key half][64-dim step]
                const int at = step % (D / 64) * 64 + 32 * half + 8 * hi, j = unit * 32 + step / (D / 64) * 16 + lo;
                const q8_h8 h = *reinterpret_cast<const q8_h8*>(rows + j * pitch + at);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    x[k] = h[k];
                    y[k] = h[4 + k];
                }
            } else {
                const h4 h0 = transposed(unit * 32, 2 * step + half), h1 = transposed(unit * 32 + 16, 2 * step + half);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    x[k] = h0[k];
                    y[k] = h1[k];
                }
            }
            w[2 * half] = Q.template codes4<FMT>(x);
            w[2 * half + 1] = Q.template codes4<FMT>(y);
        }
        *reinterpret_cast<v4u*>(codes + (size_t)i * 16) = w;
    }
}

struct Q8ReadParams {
    HeadsView dst[2];
    const uint8_t* codes[2];
    const float4* sc;
    const __half* tail[2];
    size_t head_bytes;
    int blocks, block, unit_shift, fmt;
    int first, rows, coded;
};

// Reads rows back. Block: one unit of one KV head, K or V. The unit's codes (or
// fp16 rows) meet in LDS row by row, then leave as rows.
template <int D>
__global__ __launch_bounds__(256) void q8_read_kernel(Q8ReadParams P) {
    constexpr int pitch = D + 16, pieces = D / 8;
    __shared__ __attribute__((aligned(16))) uint8_t bytes[32 * pitch];
    const int which = blockIdx.z, g = blockIdx.y, tid = threadIdx.x;
    const HeadsView dst = which ? P.dst[1] : P.dst[0];
    if (!dst.data) return;
    const int unit = (P.first >> 5) + blockIdx.x, key0 = unit * 32;
    const bool coded = key0 < P.coded;
    const int j0 = max(0, P.first - key0), j1 = min(32, P.first + P.rows - key0);
    float scale = 1.0f;
    if (coded) {
        scale = q8_scale(P.sc[(size_t)g * P.blocks + (unit >> P.unit_shift)], which);
        const uint8_t* src = (which ? P.codes[1] : P.codes[0]) + (size_t)g * P.head_bytes + (size_t)key0 * D;
        for (int i = tid; i < 2 * D; i += 256) {
            const v4u x = *reinterpret_cast<const v4u*>(src + i * 16);
            const int lane = i & 63, lo = lane & 15, hi = lane >> 4;
            if (which == 0) {
                const int j = (i >> 6) / (D >> 6) * 16 + lo, d = (i >> 6) % (D >> 6) * 64 + 8 * hi;
                *reinterpret_cast<uint2*>(bytes + j * pitch + d) = uint2{x[0], x[1]};
                *reinterpret_cast<uint2*>(bytes + j * pitch + d + 32) = uint2{x[2], x[3]};
            } else {
#pragma unroll
                for (int k = 0; k < 16; ++k)
                    bytes[(((k >> 2) & 1) * 16 + 4 * hi + (k & 3)) * pitch + (i >> 6) * 32 + (k >> 3) * 16 + lo] =
                        (uint8_t)(x[k >> 2] >> (8 * (k & 3)));
            }
        }
        __syncthreads();
    }
    const __half* tail = (which ? P.tail[1] : P.tail[0]) + (size_t)g * P.block * D + (coded ? 0 : (size_t)(key0 - P.coded) * D);
    for (int i = j0 * pieces + tid; i < j1 * pieces; i += 256) {
        const int j = i / pieces, d = i % pieces * 8;
        float y[8];
        if (coded) {
            const uint2 x = *reinterpret_cast<const uint2*>(bytes + j * pitch + d);
#pragma unroll
            for (int k = 0; k < 8; ++k)
                y[k] = q8_value(((k < 4 ? x.x : x.y) >> (8 * (k & 3))) & 255u, P.fmt) * scale;
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) y[k] = __half2float(tail[which ? q8_vt_at(j, d + k) : q8_kt_at(D, j, d + k)]);
        }
        const long long at = g * dst.head + (long long)(key0 + j - P.first) * dst.row + d;
        if (dst.f32) {
            float* p = static_cast<float*>(dst.data) + at;
            *reinterpret_cast<q8_f4a4*>(p) = q8_f4a4{y[0], y[1], y[2], y[3]};
            *reinterpret_cast<q8_f4a4*>(p + 4) = q8_f4a4{y[4], y[5], y[6], y[7]};
        } else {
            v4u w;
#pragma unroll
            for (int k = 0; k < 4; ++k)
                w[k] = __half_as_ushort(__float2half_rn(y[2 * k])) |
                       ((unsigned)__half_as_ushort(__float2half_rn(y[2 * k + 1])) << 16);
            *reinterpret_cast<q8_u4a2*>(static_cast<__half*>(dst.data) + at) = q8_u4a2(w);
        }
    }
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------
// Which fp16 rows the three kept slots hold, and what the cache reads: keys below
// `coded` as codes, the others (of block `length` / B) from slot `open`.
struct Q8Rows {
    int length = 0, coded = 0, open = -1;
    int block[Q8_SLOTS] = {-1, -1, -1};  // the token block a slot holds the first `rows` rows of
    int rows[Q8_SLOTS] = {0, 0, 0};

    // A slot to write, none of a, b, c: an empty one, else that of the earliest block.
    int pick(int a, int b, int c) const {
        int best = -1;
        for (int i = 0; i < Q8_SLOTS; ++i)
            if (i != a && i != b && i != c && (best < 0 || block[i] < block[best])) best = i;
        return best;
    }
    void forget_from(int b) {  // blocks b and later
        for (int i = 0; i < Q8_SLOTS; ++i)
            if (block[i] >= b) block[i] = -1, rows[i] = 0;
    }
    void truncate(int B, int len) {
        const int b = len / B, t = len % B;
        forget_from(b + 1);
        int at = -1;
        for (int i = 0; i < Q8_SLOTS; ++i) {
            if (block[i] != b) continue;
            rows[i] = std::min(rows[i], t);
            if (rows[i] == t && t > 0) at = i;
            if (rows[i] == 0) block[i] = -1;
        }
        length = len;
        open = at;
        coded = at >= 0 || t == 0 ? b * B : (b + 1) * B;
    }
};

// One append: the slot its old rows come from (-1: none, or codes), the slots the
// last complete and the new open block go to (-1: none), the bookkeeping after.
// Kept then: these three. The old rows' slot is written only after them, so the
// call can be undone, and a captured one repeated.
// A call in several pieces, all but the last of which end with a block, leaves the
// rows it began with where they are, and its last complete block: slots `begun` and
// `done` (-1: none). Pieces behind the first have no old rows, so there is a slot for
// each of last and open.
struct Q8Step {
    int from, last, open;
    Q8Rows after;
};
static Q8Step q8_step(const Q8Rows& now, int B, int n, int begun, int done) {
    Q8Step s{now.open, -1, -1, now};
    Q8Rows& a = s.after;
    a.length = now.length + n;
    const int b0 = now.length / B, b1 = a.length / B, r = a.length % B;
    if (now.open < 0) a.forget_from(b0);  // (rows of a block that is rewritten from its codes)
    if (b1 > b0) {
        s.last = b1 - 1 == b0 && s.from >= 0 ? s.from : a.pick(s.from, begun, -1);
        done = s.last;
        a.block[s.last] = b1 - 1;
        a.rows[s.last] = B;
    }
    if (r > 0) {
        s.open = b1 == b0 && s.from >= 0 ? s.from : a.pick(s.from, begun, done);
        a.block[s.open] = b1;
        a.rows[s.open] = r;
    }
    a.open = s.open;
    a.coded = b1 * B;
    for (int i = 0; i < Q8_SLOTS; ++i)
        if (i != s.from && i != s.open && i != begun && i != done) a.block[i] = -1, a.rows[i] = 0;
    return s;
}

struct Q8Cache {
    uint32_t magic;
    Domain* domain;
    rk_npu_hip_attention_q8_config cfg;
    uint8_t* codes[2];  // K, V: [kv_heads][capacity * D]
    float4* sc;         // [kv_heads][capacity / block]
    __half* kept[2];    // [slots][kv_heads][block * D]
    int capacity;
    size_t code_bytes, scale_bytes, kept_bytes;  // of one array each
    uint64_t generation;
    Q8Rows rows;
    std::shared_mutex mu;  // the fields above, against calls from several threads; a host run holds it to its end
    DevFence fence;  // device-path appends, reads and runs
    hipStream_t stream = nullptr;  // host-buffer appends and reads (created on the first)
    HostStage hs;                  // their pinned staging
};

static Q8Cache* as_q8(const void* p) {
    Q8Cache* c = static_cast<Q8Cache*>(const_cast<void*>(p));
    return (c && c->magic == MAGIC_Q8_CACHE) ? c : nullptr;
}

static bool valid_q8(const rk_npu_hip_attention_q8_config* c) {
    return c && valid_config(&c->attention) && (c->format == RK_NPU_HIP_KV_I8 || c->format == RK_NPU_HIP_KV_E4M3) &&
           (c->block == 32 || c->block == 64 || c->block == 128) && c->attention.max_capacity <= INT_MAX - 255;
}
static size_t q8_code_bytes(const rk_npu_hip_attention_q8_config& c, int capacity) {
    return (size_t)c.attention.kv_heads * capacity * c.attention.head_dim;
}
static size_t q8_scale_bytes(const rk_npu_hip_attention_q8_config& c, int capacity) {
    return (size_t)c.attention.kv_heads * (capacity / c.block) * sizeof(float4);
}
static size_t q8_kept_bytes(const rk_npu_hip_attention_q8_config& c) {
    return (size_t)Q8_SLOTS * c.attention.kv_heads * c.block * c.attention.head_dim * sizeof(__half);
}
static int q8_max_capacity(const Q8Cache* c) { return round_up(c->cfg.attention.max_capacity, c->cfg.block); }
static __half* q8_slot(const Q8Cache* c, int which, int slot) {
    if (slot < 0) return nullptr;
    return c->kept[which] + (size_t)slot * c->cfg.attention.kv_heads * c->cfg.block * c->cfg.attention.head_dim;
}

// Storage of `capacity` rows into k, v, sc; false (nothing kept) when the device
// has no room.
static bool q8_alloc(Q8Cache* c, int capacity, uint8_t* (&codes)[2], float4*& sc) {
    const size_t cb = q8_code_bytes(c->cfg, capacity), sb = q8_scale_bytes(c->cfg, capacity);
    codes[0] = static_cast<uint8_t*>(domain_alloc(c->domain, cb));
    codes[1] = codes[0] ? static_cast<uint8_t*>(domain_alloc(c->domain, cb)) : nullptr;
    sc = codes[1] ? static_cast<float4*>(domain_alloc(c->domain, sb)) : nullptr;
    if (sc) return true;
    domain_free(c->domain, codes[0], cb);
    domain_free(c->domain, codes[1], cb);
    return false;
}

static int q8_grow(Q8Cache* c, int capacity) {
    if (capacity > q8_max_capacity(c)) return RK_NPU_ERR_PARAM;
    capacity = round_up(capacity, c->cfg.block);
    if (capacity <= c->capacity) return RK_NPU_OK;
    uint8_t* codes[2];
    float4* sc;
    if (!q8_alloc(c, capacity, codes, sc)) return RK_NPU_ERR_NOMEM;
    const size_t cb = q8_code_bytes(c->cfg, capacity), sb = q8_scale_bytes(c->cfg, capacity);
    const int kh = c->cfg.attention.kv_heads, D = c->cfg.attention.head_dim, B = c->cfg.block;
    bool ok = true;
    if (c->rows.coded > 0) {
        const size_t held = (size_t)c->rows.coded * D;
        for (int i = 0; i < 2; ++i)
            ok = ok && hipMemcpy2D(codes[i], (size_t)capacity * D, c->codes[i], (size_t)c->capacity * D, held, kh,
                                   hipMemcpyDeviceToDevice) == hipSuccess;
        ok = ok && hipMemcpy2D(sc, (size_t)(capacity / B) * sizeof(float4), c->sc,
                               (size_t)(c->capacity / B) * sizeof(float4),
                               (size_t)(c->rows.coded / B) * sizeof(float4), kh, hipMemcpyDeviceToDevice) == hipSuccess;
        // (copies within the device may return before they are done)
        ok = ok && hipStreamSynchronize(nullptr) == hipSuccess;
    }
    if (!ok) {
        for (int i = 0; i < 2; ++i) domain_free(c->domain, codes[i], cb);
        domain_free(c->domain, sc, sb);
        return RK_NPU_ERR_DEVICE;
    }
    for (int i = 0; i < 2; ++i) {
        domain_free(c->domain, c->codes[i], c->code_bytes);
        c->codes[i] = codes[i];
    }
    domain_free(c->domain, c->sc, c->scale_bytes);
    c->sc = sc;
    c->capacity = capacity;
    c->code_bytes = cb;
    c->scale_bytes = sb;
    c->generation += 1;
    return RK_NPU_OK;
}

template <int D, int FMT>
static void q8_launch_write(const Q8WriteParams& P, int B, const dim3& grid, hipStream_t s) {
    if (B == 32)
        hipLaunchKernelGGL((q8_write_kernel<D, 32, FMT>), grid, dim3(q8_write_threads(D, 32)), 0, s, P);
    else if (B == 64)
        hipLaunchKernelGGL((q8_write_kernel<D, 64, FMT>), grid, dim3(q8_write_threads(D, 64)), 0, s, P);
    else
        hipLaunchKernelGGL((q8_write_kernel<D, 128, FMT>), grid, dim3(q8_write_threads(D, 128)), 0, s, P);
}
template <int FMT>
static void q8_launch_write(const Q8WriteParams& P, int D, int B, const dim3& grid, hipStream_t s) {
    if (D == 64)
        q8_launch_write<64, FMT>(P, B, grid, s);
    else if (D == 128)
        q8_launch_write<128, FMT>(P, B, grid, s);
    else
        q8_launch_write<256, FMT>(P, B, grid, s);
}

// Enqueues an append (room and views checked) and advances the bookkeeping.
static int q8_enqueue_append(Q8Cache* c, const HeadsView& k, const HeadsView& v, int n, hipStream_t s,
                             int begun = -1, int* done = nullptr) {
    const int B = c->cfg.block, D = c->cfg.attention.head_dim;
    const Q8Step st = q8_step(c->rows, B, n, begun, done ? *done : -1);
    Q8WriteParams P;
    P.src[0] = k;
    P.src[1] = v;
    for (int i = 0; i < 2; ++i) {
        P.codes[i] = c->codes[i];
        P.old_rows[i] = q8_slot(c, i, st.from);
        P.open_rows[i] = q8_slot(c, i, st.open);
        P.last_rows[i] = q8_slot(c, i, st.last);
    }
    P.sc = c->sc;
    P.head_bytes = (size_t)c->capacity * D;
    P.blocks = c->capacity / B;
    P.length = c->rows.length;
    P.rows = n;
    const int blocks = (c->rows.length + n - 1) / B - c->rows.length / B + 1;
    const dim3 grid(blocks, c->cfg.attention.kv_heads, 2);
    if (c->cfg.format == RK_NPU_HIP_KV_I8)
        q8_launch_write<RK_NPU_HIP_KV_I8>(P, D, B, grid, s);
    else
        q8_launch_write<RK_NPU_HIP_KV_E4M3>(P, D, B, grid, s);
    if (hipGetLastError() != hipSuccess) return RK_NPU_ERR_DEVICE;
    c->rows = st.after;
    if (done && st.last >= 0) *done = st.last;
    return RK_NPU_OK;
}

static int q8_enqueue_read(Q8Cache* c, int first, int n, const HeadsView& k, const HeadsView& v, hipStream_t s) {
    const int B = c->cfg.block, D = c->cfg.attention.head_dim;
    Q8ReadParams P;
    P.dst[0] = k;
    P.dst[1] = v;
    for (int i = 0; i < 2; ++i) {
        P.codes[i] = c->codes[i];
        P.tail[i] = q8_slot(c, i, std::max(c->rows.open, 0));
    }
    P.sc = c->sc;
    P.head_bytes = (size_t)c->capacity * D;
    P.blocks = c->capacity / B;
    P.block = B;
    P.unit_shift = B == 32 ? 0 : B == 64 ? 1 : 2;
    P.fmt = c->cfg.format;
    P.first = first;
    P.rows = n;
    P.coded = c->rows.coded;
    const int units = (first + n - 1) / 32 - first / 32 + 1;
    const dim3 grid(units, c->cfg.attention.kv_heads, 2);
    if (D == 64)
        hipLaunchKernelGGL(q8_read_kernel<64>, grid, dim3(256), 0, s, P);
    else if (D == 128)
        hipLaunchKernelGGL(q8_read_kernel<128>, grid, dim3(256), 0, s, P);
    else
        hipLaunchKernelGGL(q8_read_kernel<256>, grid, dim3(256), 0, s, P);
    return hipGetLastError() == hipSuccess ? RK_NPU_OK : RK_NPU_ERR_DEVICE;
}

// Many splits or few rows: a block for 64 dims of a row, whose threads load 128 splits
// at once (8 rows of 2 heads of 256, 126 splits: 4.5 us; 6.6 with a block for all 256
// dims, 5.3 with one of 1024 threads). Else rows a block, as many as leave a row the threads for its dims.
template <int D>
static void q8_combine(const AttnQ8Params& P, int R, hipStream_t s) {
    constexpr int MANY = D == 256 ? 4 : 8;
    if (P.splits > 16 || R * P.kh < 512)
        hipLaunchKernelGGL((attn_q8_combine_kernel<D, 1, 64>), dim3(R, P.kh, D / 64), dim3(256), 0, s, P);
    else
        hipLaunchKernelGGL((attn_q8_combine_kernel<D, MANY, D>), dim3((R + MANY - 1) / MANY, P.kh), dim3(256), 0, s,
                           P);
}

// The kernel, for R query rows of each KV head. attn_q8_kernel converts a unit's codes
// in every wave: in blocks of one row group, for few rows, on 4 waves (8 on half as many
// splits: one row of 32 heads over 8 of 128 and 3981 keys 8.5 us instead of 8.0, 64
// heads over 8 of 256 and 16001 keys 19.4 and 17.0), or of two, which share a unit's
// conversion. Two of 256 dims take every register of a SIMD, and pay over many keys
// only: i8, 2 KV heads, 512 rows x 16000 keys 45.4 with one and 35.5 with two, x 8000
// 27.5 and 24.6, x 4000 17.7 and 20.0; 2048 x 4000 35.9 and 35.6 (e4m3 27.8 and 32.1).
//
// attn_q8_tile_kernel converts once a block, which takes rows enough to fill 128- or
// 256-row blocks and keys enough to fill its stages; the more, the cheaper the
// conversion. `cross`: where they do, in million rows x keys x dims a CU; the more rows
// for the same work the later. Measured, us, in every wave and once a block, 8 KV heads
// (256 dims: 2), 512 rows:
//   64 dims, i8: 32000 keys (16) 37.6 and 41.8, 64000 (33) 67.4 and 60.2; f32 output 46.3
//   and 49.5, 84.6 and 76.3; e4m3: (33) 62.0 and 59.7, (66) 114 and 103, but 1024 rows (33)
//   54.8 and 62.7, (66) 104 and 103; f32: (33) 77.8 and 74.1, 1024 rows 71.0 and 77.2;
//   128 dims, i8: 16000 (33) 53.6 and 52.0, 1024 rows 45.2 and 54.6, (66) 88.6 and 83.7;
//   f32: 65.1 and 63.8, 59.4 and 65.2, 115 and 108; e4m3: (33) 48.7 and 50.6, (66) 84.1 and
//   80.9, 1024 rows 79.5 and 81.6, (131) 151 and 140; f32: (66) 111 and 106, 102 and 106;
//   256 dims, 1024 rows, i8: 8000 (16) 35.3 and 37.8, (33) 57.1 and 55.7, (66) 100 and 91;
//   f32: 40.8 and 43.2, 67.7 and 65.2; e4m3: (33) 50.6 and 54.2, (66) 87.2 and 88.8, (131)
//   159 and 157; f32: 61.4 and 63.9, 110 and 106.
static Q8Plan q8_plan(int D, int R, int kv_heads, int units, bool i8, bool f16) {
    static const float cross[3][3] = {{30, 45, 33}, {45, 70, 60}, {55, 70, 100}};  // by head_dim 64, 128, 256
    const int forced = attention_q8_tile_switch();
    const double work = 1e-6 * D * R * kv_heads * units * 32 / device_cus();
    const double most = cross[i8 ? 0 : f16 ? 2 : 1][D / 128];
    if (forced == 1 || (forced < 0 && R > 16 && work > most)) return Q8Plan{true, D == 256 ? 1 : 2, 8};
    if (R <= 16) return Q8Plan{false, 1, 4};
    if (D < 256) return Q8Plan{false, 2, 8};
    return Q8Plan{false, forced == 2 || (forced < 0 && work > 10 && units > 200) ? 2 : 1, 4};
}

// Key splits: a block for each CU, but no more, as a block's rows leave partials (512
// rows of 8 heads over 4096 keys 21.9 us, 27.6 with 512 blocks, 25.5 with 128; one row
// of 16 heads over 2 of 256 and 20000 keys 11.3, 16.2 with 512). 4 waves of 64 dims have
// too few bytes on their way for a CU, which two blocks make up for once they are long
// (one row of 16 heads over 8 of 64: 300000 keys 55 us, 76 with 256 blocks, 40000 13.5
// and 14.5, 20000 9.6 and 9.7; over 2: 131000 12.7 and 12.8, 65000 10.4 and 9.6).
// A split holds at least a unit for each wave, or two stages. Few keys are not split: a
// wave walks its 4 to 6 units in the time of the join's launch, 3 us. One row of 32
// heads over 8 of 128: 768 keys 6.5, split 7.1, 1000 keys 8.5 and 7.7; of 16 over 2 of
// 256: 480 keys 7.4 and 7.9, 768 keys 9.3 and 8.2; 64 rows of 32 over 8 of 128 (8
// waves): 1000 keys 11.2 and 12.8, 1500 keys 13.7 and 13.5.
static void q8_splits(AttnQ8Params& P, int D, int R, const Q8Plan& plan) {
    const int rows = plan.rows();
    P.row_tiles = (R + rows - 1) / rows;
    P.rows_pad = P.row_tiles * rows;
    const int base = P.row_tiles * P.kh, least = plan.tile ? 4 : plan.waves;
    const int cus = device_cus();
    const int blocks = D == 64 && plan.waves == 4 && (long)P.units * base > 32 * cus ? 2 * cus : cus;
    const int few = D == 256 ? 16 : plan.waves == 4 ? 24 : 32;
    const size_t room = attn_partial_rows(D) / ((size_t)P.rows_pad * P.kh);
    int want = std::max(1, std::min((blocks + base - 1) / base, (P.units + least - 1) / least));
    want = (int)std::min<size_t>(std::min(want, Q8_MAX_SPLITS), std::max<size_t>(1, room));
    if (P.units <= few) want = 1;
    P.units_per_split = ((P.units + want - 1) / want + least - 1) / least * least;
    P.splits = (P.units + P.units_per_split - 1) / P.units_per_split;
}

static int q8_enqueue_run(AttnWork* w, Q8Cache* c, const HeadsView& q, int rows, int pos, const HeadsView& out,
                          hipStream_t s) {
    const rk_npu_attention_f16_config& cfg = c->cfg.attention;
    const bool causal = cfg.mask_mode == RK_NPU_ATTENTION_F16_CAUSAL;
    const int len = c->rows.length, D = cfg.head_dim, B = c->cfg.block;
    if (rows < 1 || rows > w->cfg.max_query_rows || pos < 0 || len < 1) return RK_NPU_ERR_PARAM;
    if (causal && (long)pos + rows > len) return RK_NPU_ERR_PARAM;
    AttnQ8Params P;
    P.q = q.data;
    P.q_f32 = q.f32;
    P.q_head = q.head;
    P.q_row = q.row;
    P.out = out.data;
    P.out_f16 = !out.f32;
    P.o_head = out.head;
    P.o_row = out.row;
    P.k = c->codes[0];
    P.v = c->codes[1];
    P.sc = c->sc;
    P.kt = q8_slot(c, 0, std::max(c->rows.open, 0));
    P.vt = q8_slot(c, 1, std::max(c->rows.open, 0));
    P.part = w->part;
    P.qh = cfg.query_heads;
    P.kh = cfg.kv_heads;
    P.m = rows;
    P.len = len;
    P.pos = causal ? pos : 0;
    P.causal = causal ? 1 : 0;
    P.scale = cfg.softmax_scale;
    P.head_bytes = (size_t)c->capacity * D;
    P.blocks = c->capacity / B;
    P.unit_shift = B == 32 ? 0 : B == 64 ? 1 : 2;
    P.block_values = B * D;
    P.coded = c->rows.coded;
    P.units = ((causal ? std::min(len, pos + rows) : len) + 31) / 32;
    const int R = cfg.query_heads / cfg.kv_heads * rows;
    const Q8Plan plan = q8_plan(D, R, cfg.kv_heads, P.units, c->cfg.format == RK_NPU_HIP_KV_I8, P.out_f16);
    q8_splits(P, D, R, plan);
    // Weights as two fp16: always for f32 output, and for fp16 output where it costs
    // little, so that the output's rounding is all that is lost: one row of 32 heads over 8
    // of 128, 4000 keys 7.9 us (one fp16 7.8), 16000 10.8 (10.4), 131000 45.4 (44.5).
    const bool two = !P.out_f16 || (!plan.tile && R <= 16);
    (c->cfg.format == RK_NPU_HIP_KV_I8 ? launch_attn_q8_i8 : launch_attn_q8_e4m3)(P, D, plan, two, s);
    if (P.splits > 1) {
        if (D == 64)
            q8_combine<64>(P, R, s);
        else if (D == 128)
            q8_combine<128>(P, R, s);
        else
            q8_combine<256>(P, R, s);
    }
    return hipGetLastError() == hipSuccess ? RK_NPU_OK : RK_NPU_ERR_DEVICE;
}

static bool same_geometry(const AttnWork* w, const Q8Cache* c) {
    const rk_npu_attention_f16_config &a = w->cfg, &b = c->cfg.attention;
    return a.query_heads == b.query_heads && a.kv_heads == b.kv_heads && a.head_dim == b.head_dim &&
           a.mask_mode == b.mask_mode && a.softmax_scale == b.softmax_scale && device_of(w->domain) == device_of(c->domain);
}

// The cache's own stream and a stage of at least `bytes`.
static void* q8_stage(Q8Cache* c, size_t bytes) {
    if (!c->stream && hipStreamCreateWithFlags(&c->stream, hipStreamNonBlocking) != hipSuccess) {
        (void)hipGetLastError();
        c->stream = nullptr;
        return nullptr;
    }
    return stage_reserve(c->hs, bytes);
}
// Rows that a staged piece of a host call holds: the stage's 8 MiB at most.
static int q8_stage_rows(const Q8Cache* c, int rows) {
    const size_t row = (size_t)c->cfg.attention.kv_heads * c->cfg.attention.head_dim * sizeof(__half);
    return (int)std::min<size_t>(rows, std::max<size_t>(1, ((size_t)8 << 20) / (2 * row)));
}
static bool q8_stage_done(Q8Cache* c, void* st) {
    const bool word = host_kernels_enabled() && c->hs.done;
    if (stage_download(c->hs, word, st, nullptr, nullptr, 0, c->stream)) return true;
    (void)hipStreamSynchronize(c->stream);
    return false;
}

// Host rows through the pinned stage, which the write kernel reads (each row
// once); a piece at a time, done on return. Room is there.
static int q8_put_host(Q8Cache* c, const uint16_t* k, const uint16_t* v, int rows) {
    const int kh = c->cfg.attention.kv_heads, D = c->cfg.attention.head_dim, step = q8_stage_rows(c, rows);
    const size_t each = (size_t)kh * step * D;
    uint16_t* st = static_cast<uint16_t*>(q8_stage(c, 2 * each * sizeof(uint16_t)));
    if (!st) return RK_NPU_ERR_NOMEM;
    const int start = c->rows.length, begun = c->rows.open;
    int done = -1;
    for (int r = 0, n; r < rows; r += n) {
        n = std::min(step, rows - r);
        if (r + n < rows) n -= (start + r + n) % c->cfg.block;  // (step is at least 256: the stage holds them)
        for (int g = 0; g < kh; ++g) {
            const size_t at = ((size_t)g * rows + r) * D, to = (size_t)g * n * D;
            std::memcpy(st + to, k + at, (size_t)n * D * sizeof(uint16_t));
            std::memcpy(st + each + to, v + at, (size_t)n * D * sizeof(uint16_t));
        }
        uint16_t* dev = static_cast<uint16_t*>(c->hs.dev);
        int rc = q8_enqueue_append(c, HeadsView{dev, 0, (long long)n * D, D},
                                   HeadsView{dev + each, 0, (long long)n * D, D}, n, c->stream, begun, &done);
        if (rc == RK_NPU_OK && !q8_stage_done(c, st)) rc = RK_NPU_ERR_DEVICE;
        if (rc != RK_NPU_OK) {
            c->rows.truncate(c->cfg.block, start);  // (nothing of a failed call stays)
            return rc;
        }
    }
    return RK_NPU_OK;
}

static int q8_run_host(rk_npu_attention_f16_workspace* workspace, rk_npu_hip_attention_q8_cache* cache,
                       const uint16_t* q, int rows, int pos, void* out, bool out_f16,
                       rk_npu_attention_f16_timings* t) {
    AttnWork* w = as_attn_work(workspace);
    Q8Cache* c = as_q8(cache);
    if (!w || !c || !q || !out || !same_geometry(w, c)) return RK_NPU_ERR_PARAM;
    if (rows < 1 || rows > w->cfg.max_query_rows) return RK_NPU_ERR_PARAM;
    BusyGuard busy(w->busy);
    if (!busy.ok) return RK_NPU_ERR_BUSY;
    DeviceGuard dev(device_of(w->domain));
    if (!dev.ok) return RK_NPU_ERR_DEVICE;
    std::shared_lock<std::shared_mutex> lock(c->mu);
    const double t0 = now_us();
    const int D = c->cfg.attention.head_dim;
    const size_t n = (size_t)c->cfg.attention.query_heads * rows * D;
    const size_t qb = n * sizeof(__half), ob = n * (out_f16 ? sizeof(__half) : sizeof(float));
    if (c->fence.wait(w->stream) != hipSuccess || w->fence.wait(w->stream) != hipSuccess) return RK_NPU_ERR_DEVICE;
    void* st = stage_reserve(w->hs, std::max(qb, ob));
    const bool small = stage_small(w->hs, st, qb, ob);
    const HostSeg seg{q, w->q, qb, 0};
    int rc = RK_NPU_OK;
    if (!stage_upload(w->hs, small, st, &seg, 1, w->stream) || (t && hipStreamSynchronize(w->stream) != hipSuccess))
        rc = RK_NPU_ERR_DEVICE;
    const double t1 = now_us();
    if (rc == RK_NPU_OK)
        rc = q8_enqueue_run(w, c, HeadsView{w->q, 0, (long long)rows * D, D}, rows, pos,
                            HeadsView{w->out, out_f16 ? 0 : 1, (long long)rows * D, D}, w->stream);
    if (rc == RK_NPU_OK && t && hipStreamSynchronize(w->stream) != hipSuccess) rc = RK_NPU_ERR_DEVICE;
    const double t2 = now_us();
    if (rc == RK_NPU_OK && !stage_download(w->hs, small, st, out, w->out, ob, w->stream)) rc = RK_NPU_ERR_DEVICE;
    if (rc != RK_NPU_OK) (void)hipStreamSynchronize(w->stream);
    const double t3 = now_us();
    if (t) {
        t->upload_us = t1 - t0;
        t->device_us = t2 - t1;
        t->download_us = t3 - t2;
        t->total_us = t3 - t0;
    }
    return rc;
}

}  // namespace hm

using namespace hm;

extern "C" {

void rk_npu_hip_attention_q8_config_init(rk_npu_hip_attention_q8_config* c) {
    if (!c) return;
    std::memset(c, 0, sizeof(*c));
    rk_npu_attention_f16_config_init(&c->attention);
    c->format = RK_NPU_HIP_KV_I8;
    c->block = 32;
}

int rk_npu_hip_attention_q8_query(const rk_npu_hip_attention_q8_config* c, int32_t capacity, int32_t query_rows,
                                  rk_npu_attention_f16_sizes* sizes) {
    if (!valid_q8(c) || !sizes || capacity < 0 || capacity > INT_MAX - 255) return RK_NPU_ERR_PARAM;
    const int rc = rk_npu_attention_f16_query(&c->attention, 0, query_rows, 0, sizes);
    if (rc != RK_NPU_OK) return rc;
    const int cap = round_up(capacity, c->block);
    sizes->key_bytes = sizes->value_bytes = q8_code_bytes(*c, cap) + q8_scale_bytes(*c, cap) / 2;
    sizes->tail_bytes = 2 * q8_kept_bytes(*c);
    return RK_NPU_OK;
}

int rk_npu_hip_attention_q8_cache_create(rk_npu_iommu_domain* domain, const rk_npu_hip_attention_q8_config* config,
                                         rk_npu_hip_attention_q8_cache** out) {
    if (out) *out = nullptr;
    Domain* d = static_cast<Domain*>(domain);
    if (!d || !out || !valid_q8(config)) return RK_NPU_ERR_PARAM;
    if (!supported_dim(config->attention.head_dim)) return RK_NPU_ERR_UNSUPPORTED;
    DeviceGuard dev(device_of(d));
    if (!dev.ok) return RK_NPU_ERR_DEVICE;
    Q8Cache* c = new (std::nothrow) Q8Cache();
    if (!c) return RK_NPU_ERR_NOMEM;
    c->magic = MAGIC_Q8_CACHE;
    c->domain = d;
    c->cfg = *config;
    c->generation = 0;
    c->capacity = std::max(config->block, round_up(config->attention.initial_capacity, config->block));
    c->code_bytes = q8_code_bytes(c->cfg, c->capacity);
    c->scale_bytes = q8_scale_bytes(c->cfg, c->capacity);
    c->kept_bytes = q8_kept_bytes(c->cfg);
    c->codes[0] = c->codes[1] = nullptr;
    c->sc = nullptr;
    c->kept[1] = nullptr;
    c->kept[0] = static_cast<__half*>(domain_alloc(d, c->kept_bytes));
    if (c->kept[0]) c->kept[1] = static_cast<__half*>(domain_alloc(d, c->kept_bytes));
    if (!c->kept[1] || !q8_alloc(c, c->capacity, c->codes, c->sc)) {
        c->codes[0] = c->codes[1] = nullptr;
        rk_npu_hip_attention_q8_cache_free(reinterpret_cast<rk_npu_hip_attention_q8_cache*>(c));
        return RK_NPU_ERR_NOMEM;
    }
    *out = reinterpret_cast<rk_npu_hip_attention_q8_cache*>(c);
    return RK_NPU_OK;
}

void rk_npu_hip_attention_q8_cache_free(rk_npu_hip_attention_q8_cache* cache) {
    Q8Cache* c = as_q8(cache);
    if (!c) return;
    DeviceGuard dev(device_of(c->domain));
    (void)c->fence.wait(nullptr);
    c->fence.destroy();
    if (c->stream) {
        (void)hipStreamSynchronize(c->stream);
        (void)hipStreamDestroy(c->stream);
    }
    stage_release(c->hs);
    for (int i = 0; i < 2; ++i) {
        domain_free(c->domain, c->codes[i], c->code_bytes);
        domain_free(c->domain, c->kept[i], c->kept_bytes);
    }
    domain_free(c->domain, c->sc, c->scale_bytes);
    c->magic = 0;
    delete c;
}

int rk_npu_hip_attention_q8_cache_reserve(rk_npu_ctx* ctx, rk_npu_hip_attention_q8_cache* cache, int32_t capacity) {
    Q8Cache* c = as_q8(cache);
    if (!ctx || !c || capacity < 0) return RK_NPU_ERR_PARAM;
    std::lock_guard<std::shared_mutex> lock(c->mu);
    DeviceGuard dev(device_of(c->domain));
    if (!dev.ok || c->fence.wait(nullptr) != hipSuccess) return RK_NPU_ERR_DEVICE;
    return q8_grow(c, capacity);
}

int rk_npu_hip_attention_q8_cache_truncate(rk_npu_hip_attention_q8_cache* cache, int32_t length) {
    Q8Cache* c = as_q8(cache);
    if (!c) return RK_NPU_ERR_PARAM;
    std::lock_guard<std::shared_mutex> lock(c->mu);
    if (length < 0 || length > c->rows.length) return RK_NPU_ERR_PARAM;
    if (length < c->rows.length) c->rows.truncate(c->cfg.block, length);
    return RK_NPU_OK;
}

int rk_npu_hip_attention_q8_cache_get_info(const rk_npu_hip_attention_q8_cache* cache,
                                           rk_npu_attention_f16_cache_info* info) {
    Q8Cache* c = as_q8(cache);
    if (!c || !info) return RK_NPU_ERR_PARAM;
    std::shared_lock<std::shared_mutex> lock(c->mu);
    info->length = c->rows.length;
    info->capacity = c->capacity;
    info->max_capacity = q8_max_capacity(c);
    info->generation = c->generation;
    info->key_bytes = info->value_bytes = c->code_bytes + c->scale_bytes / 2;
    info->tail_bytes = 2 * c->kept_bytes;
    return RK_NPU_OK;
}

int rk_npu_hip_attention_q8_cache_load(rk_npu_ctx* ctx, rk_npu_hip_attention_q8_cache* cache, const uint16_t* k,
                                       const uint16_t* v, int32_t rows) {
    Q8Cache* c = as_q8(cache);
    if (!ctx || !c || rows < 0 || (rows > 0 && (!k || !v))) return RK_NPU_ERR_PARAM;
    std::lock_guard<std::shared_mutex> lock(c->mu);
    if (rows > q8_max_capacity(c)) return RK_NPU_ERR_PARAM;
    DeviceGuard dev(device_of(c->domain));
    if (!dev.ok || c->fence.wait(nullptr) != hipSuccess) return RK_NPU_ERR_DEVICE;
    c->rows = Q8Rows();
    c->generation += 1;  // the contents are replaced (a reset when rows == 0)
    if (rows == 0) return RK_NPU_OK;
    const int rc = q8_grow(c, rows);
    return rc != RK_NPU_OK ? rc : q8_put_host(c, k, v, rows);
}

int rk_npu_hip_attention_q8_cache_append(rk_npu_ctx* ctx, rk_npu_hip_attention_q8_cache* cache, const uint16_t* k,
                                         const uint16_t* v, int32_t rows) {
    Q8Cache* c = as_q8(cache);
    if (!ctx || !c || rows < 1 || !k || !v) return RK_NPU_ERR_PARAM;
    std::lock_guard<std::shared_mutex> lock(c->mu);
    const int most = q8_max_capacity(c);
    if (rows > most - c->rows.length) return RK_NPU_ERR_PARAM;
    DeviceGuard dev(device_of(c->domain));
    if (!dev.ok || c->fence.wait(nullptr) != hipSuccess) return RK_NPU_ERR_DEVICE;
    const int length = c->rows.length + rows;
    if (length > c->capacity) {
        const int rc = q8_grow(c, std::min(most, std::max(length, c->capacity > most / 2 ? most : 2 * c->capacity)));
        if (rc != RK_NPU_OK) return rc;
    }
    return q8_put_host(c, k, v, rows);
}

int rk_npu_hip_attention_q8_cache_read(rk_npu_ctx* ctx, rk_npu_hip_attention_q8_cache* cache, int32_t first,
                                       int32_t rows, uint16_t* k, uint16_t* v) {
    Q8Cache* c = as_q8(cache);
    if (!ctx || !c || first < 0 || rows < 1 || !k || !v) return RK_NPU_ERR_PARAM;
    std::lock_guard<std::shared_mutex> lock(c->mu);
    if (first > c->rows.length - rows) return RK_NPU_ERR_PARAM;
    DeviceGuard dev(device_of(c->domain));
    if (!dev.ok || c->fence.wait(nullptr) != hipSuccess) return RK_NPU_ERR_DEVICE;
    const int kh = c->cfg.attention.kv_heads, D = c->cfg.attention.head_dim, step = q8_stage_rows(c, rows);
    const size_t each = (size_t)kh * step * D;
    uint16_t* st = static_cast<uint16_t*>(q8_stage(c, 2 * each * sizeof(uint16_t)));
    if (!st) return RK_NPU_ERR_NOMEM;
    for (int r = 0; r < rows; r += step) {
        const int n = std::min(step, rows - r);
        uint16_t* to = static_cast<uint16_t*>(c->hs.dev);
        const int rc = q8_enqueue_read(c, first + r, n, HeadsView{to, 0, (long long)n * D, D},
                                       HeadsView{to + each, 0, (long long)n * D, D}, c->stream);
        if (rc != RK_NPU_OK) return rc;
        if (!q8_stage_done(c, st)) return RK_NPU_ERR_DEVICE;
        for (int g = 0; g < kh; ++g) {
            const size_t at = ((size_t)g * rows + r) * D, from = (size_t)g * n * D;
            std::memcpy(k + at, st + from, (size_t)n * D * sizeof(uint16_t));
            std::memcpy(v + at, st + each + from, (size_t)n * D * sizeof(uint16_t));
        }
    }
    return RK_NPU_OK;
}

int rk_npu_hip_attention_q8_run(rk_npu_ctx* ctx, rk_npu_attention_f16_workspace* workspace,
                                rk_npu_hip_attention_q8_cache* cache, const uint16_t* q, int32_t rows,
                                int32_t position, float* output, rk_npu_attention_f16_timings* timings) {
    if (!ctx) return RK_NPU_ERR_PARAM;
    return q8_run_host(workspace, cache, q, rows, position, output, false, timings);
}

int rk_npu_hip_attention_q8_run_half(rk_npu_ctx* ctx, rk_npu_attention_f16_workspace* workspace,
                                     rk_npu_hip_attention_q8_cache* cache, const uint16_t* q, int32_t rows,
                                     int32_t position, uint16_t* output, rk_npu_attention_f16_timings* timings) {
    if (!ctx) return RK_NPU_ERR_PARAM;
    return q8_run_host(workspace, cache, q, rows, position, output, true, timings);
}

int rk_npu_hip_attention_q8_device_append(rk_npu_hip_attention_q8_cache* cache, const rk_npu_hip_heads* k,
                                          const rk_npu_hip_heads* v, int32_t rows, void* stream) {
    Q8Cache* c = as_q8(cache);
    if (!c || rows < 1) return RK_NPU_ERR_PARAM;
    const int device = device_of(c->domain), kh = c->cfg.attention.kv_heads, D = c->cfg.attention.head_dim;
    if (!valid_heads(k, device, D, false, kh, rows) || !valid_heads(v, device, D, false, kh, rows))
        return RK_NPU_ERR_PARAM;
    std::lock_guard<std::shared_mutex> lock(c->mu);
    if (rows > c->capacity - c->rows.length) return RK_NPU_ERR_PARAM;  // (reserve first: no allocation here)
    DeviceGuard dev(device);
    if (!dev.ok) return RK_NPU_ERR_DEVICE;
    if (c->rows.open < 0 && c->rows.length % c->cfg.block) {
        // Continues from codes, which it replaces: a captured one could not be repeated.
        hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
        if (hipStreamIsCapturing(static_cast<hipStream_t>(stream), &st) != hipSuccess ||
            st != hipStreamCaptureStatusNone) {
            (void)hipGetLastError();
            return RK_NPU_ERR_UNSUPPORTED;
        }
    }
    const int rc = q8_enqueue_append(c, view_of(*k), view_of(*v), rows, static_cast<hipStream_t>(stream));
    if (rc == RK_NPU_OK) c->fence.note(static_cast<hipStream_t>(stream));
    return rc;
}

int rk_npu_hip_attention_q8_device_read(rk_npu_hip_attention_q8_cache* cache, int32_t first, int32_t rows,
                                        const rk_npu_hip_heads* k, const rk_npu_hip_heads* v, void* stream) {
    Q8Cache* c = as_q8(cache);
    if (!c || first < 0 || rows < 1 || (!k && !v)) return RK_NPU_ERR_PARAM;
    const int device = device_of(c->domain), kh = c->cfg.attention.kv_heads, D = c->cfg.attention.head_dim;
    if ((k && !valid_heads(k, device, D, true, kh, rows)) || (v && !valid_heads(v, device, D, true, kh, rows)))
        return RK_NPU_ERR_PARAM;
    std::lock_guard<std::shared_mutex> lock(c->mu);
    if (first > c->rows.length - rows) return RK_NPU_ERR_PARAM;
    DeviceGuard dev(device);
    if (!dev.ok) return RK_NPU_ERR_DEVICE;
    const HeadsView none{nullptr, 0, 0, 0};
    const int rc = q8_enqueue_read(c, first, rows, k ? view_of(*k) : none, v ? view_of(*v) : none,
                                   static_cast<hipStream_t>(stream));
    if (rc == RK_NPU_OK) c->fence.note(static_cast<hipStream_t>(stream));
    return rc;
}

int rk_npu_hip_attention_q8_device_run(rk_npu_attention_f16_workspace* workspace,
                                       rk_npu_hip_attention_q8_cache* cache, const rk_npu_hip_heads* q, int32_t rows,
                                       int32_t position, const rk_npu_hip_heads* out, void* stream) {
    AttnWork* w = as_attn_work(workspace);
    Q8Cache* c = as_q8(cache);
    if (!w || !c || rows < 1 || rows > w->cfg.max_query_rows || !same_geometry(w, c)) return RK_NPU_ERR_PARAM;
    const int device = device_of(c->domain), qh = c->cfg.attention.query_heads, D = c->cfg.attention.head_dim;
    if (!valid_heads(q, device, D, false, qh, rows) || !valid_heads(out, device, D, true, qh, rows))
        return RK_NPU_ERR_PARAM;
    std::shared_lock<std::shared_mutex> lock(c->mu);
    DeviceGuard dev(device);
    if (!dev.ok) return RK_NPU_ERR_DEVICE;
    const int rc = q8_enqueue_run(w, c, view_of(*q), rows, position, view_of(*out), static_cast<hipStream_t>(stream));
    if (rc == RK_NPU_OK) {
        c->fence.note(static_cast<hipStream_t>(stream));
        w->fence.note(static_cast<hipStream_t>(stream));
    }
    return rc;
}

}  // extern "C"
