// xestrata-win_amd/csrc/xs_block.h - what block_norm.hip and w8a8.hip share: the types of float rows, the int8 rule, and
// the entry points' argument checks (include/xs_block.h).
#pragma once

#include "../../include/xs_block.h"
#include "../../include/xs_moe.h"
#include "xs_device.h"
#include "xs_error.h"
#include "xs_kernels.h"

#include <cstdarg>
#include <cstdio>
#include <type_traits>

namespace xs {

__host__ __device__ constexpr int float_bytes(int t) { return t == XS_F32 ? 4 : 2; }

// ---------------------------------------------------------------- the int8 rule
// The scale of a row whose largest |v| has the bits `amax`: never under the smallest normal number, so that 1 / s is finite
// and a code's product with it exact; NaN where the row holds an infinity or a NaN (their bits are the largest of all).  The
// product with the rounded 1 / 127 (0.06 steps off at most) is within 0.57 steps of the quotient, where a division is within 0.5
// (4.7% of the scales differ by one step); it is how the q8_1 rows take theirs.  What the codes stand for is as near either way:
// they are the nearest to v / s for the s that is stored, and the largest |v| / s is within 127 (1 + 2^-23), which is 127.
__device__ __forceinline__ float int8_scale(uint32_t amax) {
    if (amax >= 0x7F800000u) return u2f(0x7FC00000u);
    return fmaxf(u2f(amax) * (1.0f / 127.0f), 1.17549435e-38f);
}
// The integer nearest v / s, halves to even.  v times the rounded 1 / s is within one of it; the remainder v - q s that says
// which way it is off is a multiple of the last place of v or of s, whichever is less, and so small that the fused
// multiply-add gives it exactly where it is near s / 2 (doubled, so that half of the smallest s needs no bit below 2^-149).
__device__ __forceinline__ int int8_code(float v, float s, float inv) {
    float q = rintf(v * inv);
    const float r2 = 2.0f * __builtin_fmaf(-q, s, v);
    const bool odd = ((int)q & 1) != 0;
    if (r2 > s || (r2 == s && odd)) q += 1.0f;
    if (r2 < -s || (r2 == -s && odd)) q -= 1.0f;
    return (int)q;
}

// ---------------------------------------------------------------- float rows
// Value (i, j) of a thread is at (i n_threads + tid) 8 + j (VEC: 16- and 32-byte accesses; the row's start is aligned and its
// length a multiple of 8) or at (8 i + j) n_threads + tid (any row: neighbouring lanes, neighbouring values).
template <bool VEC>
__device__ __forceinline__ int value_at(int i, int j, int tid, int n_threads) {
    return VEC ? (i * n_threads + tid) * 8 + j : (8 * i + j) * n_threads + tid;
}

// the row's words as they are in memory; they become floats (row_floats) where they are used, so that nothing waits before
template <int CH>
struct RowWords {
    uint32_t w[CH][8];
};
template <int CH, bool VEC>
__device__ __forceinline__ void load_row(RowWords<CH>& r, const void* row, int type, int n, int tid, int nt) {
#pragma unroll
    for (int i = 0; i < CH; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) r.w[i][j] = 0;
    if (type == XS_F32) {
        const uint32_t* p = (const uint32_t*)row;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            if (VEC) {
                const int c = value_at<true>(i, 0, tid, nt);
                if (c < n) {
                    const uint4 a = *(const uint4*)(p + c), b = *(const uint4*)(p + c + 4);
                    r.w[i][0] = a.x, r.w[i][1] = a.y, r.w[i][2] = a.z, r.w[i][3] = a.w;
                    r.w[i][4] = b.x, r.w[i][5] = b.y, r.w[i][6] = b.z, r.w[i][7] = b.w;
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int c = value_at<false>(i, j, tid, nt);
                    if (c < n) r.w[i][j] = p[c];
                }
            }
        }
    } else {
        const uint16_t* p = (const uint16_t*)row;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            if (VEC) {
                const int c = value_at<true>(i, 0, tid, nt);
                if (c < n) {
                    const uint4 a = *(const uint4*)(p + c);
                    r.w[i][0] = a.x, r.w[i][1] = a.y, r.w[i][2] = a.z, r.w[i][3] = a.w;
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int c = value_at<false>(i, j, tid, nt);
                    if (c < n) r.w[i][j] = p[c];
                }
            }
        }
    }
}
// two floats to the two halves of a word, to nearest even (v_cvt_pk_bf16_f32 / v_cvt_f16_f32)
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
template <int TYPE>
__device__ __forceinline__ uint32_t to_halves(float a, float b) {
    if (TYPE == XS_BF16) return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t){a, b}, bf16x2_t));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t){a, b}, f16x2_t));
}
template <int TYPE>
__device__ __forceinline__ float from_half(uint32_t v) {   // the low 16 bits
    return TYPE == XS_BF16 ? u2f(v << 16) : h2f((uint16_t)v);
}
// f with the type as a constant (the branch is uniform and outside the loops over a row's values)
template <typename F>
__device__ __forceinline__ void by_type(int type, F&& f) {
    if (type == XS_F32)
        f(std::integral_constant<int, XS_F32>{});
    else if (type == XS_BF16)
        f(std::integral_constant<int, XS_BF16>{});
    else
        f(std::integral_constant<int, XS_F16>{});
}
template <int CH, bool VEC>
__device__ __forceinline__ void row_floats(float (&v)[CH][8], const RowWords<CH>& r, int type) {
    by_type(type, [&](auto tc) {
        constexpr int T = decltype(tc)::value;
#pragma unroll
        for (int i = 0; i < CH; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (T == XS_F32)
                    v[i][j] = u2f(r.w[i][j]);
                else
                    v[i][j] = from_half<T>(!VEC ? r.w[i][j] : (j & 1) ? r.w[i][j / 2] >> 16 : r.w[i][j / 2]);
            }
    });
}
// the values as a row of the type would hold them
template <int CH>
__device__ __forceinline__ void round_row(float (&v)[CH][8], int type) {
    if (type == XS_F32) return;
    by_type(type, [&](auto tc) {
        constexpr int T = decltype(tc)::value;
        if (T == XS_F32) return;
#pragma unroll
        for (int i = 0; i < CH; ++i)
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const uint32_t w = to_halves<T>(v[i][j], v[i][j + 1]);
                v[i][j] = from_half<T>(w), v[i][j + 1] = from_half<T>(w >> 16);
            }
    });
}
template <int CH, bool VEC>
__device__ __forceinline__ void store_row(void* row, int type, const float (&v)[CH][8], int n, int tid, int nt) {
    by_type(type, [&](auto tc) {
        constexpr int T = decltype(tc)::value;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int c0 = value_at<VEC>(i, 0, tid, nt);
            if (VEC && c0 >= n) continue;
            if (VEC && T == XS_F32) {
                float* p = (float*)row + c0;
                *(float4*)p = make_float4(v[i][0], v[i][1], v[i][2], v[i][3]);
                *(float4*)(p + 4) = make_float4(v[i][4], v[i][5], v[i][6], v[i][7]);
            } else if (VEC) {
                *(uint4*)((uint16_t*)row + c0) = make_uint4(to_halves<T>(v[i][0], v[i][1]), to_halves<T>(v[i][2], v[i][3]),
                                                            to_halves<T>(v[i][4], v[i][5]), to_halves<T>(v[i][6], v[i][7]));
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int c = value_at<false>(i, j, tid, nt);
                    if (c >= n) continue;
                    if (T == XS_F32)
                        ((float*)row)[c] = v[i][j];
                    else
                        ((uint16_t*)row)[c] = (uint16_t)to_halves<T>(v[i][j], v[i][j]);
                }
            }
        }
    });
}
template <int CH, bool VEC>
__device__ __forceinline__ void store_codes(int8_t* row, const float (&v)[CH][8], float s, int n, int tid, int nt) {
    const bool good = s == s;
    const float inv = good ? 1.0f / s : 0.0f;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        int q[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) q[j] = good ? int8_code(v[i][j], s, inv) : 0;
        if (VEC) {
            const int c = value_at<true>(i, 0, tid, nt);
            uint32_t w[2];
#pragma unroll
            for (int j = 0; j < 2; ++j)
                w[j] = (uint32_t)(uint8_t)q[4 * j] | (uint32_t)(uint8_t)q[4 * j + 1] << 8 |
                       (uint32_t)(uint8_t)q[4 * j + 2] << 16 | (uint32_t)(uint8_t)q[4 * j + 3] << 24;
            if (c < n) *(uint2*)(row + c) = make_uint2(w[0], w[1]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int c = value_at<false>(i, j, tid, nt);
                if (c < n) row[c] = (int8_t)q[j];
            }
        }
    }
}

// sums and maxima over the row's NW waves (NW 1: one wave a row); `slots`: NW words of LDS of this reduction's own
template <int NW>
__device__ __forceinline__ double row_sum(double v, double* slots, int wave) {
    v = wave_sum_d(v);
    if (NW == 1) return v;
    if ((threadIdx.x & 63) == 0) slots[wave] = v;
    __syncthreads();
    v = 0.0;
#pragma unroll
    for (int i = 0; i < NW; ++i) v += slots[i];
    return v;
}
template <int NW>
__device__ __forceinline__ uint32_t row_max_bits(uint32_t v, uint32_t* slots, int wave) {
    v = wave_max_u32(v);
    if (NW == 1) return v;
    if ((threadIdx.x & 63) == 0) slots[wave] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) v = max(v, slots[i]);
    return v;
}
template <int CH>
__device__ __forceinline__ uint32_t thread_max_bits(const float (&v)[CH][8]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < CH; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max(m, f2u(v[i][j]) & 0x7FFFFFFFu);
    return m;
}

// ---------------------------------------------------------------- argument checks
namespace block {
inline int fail(int code, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    std::vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    return set_error(code, buf);
}
// after a launch; a NULL stream: the default stream, then a wait
inline int finish(void* stream, hipError_t e, const char* what) {
    if (e == hipSuccess && !stream) e = hipStreamSynchronize(nullptr);
    return e == hipSuccess ? XS_OK : fail(XS_EDEVICE, "%s: %s", what, hipGetErrorString(e));
}
inline bool is_float_type(int t) { return t == XS_F32 || t == XS_F16 || t == XS_BF16; }
inline bool aligned(const void* p, size_t a) { return p && (uintptr_t)p % a == 0; }

constexpr int64_t kMaxRows = 1ll << 21, kMaxLd = 1ll << 31;   // (a grid's threads are counted in 32 bits)

struct Span {   // rows `row` bytes long and `stride` bytes apart (0: one piece), `bytes` from the first's start to the last's end
    const void* p;
    uint64_t bytes, stride = 0, row = 0;
};
inline Span rows_span(const void* p, int64_t rows, int64_t ld, int64_t n, int bytes) {
    return {p, ((uint64_t)(rows - 1) * (uint64_t)ld + (uint64_t)n) * (uint64_t)bytes, (uint64_t)ld * (uint64_t)bytes,
            (uint64_t)n * (uint64_t)bytes};
}
// Rows of one stride that lie between each other's (columns of one buffer) do not overlap; else spans that meet do.
inline bool overlap(const Span& a, const Span& b) {
    const auto x = (uintptr_t)a.p, y = (uintptr_t)b.p;
    if (!a.p || !b.p || x >= y + b.bytes || y >= x + a.bytes) return false;
    if (a.stride == 0 || a.stride != b.stride) return true;
    const uint64_t after = (y >= x ? y - x : a.stride - (x - y) % a.stride) % a.stride;   // b's rows' starts behind a's
    return after < a.row || after + b.row > a.stride;
}
// float rows: `type`, `ld`, alignment
inline int check_rows(const char* what, const char* name, const void* p, int type, int64_t ld, int64_t n) {
    if (!is_float_type(type)) return fail(XS_EINVAL, "%s: %s has type %d (F32 0, F16 1, BF16 30)", what, name, type);
    if (!aligned(p, (size_t)float_bytes(type))) return fail(XS_EINVAL, "%s: %s is missing or misaligned", what, name);
    if (ld < n || ld > kMaxLd) return fail(XS_EINVAL, "%s: %s has %lld values a row, %lld apart", what, name, (long long)n, (long long)ld);
    return XS_OK;
}
inline int check_codes(const char* what, const int8_t* q, int64_t ldq, const float* scale, int64_t n) {
    if (!q || !aligned(scale, 4)) return fail(XS_EINVAL, "%s: the int8 rows need both codes and scales (4-byte aligned)", what);
    if (ldq < n || ldq > kMaxLd) return fail(XS_EINVAL, "%s: int8 rows of %lld values, %lld bytes apart", what, (long long)n, (long long)ldq);
    return XS_OK;
}
// no output overlaps an input or another output (null spans never do)
template <int NO, int NI>
int check_overlap(const char* what, const Span (&out)[NO], const Span (&in)[NI]) {
    for (int i = 0; i < NO; ++i) {
        for (int j = 0; j < NI; ++j)
            if (overlap(out[i], in[j])) return fail(XS_EINVAL, "%s: an output overlaps an input", what);
        for (int j = 0; j < i; ++j)
            if (overlap(out[i], out[j])) return fail(XS_EINVAL, "%s: two outputs overlap", what);
    }
    return XS_OK;
}
inline bool vec_rows(const void* p, int64_t ld, int bytes, int unit) {   // every row's start `unit`-byte aligned (NULL: yes)
    return !p || ((uintptr_t)p % (size_t)unit == 0 && (uint64_t)ld * (uint64_t)bytes % (uint64_t)unit == 0);
}
}  // namespace block
}  // namespace xs
