// xestrata-win_amd/csrc/block_norm.hip - the norm before a block and the join after one (include/xs_block.h).
//
//   norm   y = fl(fl(x r) w), r = fl(1 / sqrt(sum x^2 / n + eps)), the sum and the root in 64 bits
//   join   b = the block's output (or the weighted parts, summed as combine.hip does but for a shared gate's
//          sigmoid, which is taken in 64 bits here); b = norm(b); b = fl(b g);
//          out = fl(fl(rs residual) + fl(bs b)); next = norm(out as stored), its int8 rows beside it
//
// Bound by memory: each row is read once into registers, 8 values a thread and step (16- or 32-byte accesses), normed there
// and written once.  The squares are summed in 64 bits and r is rounded to 24, so that another order of the sum, which moves it by
// some 2^-53, moves r's last bit once in 10^8 rows.  The order goes by how a row is split over lanes (pick_split): for rows that
// 16-byte accesses take, by their length alone, so that a token's result, int8 codes included, is the same in every batch, and up
// to 4096 values in norms and joins alike (a wave's sum is that of 512 neighbouring values, the waves' are added in turn).  The
// 64-bit adds are two a value beside 4 or more bytes of memory traffic a value.
#include "xs_block.h"

#include <type_traits>

namespace xs {

struct NormArgs {
    const void* x;
    const float* w;
    void* y;
    int8_t* q;
    float* q_scale;
    int64_t ldx, ldy, ldq, n_tok;
    int x_type, y_type, n;
    float eps;
    double inv_n;
};

struct JoinArgs {
    xs_block_join_cfg_t j;
    const void* y;        // the block's rows, or
    const float* parts;   // k rows a token with their weights, a shared row and its gate
    const float* weights;
    const float* shared;
    const float* shared_gate;
    const void* residual;
    void* out;
    void* next;
    int8_t* q;
    float* q_scale;
    int64_t ldy, ldr, ld_next, ldq, n_tok;
    int y_type, r_type, next_type, n, k;
    double inv_n;
};

// the squares' sum of a thread's values in 64 bits (each square is exact there)
template <int CH>
__device__ __forceinline__ double squares(const float (&v)[CH][8]) {
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < CH; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) s = __builtin_fma((double)v[i][j], (double)v[i][j], s);
    return s;
}
// 1 / sqrt(ss / n + eps): the hardware's estimate (about 24 bits) with one step of third order, which leaves 64-bit rounding
// (a division and a root of the library's take some 100 dependent instructions more, twice a row in the join)
__device__ __forceinline__ float norm_factor(double ss, double inv_n, float eps) {
    const double m = __builtin_fma(ss, inv_n, (double)eps), y = __builtin_amdgcn_rsq(m);
    const double e = __builtin_fma(-m * y, y, 1.0);
    const double r = __builtin_fma(y * e, __builtin_fma(e, 0.375, 0.5), y);
    return (float)(m < __builtin_inf() ? r : y);   // (an infinite sum: 0; a NaN: NaN)
}
template <int CH, bool VEC>
__device__ __forceinline__ void apply_norm(float (&v)[CH][8], float r, bool weighted, const RowWords<CH>& w) {
    float wf[CH][8];
    row_floats<CH, VEC>(wf, w, XS_F32);
#pragma unroll
    for (int i = 0; i < CH; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[i][j] = v[i][j] * r;
            if (weighted) v[i][j] = v[i][j] * wf[i][j];
        }
}
// 1 / (1 + exp(-z)) in 64 bits, rounded once
__device__ __forceinline__ float sigmoid64(float z) { return (float)(1.0 / (1.0 + exp(-(double)z))); }

template <int NW, int CH, bool VEC>
__global__ __launch_bounds__(NW == 1 ? 256 : 64 * NW) void block_norm_kernel(const NormArgs a) {
    __shared__ double sums[NW];
    __shared__ uint32_t tops[NW];
    constexpr int NT = 64 * NW;
    const int wave = threadIdx.x >> 6, tid = NW == 1 ? threadIdx.x & 63 : threadIdx.x;
    const int64_t t = NW == 1 ? (int64_t)blockIdx.x * 4 + wave : blockIdx.x;
    if (t >= a.n_tok) return;
    RowWords<CH> xw, ww;
    load_row<CH, VEC>(xw, (const uint8_t*)a.x + t * a.ldx * float_bytes(a.x_type), a.x_type, a.n, tid, NT);
    if (a.w) load_row<CH, VEC>(ww, a.w, XS_F32, a.n, tid, NT);
    float v[CH][8];
    row_floats<CH, VEC>(v, xw, a.x_type);
    const double ss = row_sum<NW>(squares(v), sums, wave);
    apply_norm<CH, VEC>(v, norm_factor(ss, a.inv_n, a.eps), a.w != nullptr, ww);
    if (a.y) store_row<CH, VEC>((uint8_t*)a.y + t * a.ldy * float_bytes(a.y_type), a.y_type, v, a.n, tid, NT);
    if (a.q) {
        const float s = int8_scale(row_max_bits<NW>(thread_max_bits(v), tops, wave));
        store_codes<CH, VEC>(a.q + t * a.ldq, v, s, a.n, tid, NT);
        if (tid == 0) a.q_scale[t] = s;
    }
}

template <int NW, int CH, bool VEC, bool PARTS>
__global__ __launch_bounds__(NW == 1 ? 256 : 64 * NW) void block_join_kernel(const JoinArgs a) {
    __shared__ double sums[2][NW];
    __shared__ uint32_t tops[NW];
    constexpr int NT = 64 * NW;
    const int wave = threadIdx.x >> 6, tid = NW == 1 ? threadIdx.x & 63 : threadIdx.x;
    const int64_t t = NW == 1 ? (int64_t)blockIdx.x * 4 + wave : blockIdx.x;
    if (t >= a.n_tok) return;
    const bool next = a.next || a.q;
    const int rb = float_bytes(a.r_type);
    RowWords<CH> rw, nw, gw, bw;
    float b[CH][8];
    float token_gate = 0.0f, shared_gate = 0.0f;   // (asked for first, taken to their sigmoids while the rows are on their way)
    if (a.j.gate_kind == XS_GATE_TOKEN) token_gate = a.j.gate[t];
    if (PARTS && a.shared_gate) shared_gate = a.shared_gate[t];
    if (!PARTS) load_row<CH, VEC>(bw, (const uint8_t*)a.y + t * a.ldy * float_bytes(a.y_type), a.y_type, a.n, tid, NT);
    load_row<CH, VEC>(rw, (const uint8_t*)a.residual + t * a.ldr * rb, a.r_type, a.n, tid, NT);
    RowWords<CH> ow;
    if (a.j.gate_kind >= XS_GATE_CHANNEL)
        load_row<CH, VEC>(gw, a.j.gate + (a.j.gate_kind == XS_GATE_VALUE ? t * a.j.ld_gate : 0), XS_F32, a.n, tid, NT);
    if (a.j.norm && a.j.norm_w) load_row<CH, VEC>(ow, a.j.norm_w, XS_F32, a.n, tid, NT);
    if (next && a.j.next_w) load_row<CH, VEC>(nw, a.j.next_w, XS_F32, a.n, tid, NT);
    if (a.j.gate_kind == XS_GATE_TOKEN) token_gate = sigmoid64(token_gate);
    if (PARTS && a.shared_gate) shared_gate = sigmoid64(shared_gate);
    if (PARTS) {
        const float* p = a.parts + t * a.k * a.n;
        const float* w = a.weights + t * a.k;
        constexpr int kAhead = CH == 1 ? 8 : NW == 16 ? 1 : 2;   // parts in flight (16 waves: 128 registers a lane)
        for (int e0 = 0; e0 < a.k; e0 += kAhead) {
            RowWords<CH> pw[kAhead];
            float we[kAhead];
#pragma unroll
            for (int e = 0; e < kAhead; ++e)
                if (e0 + e < a.k) {
                    load_row<CH, VEC>(pw[e], p + (int64_t)(e0 + e) * a.n, XS_F32, a.n, tid, NT);
                    we[e] = w[e0 + e];
                }
#pragma unroll
            for (int e = 0; e < kAhead; ++e)
                if (e0 + e < a.k) {
#pragma unroll
                    for (int i = 0; i < CH; ++i)
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const float prod = u2f(pw[e].w[i][j]) * we[e];
                            b[i][j] = e0 + e == 0 ? prod : b[i][j] + prod;
                        }
                }
        }
        if (a.shared) {
            RowWords<CH> sw;
            load_row<CH, VEC>(sw, a.shared + t * a.n, XS_F32, a.n, tid, NT);
#pragma unroll
            for (int i = 0; i < CH; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float s = u2f(sw.w[i][j]);
                    b[i][j] = b[i][j] + (a.shared_gate ? s * shared_gate : s);
                }
        }
    } else {
        row_floats<CH, VEC>(b, bw, a.y_type);
    }
    if (a.j.norm) {
        const double ss = row_sum<NW>(squares(b), sums[0], wave);
        apply_norm<CH, VEC>(b, norm_factor(ss, a.inv_n, a.j.norm_eps), a.j.norm_w != nullptr, ow);
    }
    if (a.j.gate_kind == XS_GATE_TOKEN) {
#pragma unroll
        for (int i = 0; i < CH; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) b[i][j] = b[i][j] * token_gate;
    } else if (a.j.gate_kind != XS_GATE_NONE) {
#pragma unroll
        for (int i = 0; i < CH; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) b[i][j] = b[i][j] * u2f(gw.w[i][j]);
    }
    float r[CH][8];
    row_floats<CH, VEC>(r, rw, a.r_type);
#pragma unroll
    for (int i = 0; i < CH; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float rs = a.j.residual_scale * r[i][j], bs = a.j.branch_scale * b[i][j];
            r[i][j] = rs + bs;
        }
    round_row(r, a.r_type);   // as it is stored
    store_row<CH, VEC>((uint8_t*)a.out + t * a.ldr * rb, a.r_type, r, a.n, tid, NT);
    if (!next) return;
    const double ss = row_sum<NW>(squares(r), sums[1], wave);
    apply_norm<CH, VEC>(r, norm_factor(ss, a.inv_n, a.j.next_eps), a.j.next_w != nullptr, nw);
    if (a.next) store_row<CH, VEC>((uint8_t*)a.next + t * a.ld_next * float_bytes(a.next_type), a.next_type, r, a.n, tid, NT);
    if (a.q) {
        const float s = int8_scale(row_max_bits<NW>(thread_max_bits(r), tops, wave));
        store_codes<CH, VEC>(a.q + t * a.ldq, r, s, a.n, tid, NT);
        if (tid == 0) a.q_scale[t] = s;
    }
}

// Rows of any length up to 65536 to int8 rows.  Bound by memory; past 32768 values a row's 64 values a thread take all of 128
// registers and spill 2 to 4 (4096 x 65536 fp32 302 us, 4.4 TB/s; bf16 219 us; 4096 x 7168 26.2 us, 5.6 TB/s).
struct QuantArgs {
    const void* x;
    int8_t* q;
    float* q_scale;
    int64_t ldx, ldq, rows;
    int x_type, n;
};
template <int NW, int CH, bool VEC>
__global__ __launch_bounds__(NW == 1 ? 256 : 64 * NW) void w8a8_quantize_kernel(const QuantArgs a) {
    __shared__ uint32_t tops[NW];
    constexpr int NT = 64 * NW;
    const int wave = threadIdx.x >> 6, tid = NW == 1 ? threadIdx.x & 63 : threadIdx.x;
    const int64_t t = NW == 1 ? (int64_t)blockIdx.x * 4 + wave : blockIdx.x;
    if (t >= a.rows) return;
    RowWords<CH> xw;
    load_row<CH, VEC>(xw, (const uint8_t*)a.x + t * a.ldx * float_bytes(a.x_type), a.x_type, a.n, tid, NT);
    float v[CH][8];
    row_floats<CH, VEC>(v, xw, a.x_type);
    const float s = int8_scale(row_max_bits<NW>(thread_max_bits(v), tops, wave));
    store_codes<CH, VEC>(a.q + t * a.ldq, v, s, a.n, tid, NT);
    if (tid == 0) a.q_scale[t] = s;
}

namespace {

template <int N>
using Int = std::integral_constant<int, N>;

// How a row is split: 8 values a thread, so that every row a call reads is asked for at once; past 4096 values 16, whose
// work-groups are smaller.  Measured (norm of fp32 rows to bf16, join with norms on both sides, us): 2048 x 2048 7.1, 12.4 with 8
// values a thread, 7.7, 15.0 with 16, 9.8, 20.6 with 32; 2048 x 4096 10.9, 24.9 / 11.3, 26.1 / 12.5, 32.4; 1024 x 7168 11.2, 23.6 /
// 10.5, 24.8 / 12.6, 27.1; one row of 2048 2.5, 4.4 / 4.0, 4.6 / 4.3, 5.8.
// Rows of 16-byte accesses (VEC) are split the same in a call of any number of rows, so that their sums have one order; few rows
// past 4096 values gain by it more than they lose (norm, join, join of 8 parts with 16 values a thread / 8: 7 x 7168 3.07, 4.54,
// 7.8 / 3.08, 4.67, 8.2; 1 x 5120 2.79, 4.05, 6.8 / 2.75, 4.18, 6.4; 511 x 8192 7.07, 16.4, 38.8 / 6.78, 15.8, 39.7).  Others, one
// value an access, take 8 values a thread below 512 rows (7 x 5121 3.39, 5.68, 8.2 / 3.70, 6.35, 10.4 with 16; 4096 x 5121 norm to
// bf16 27.9 / 22.0), and so do int8 rows, whose maximum has no order.
// TRIM, the waves that a row needs instead of the next power of two: 2 for norms and int8 rows (4096 x 2560, 5 waves / 8: norm to
// int8 14.1 / 18.0, int8 rows 11.0 / 13.4; 4096 x 5120, 5 waves with 16 values a thread / 8: 22.2 / 28.0, 18.4 / 21.2); 1, up to
// 4096 values, for a join of rows (bf16, 4096 x 2560 17.0 / 19.8, but 4096 x 5120 46.9 / 39.7); 0 for a join of parts, whose many
// loads want the lanes (1024 x 2560 24.1 / 22.8, 1024 x 6144 52.5 / 49.0).
template <int TRIM, typename F>
hipError_t pick_split(bool one_order, int64_t rows, int n, F&& launch) {
    if (n <= 512) return launch(Int<1>{}, Int<1>{});
    if (n <= 1024) return launch(Int<2>{}, Int<1>{});
    if constexpr (TRIM > 0) {
        if (n <= 1536) return launch(Int<3>{}, Int<1>{});
    }
    if (n <= 2048) return launch(Int<4>{}, Int<1>{});
    if constexpr (TRIM > 0) {
        if (n <= 2560) return launch(Int<5>{}, Int<1>{});
        if (n <= 6 * 512) return launch(Int<6>{}, Int<1>{});
        if (n <= 3584) return launch(Int<7>{}, Int<1>{});
    }
    if (n <= 4096) return launch(Int<8>{}, Int<1>{});
    if (n > 8192) return launch(Int<16>{}, Int<2>{});
    if (!one_order && rows < 512) return launch(Int<16>{}, Int<1>{});
    if constexpr (TRIM > 1) {
        if (n <= 5120) return launch(Int<5>{}, Int<2>{});
        if (n <= 6144) return launch(Int<6>{}, Int<2>{});
        if (n <= 7168) return launch(Int<7>{}, Int<2>{});
    }
    return launch(Int<8>{}, Int<2>{});
}
template <int NW>
dim3 row_grid(int64_t rows) {
    return dim3((unsigned)(NW == 1 ? (rows + 3) / 4 : rows));
}
template <int NW>
dim3 row_block() {
    return dim3(NW == 1 ? 256 : 64 * NW);
}

hipError_t launch_norm(const NormArgs& a, bool vec, hipStream_t s) {
    return pick_split<2>(vec, a.n_tok, a.n, [&](auto nw, auto ch) {
        constexpr int NW = decltype(nw)::value, CH = decltype(ch)::value;
        if (vec)
            hipLaunchKernelGGL((block_norm_kernel<NW, CH, true>), row_grid<NW>(a.n_tok), row_block<NW>(), 0, s, a);
        else
            hipLaunchKernelGGL((block_norm_kernel<NW, CH, false>), row_grid<NW>(a.n_tok), row_block<NW>(), 0, s, a);
        return hipGetLastError();
    });
}
template <bool PARTS>
hipError_t launch_join(const JoinArgs& a, bool vec, hipStream_t s) {
    return pick_split<PARTS ? 0 : 1>(vec, a.n_tok, a.n, [&](auto nw, auto ch) {
        constexpr int NW = decltype(nw)::value, CH = decltype(ch)::value;
        if (vec)
            hipLaunchKernelGGL((block_join_kernel<NW, CH, true, PARTS>), row_grid<NW>(a.n_tok), row_block<NW>(), 0, s, a);
        else
            hipLaunchKernelGGL((block_join_kernel<NW, CH, false, PARTS>), row_grid<NW>(a.n_tok), row_block<NW>(), 0, s, a);
        return hipGetLastError();
    });
}
hipError_t launch_quantize(const QuantArgs& a, bool vec, hipStream_t s) {
    auto go = [&](auto nw, auto ch) {
        constexpr int NW = decltype(nw)::value, CH = decltype(ch)::value;
        if (vec)
            hipLaunchKernelGGL((w8a8_quantize_kernel<NW, CH, true>), row_grid<NW>(a.rows), row_block<NW>(), 0, s, a);
        else
            hipLaunchKernelGGL((w8a8_quantize_kernel<NW, CH, false>), row_grid<NW>(a.rows), row_block<NW>(), 0, s, a);
        return hipGetLastError();
    };
    if (a.n <= 16384) return pick_split<2>(false, a.rows, a.n, go);
    if (a.n <= 32768) return go(Int<16>{}, Int<4>{});
    return go(Int<16>{}, Int<8>{});
}

constexpr int64_t kMaxNormRow = 16384, kMaxInt8Row = 65536;

// the checks that every entry point of rows makes first; 1: nothing to do
int check_sizes(const char* what, int64_t rows, int64_t n, int64_t most) {
    if (rows <= 0) return -1;
    if (rows > block::kMaxRows) return block::fail(XS_EINVAL, "%s: %lld rows", what, (long long)rows);
    if (n < 1 || n > most)
        return block::fail(XS_EINVAL, "%s: rows of %lld values (1 .. %lld)", what, (long long)n, (long long)most);
    return XS_OK;
}
bool good_eps(float e) { return e >= 0.0f && e < 3.4e38f; }

// the parts common to xs_block_join and xs_moe_combine_join, with a->y or a->parts filled in
int join_common(const char* what, JoinArgs* a, void* stream) {
    using namespace block;
    const xs_block_join_cfg_t& j = a->j;
    const int64_t n = a->n, T = a->n_tok;
    const bool next = a->next || a->q;
    if (int r = check_rows(what, "residual", a->residual, a->r_type, a->ldr, n)) return r;
    if (int r = check_rows(what, "out", a->out, a->r_type, a->ldr, n)) return r;
    if (a->next)
        if (int r = check_rows(what, "next", a->next, a->next_type, a->ld_next, n)) return r;
    if (a->q || a->q_scale)
        if (int r = check_codes(what, a->q, a->ldq, a->q_scale, n)) return r;
    if (j.norm != 0 && j.norm != 1) return fail(XS_EINVAL, "%s: norm %d (0 or 1)", what, j.norm);
    if ((j.norm && !good_eps(j.norm_eps)) || (next && !good_eps(j.next_eps)))
        return fail(XS_EINVAL, "%s: an eps is negative or not finite", what);
    if ((j.norm_w && !aligned(j.norm_w, 4)) || (j.next_w && !aligned(j.next_w, 4)))
        return fail(XS_EINVAL, "%s: misaligned norm weights", what);
    if (j.gate_kind < XS_GATE_NONE || j.gate_kind > XS_GATE_VALUE)
        return fail(XS_EINVAL, "%s: gate kind %d", what, j.gate_kind);
    if (j.gate_kind != XS_GATE_NONE && !aligned(j.gate, 4)) return fail(XS_EINVAL, "%s: the gate is missing or misaligned", what);
    if (j.gate_kind == XS_GATE_VALUE && (j.ld_gate < n || j.ld_gate > kMaxLd))
        return fail(XS_EINVAL, "%s: gate rows of %lld values, %lld apart", what, (long long)n, (long long)j.ld_gate);
    const Span none{nullptr, 0};
    const int rb = float_bytes(a->r_type), yb = float_bytes(a->y_type), nb = float_bytes(a->next_type);
    const Span out = rows_span(a->out, T, a->ldr, n, rb), res = rows_span(a->residual, T, a->ldr, n, rb);
    const Span y = a->y ? rows_span(a->y, T, a->ldy, n, yb) : none;
    const Span nx = a->next ? rows_span(a->next, T, a->ld_next, n, nb) : none;
    const Span q = a->q ? rows_span(a->q, T, a->ldq, n, 1) : none, qs = {a->q_scale, 4 * (uint64_t)T};
    const Span gate = j.gate_kind == XS_GATE_NONE ? none
                      : j.gate_kind == XS_GATE_VALUE ? rows_span(j.gate, T, j.ld_gate, n, 4)
                                                     : Span{j.gate, 4 * (uint64_t)(j.gate_kind == XS_GATE_TOKEN ? T : n)};
    const Span nw{j.norm ? j.norm_w : nullptr, 4 * (uint64_t)n}, xw{next ? j.next_w : nullptr, 4 * (uint64_t)n};
    const Span parts = a->parts ? rows_span(a->parts, T * a->k, n, n, 4) : none, wt{a->weights, 4 * (uint64_t)(T * a->k)};
    const Span sh = a->shared ? rows_span(a->shared, T, n, n, 4) : none, sg{a->shared_gate, 4 * (uint64_t)T};
    const bool in_place = a->out == a->residual;
    const bool over_y = a->next && a->next == a->y && a->next_type == a->y_type && a->ld_next == a->ldy;
    if (int r = check_overlap<4, 9>(what, {out, nx, q, qs},
                                    {in_place ? none : res, over_y ? none : y, gate, nw, xw, parts, wt, sh, sg}))
        return r;
    if (int r = check_overlap<3, 1>(what, {out, q, qs}, {y})) return r;    // (what a shared pointer left out above)
    if (int r = check_overlap<3, 1>(what, {nx, q, qs}, {res})) return r;
    const bool vec = n % 8 == 0 && vec_rows(a->y, a->ldy, yb, 16) && vec_rows(a->residual, a->ldr, rb, 16) &&
                     vec_rows(a->out, a->ldr, rb, 16) && vec_rows(a->next, a->ld_next, nb, 16) &&
                     vec_rows(a->q, a->ldq, 1, 8) && vec_rows(nw.p, n, 4, 16) && vec_rows(xw.p, n, 4, 16) &&
                     vec_rows(a->parts, n, 4, 16) && vec_rows(a->shared, n, 4, 16) &&
                     (j.gate_kind < XS_GATE_CHANNEL ||
                      vec_rows(j.gate, j.gate_kind == XS_GATE_VALUE ? j.ld_gate : n, 4, 16));
    const hipStream_t s = hip_stream(stream);
    return finish(stream, a->parts ? launch_join<true>(*a, vec, s) : launch_join<false>(*a, vec, s), what);
}

}  // namespace
}  // namespace xs

using namespace xs;

extern "C" {

int xs_block_norm(const void* x, int x_type, int64_t ldx, const float* w, float eps, void* y, int y_type, int64_t ldy,
                  int8_t* q, int64_t ldq, float* q_scale, int64_t n_tok, int64_t n_embd, void* stream) {
    using namespace block;
    const char* what = "block_norm";
    if (int r = check_sizes(what, n_tok, n_embd, kMaxNormRow)) return r < 0 ? XS_OK : r;
    if (int r = check_rows(what, "x", x, x_type, ldx, n_embd)) return r;
    if (!y && !q) return fail(XS_EINVAL, "%s: neither float rows nor int8 rows are asked for", what);
    if (y)
        if (int r = check_rows(what, "y", y, y_type, ldy, n_embd)) return r;
    if (q || q_scale)
        if (int r = check_codes(what, q, ldq, q_scale, n_embd)) return r;
    if (w && !aligned(w, 4)) return fail(XS_EINVAL, "%s: misaligned norm weights", what);
    if (!good_eps(eps)) return fail(XS_EINVAL, "%s: eps %g is negative or not finite", what, (double)eps);
    if (!y) y_type = XS_F32;
    const int xb = float_bytes(x_type), yb = float_bytes(y_type);
    const Span none{nullptr, 0}, sx = rows_span(x, n_tok, ldx, n_embd, xb);
    const Span sy = y ? rows_span(y, n_tok, ldy, n_embd, yb) : none, sq = q ? rows_span(q, n_tok, ldq, n_embd, 1) : none;
    const Span qs{q_scale, 4 * (uint64_t)n_tok}, sw{w, 4 * (uint64_t)n_embd};
    const bool over_x = y == x && y_type == x_type && ldy == ldx;
    if (int r = check_overlap<3, 2>(what, {sy, sq, qs}, {over_x ? none : sx, sw})) return r;
    if (int r = check_overlap<2, 1>(what, {sq, qs}, {sx})) return r;
    const bool vec = n_embd % 8 == 0 && vec_rows(x, ldx, xb, 16) && vec_rows(y, ldy, yb, 16) && vec_rows(q, ldq, 1, 8) &&
                     vec_rows(w, n_embd, 4, 16);
    const NormArgs a{x, w, y, q, q_scale, ldx, ldy, ldq, n_tok, x_type, y_type, (int)n_embd, eps, 1.0 / (double)n_embd};
    return finish(stream, launch_norm(a, vec, hip_stream(stream)), what);
}

int xs_block_join(const xs_block_join_cfg_t* J, const void* y, int y_type, int64_t ldy, const void* residual, void* out,
                  int r_type, int64_t ldr, void* next, int next_type, int64_t ld_next, int8_t* q, int64_t ldq,
                  float* q_scale, int64_t n_tok, int64_t n_embd, void* stream) {
    const char* what = "block_join";
    if (int r = check_sizes(what, n_tok, n_embd, kMaxNormRow)) return r < 0 ? XS_OK : r;
    if (!J) return block::fail(XS_EINVAL, "%s: no configuration", what);
    if (int r = block::check_rows(what, "y", y, y_type, ldy, n_embd)) return r;
    JoinArgs a{};
    a.j = *J;
    a.y = y, a.y_type = y_type, a.ldy = ldy;
    a.residual = residual, a.out = out, a.r_type = r_type, a.ldr = ldr;
    a.next = next, a.next_type = next ? next_type : XS_F32, a.ld_next = ld_next;
    a.q = q, a.q_scale = q_scale, a.ldq = ldq;
    a.n_tok = n_tok, a.n = (int)n_embd, a.inv_n = 1.0 / (double)n_embd;
    return join_common(what, &a, stream);
}

int xs_moe_combine_join(const xs_block_join_cfg_t* J, const float* parts, const float* weights, int64_t k,
                        const float* shared, const float* shared_gate, const void* residual, void* out, int r_type,
                        int64_t ldr, void* next, int next_type, int64_t ld_next, int8_t* q, int64_t ldq,
                        float* q_scale, int64_t n_tok, int64_t n_embd, void* stream) {
    using namespace block;
    const char* what = "moe_combine_join";
    if (int r = check_sizes(what, n_tok, n_embd, kMaxNormRow)) return r < 0 ? XS_OK : r;
    if (!J) return fail(XS_EINVAL, "%s: no configuration", what);
    if (k < 1 || k > 15) return fail(XS_EINVAL, "%s: k %lld is not in 1..15", what, (long long)k);
    if (!aligned(parts, 4) || !aligned(weights, 4) || (shared && !aligned(shared, 4)) ||
        (shared_gate && !aligned(shared_gate, 4)))
        return fail(XS_EINVAL, "%s: a span is missing or misaligned", what);
    if (shared_gate && !shared) return fail(XS_EINVAL, "%s: a shared gate without shared rows", what);
    JoinArgs a{};
    a.j = *J;
    a.parts = parts, a.weights = weights, a.k = (int)k, a.shared = shared, a.shared_gate = shared_gate;
    a.y_type = XS_F32;
    a.residual = residual, a.out = out, a.r_type = r_type, a.ldr = ldr;
    a.next = next, a.next_type = next ? next_type : XS_F32, a.ld_next = ld_next;
    a.q = q, a.q_scale = q_scale, a.ldq = ldq;
    a.n_tok = n_tok, a.n = (int)n_embd, a.inv_n = 1.0 / (double)n_embd;
    return join_common(what, &a, stream);
}

int xs_w8a8_quantize(const void* x, int x_type, int64_t ldx, int8_t* q, int64_t ldq, float* q_scale, int64_t rows,
                     int64_t cols, void* stream) {
    using namespace block;
    const char* what = "w8a8_quantize";
    if (int r = check_sizes(what, rows, cols, kMaxInt8Row)) return r < 0 ? XS_OK : r;
    if (int r = check_rows(what, "x", x, x_type, ldx, cols)) return r;
    if (int r = check_codes(what, q, ldq, q_scale, cols)) return r;
    const int xb = float_bytes(x_type);
    if (int r = check_overlap<2, 1>(what, {rows_span(q, rows, ldq, cols, 1), Span{q_scale, 4 * (uint64_t)rows}},
                                    {rows_span(x, rows, ldx, cols, xb)}))
        return r;
    const bool vec = cols % 8 == 0 && vec_rows(x, ldx, xb, 16) && vec_rows(q, ldq, 1, 8);
    const QuantArgs a{x, q, q_scale, ldx, ldq, rows, x_type, (int)cols};
    return finish(stream, launch_quantize(a, vec, hip_stream(stream)), what);
}

}  // extern "C"
