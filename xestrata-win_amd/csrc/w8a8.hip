// xestrata-win_amd/csrc/w8a8.hip - products of int8 rows with a scale a token and a scale an output (include/xs_block.h):
//
//   y[t, o] = fl(fl(fl(sum_k x[t, k] w[o, k]) x_scale[t]) w_scale[o])     h = g / (1 + exp(-g)) u of two of them
//
// The sums are exact: |q| <= 128, so 65536 products stay below 2^31, and no order of them changes a bit.
#include "w8a8_shapes.h"
#include "xs_block.h"

#include <type_traits>

namespace xs {

typedef int v4i __attribute__((ext_vector_type(4)));

struct W8Args {
    const int8_t* x;
    const float* x_scale;
    const int8_t* w;        // the weights, or the gate rows
    const float* w_scale;
    const int8_t* w2;       // the up rows
    const float* w2_scale;
    void* y;
    int64_t ldx, ldw, ldy;
    int y_type, n_tok, n_in, n_out;
    int unit;               // what every row of y is aligned to: 16, 8, 4 or 2 bytes
};

// a lane's 16 bytes of a row from byte k on, those at n and past it zero
__device__ __forceinline__ v4i keep_bytes(v4i v, int k, int n) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int left = n - k - 4 * i;   // bytes of this word that count
        v[i] = left >= 4 ? v[i] : left <= 0 ? 0 : v[i] & (int)((1u << (8 * left)) - 1u);
    }
    return v;
}
__device__ __forceinline__ float scaled(int acc, float xs, float ws) { return ((float)acc * xs) * ws; }
__device__ __forceinline__ float silu_mul(float g, float u) { return g / (1.0f + expf(-g)) * u; }
// N neighbouring values of a row of n from o on, in stores of `unit` bytes: what every row's start is aligned to, up to 16 (o is a
// multiple of N, N 4 or 8).  Rows of an even number of 16-bit values, say, take 4 bytes at a time.
template <int N>
__device__ __forceinline__ void store_values(void* row, int type, int o, const float (&v)[N], int n, int unit) {
    by_type(type, [&](auto tc) {
        constexpr int T = decltype(tc)::value, B = float_bytes(T);
        uint32_t w[N * B / 4];
        uint8_t* const to = (uint8_t*)row + (int64_t)o * B;
#pragma unroll
        for (int e = 0; e < N * B / 4; ++e) w[e] = T == XS_F32 ? f2u(v[e]) : to_halves<T>(v[2 * e % N], v[(2 * e + 1) % N]);
        if (o + N <= n && unit >= 4) {
            if (unit == 16 && N * B >= 16) {
#pragma unroll
                for (int e = 0; e + 4 <= N * B / 4; e += 4) *(uint4*)(to + 4 * e) = make_uint4(w[e], w[e + 1], w[e + 2], w[e + 3]);
            } else if (unit >= 8) {
#pragma unroll
                for (int e = 0; e < N * B / 4; e += 2) *(uint2*)(to + 4 * e) = make_uint2(w[e], w[e + 1]);
            } else {
#pragma unroll
                for (int e = 0; e < N * B / 4; ++e) *(uint32_t*)(to + 4 * e) = w[e];
            }
            return;
        }
#pragma unroll
        for (int e = 0; e < N; ++e) {
            if (o + e >= n) continue;
            if (T == XS_F32)
                ((uint32_t*)to)[e] = w[e];
            else
                ((uint16_t*)to)[e] = (uint16_t)(w[e / 2] >> (16 * (e & 1)));
        }
    });
}

// Work-group b runs on XCD b % 8, which has an L2 of its own: an XCD takes neighbouring tiles, in bands of kBand token tiles, so
// that the 32 it has in flight read few different rows.
__device__ __forceinline__ void tile_of(int b, int m_tiles, int n_tiles, int& mt, int& nt) {
    constexpr int kBand = 4;
    const int total = m_tiles * n_tiles, per = total / 8, more = total % 8, x = b % 8;
    const int id = x * per + min(x, more) + b / 8;
    const int band = id / (kBand * n_tiles), first = band * kBand, high = min(kBand, m_tiles - first);
    const int in = id - band * kBand * n_tiles;
    mt = first + in % high;
    nt = in / high;
}

// LDS rows are 128 bytes of k.  The 16-byte chunk c of row r sits at chunk c ^ swz(r): the 16 lanes that ds_read_b128 serves in
// a cycle (0-3, 12-15, 20-27; 4-11, 16-19, 28-31; ...), reading chunk l / 16 of rows l % 16, meet 16 different 16-byte columns of
// the 256 bytes that LDS gives (no bank conflict is counted).
__device__ __forceinline__ int swz(int row) { return row >> 1 & 7; }
template <int N>
__device__ __forceinline__ void vm_left() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// Few tokens: a work-group takes 16 WT weight rows (GATED: 8 WT outputs, their gate and their up rows in turn) and 16 TT tokens.
// Its NW waves are dealt the rows' 128-byte units in turn; each fills a ring of U units of its own in LDS by DMA (8 rows of 128
// whole bytes an instruction) and multiplies them (v_mfma_i32_16x16x64_i8) without any barrier; the waves' sums are joined in
// LDS at the end.  ONCE: no other work-group reads these weight rows.
//
// Bound by the weights' way out of memory at one to 16 tokens (1 x 4096 x 16384: 16 us, 4.2 TB/s; one launch over 17 MB, 1 x
// 4096 x 4096, 5.6 us, most of it the start and the first misses), by what the L2s give the CUs at more.  The same units loaded
// to registers, where an instruction meets 16 rows' 64 bytes: 16 x 7168 x 2048 9.1 us, 5.5 by DMA; 37 x 7168 x 2050 12.3, 8.4;
// 64 x 4096 x 4096 10.5, 7.0.
template <int TT, int WT, int U, int NW, bool ONCE, bool GATED>
__global__ __launch_bounds__(64 * NW) void w8a8_ring_kernel(const W8Args a) {
    constexpr int R = TT + WT, NI = 2 * R, kSlot = R * 2048;
    extern __shared__ __align__(16) uint8_t lds[];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, l15 = lane & 15, quad = lane >> 4;
    const int o0 = blockIdx.x * (GATED ? 8 * WT : 16 * WT), t0 = blockIdx.y * 16 * TT;
    const int K = a.n_in, whole = K / 128;
    const int8_t* const xb = a.x + (int64_t)t0 * a.ldx;
    const int8_t* const wb = a.w + (int64_t)o0 * a.ldw;
    const int8_t* const ub = GATED ? a.w2 + (int64_t)o0 * a.ldw : nullptr;
    const int sub = lane >> 3;
    uint32_t off[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int r = (i & 1) * 8 + sub, chunk = (lane & 7) ^ swz(r), b = i / 2;
        off[i] = 16u * chunk + (b < WT ? (uint32_t)min(16 * (GATED ? b / 2 : b) + r, a.n_out - 1 - o0) * (uint32_t)a.ldw
                                       : (uint32_t)min(16 * (b - WT) + r, a.n_tok - 1 - t0) * (uint32_t)a.ldx);
    }
    const uint32_t lds0 = lds_offset(lds) + (uint32_t)(wave * U * kSlot);
    auto fetch = [&](int unit, int u) {   // (a weight tile's or a token tile's 16 rows are DMAs 2 b, 2 b + 1)
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int b = i / 2;
            const int8_t* base = b >= WT ? xb : GATED && (b & 1) ? ub : wb;
            const uint32_t to = lds0 + (uint32_t)(u * kSlot + i * 1024);
            if (ONCE && b < WT)
                dma16_nt_at(base, off[i] + 128u * unit, to);
            else
                dma16_at(base, off[i] + 128u * unit, to);
        }
    };
    v4i acc[WT][TT];
#pragma unroll
    for (int i = 0; i < WT; ++i)
#pragma unroll
        for (int j = 0; j < TT; ++j) acc[i][j] = (v4i){0, 0, 0, 0};
    const uint8_t* const mine = lds + wave * U * kSlot + l15 * 128;
    int at[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) at[h] = ((4 * h + quad) ^ swz(l15)) << 4;
    auto multiply = [&](int u) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            v4i w[WT], x[TT];
#pragma unroll
            for (int i = 0; i < WT; ++i) w[i] = *(const v4i*)(mine + u * kSlot + i * 2048 + at[h]);
#pragma unroll
            for (int j = 0; j < TT; ++j) x[j] = *(const v4i*)(mine + u * kSlot + (WT + j) * 2048 + at[h]);
#pragma unroll
            for (int i = 0; i < WT; ++i)
#pragma unroll
                for (int j = 0; j < TT; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[i], x[j], acc[i][j], 0, 0, 0);
        }
    };
    const int n = whole > wave ? (whole - wave + NW - 1) / NW : 0;   // this wave's units
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (u < n) fetch(wave + NW * u, u);
    int u = 0;
    for (int i = 0; i < n; ++i) {
        if (i + U <= n)   // (the U - 1 units after this one may be on their way)
            vm_left<(U - 1) * NI>();
        else
            vm_left<0>();
        multiply(u);
        lds_reads_done();   // before the slot is filled again
        if (i + U < n) fetch(wave + NW * (i + U), u);
        u = u + 1 == U ? 0 : u + 1;
    }
    if (128 * whole < K && wave == whole % NW) {   // the row's last bytes, those past it zero
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int k = 128 * whole + 64 * h + 16 * quad;
            const bool in = k < K;
            v4i w[WT], x[TT];
#pragma unroll
            for (int i = 0; i < WT; ++i) {
                const int8_t* base = GATED && (i & 1) ? a.w2 : a.w;
                const int64_t o = min(o0 + 16 * (GATED ? i / 2 : i) + l15, a.n_out - 1);
                w[i] = in ? *(const v4i*)(base + o * a.ldw + k) : (v4i){0, 0, 0, 0};
            }
#pragma unroll
            for (int j = 0; j < TT; ++j) {
                const int64_t t = min(t0 + 16 * j + l15, a.n_tok - 1);
                x[j] = keep_bytes(in ? *(const v4i*)(a.x + t * a.ldx + k) : (v4i){0, 0, 0, 0}, k, K);
            }
#pragma unroll
            for (int i = 0; i < WT; ++i)
#pragma unroll
                for (int j = 0; j < TT; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[i], x[j], acc[i][j], 0, 0, 0);
        }
    }
    static_assert(WT * TT * 1024 <= U * kSlot, "the sums fit where the rings were");
    __syncthreads();   // (every wave is done with its ring)
    v4i(*const red)[WT * TT][64] = (v4i(*)[WT * TT][64])lds;
#pragma unroll
    for (int i = 0; i < WT; ++i)
#pragma unroll
        for (int j = 0; j < TT; ++j) red[wave][i * TT + j][lane] = acc[i][j];
    __syncthreads();
    constexpr int kItems = (GATED ? WT / 2 : WT) * TT * 64;
    for (int it = threadIdx.x; it < kItems; it += 64 * NW) {
        const int tile = it >> 6, l = it & 63, i = tile / TT, j = tile % TT;
        const int ti = (GATED ? 2 * i : i) * TT + j;
        v4i s = red[0][ti][l], s2 = (v4i){0, 0, 0, 0};
        if (GATED) s2 = red[0][ti + TT][l];
#pragma unroll
        for (int v = 1; v < NW; ++v) {
            s += red[v][ti][l];
            if (GATED) s2 += red[v][ti + TT][l];
        }
        const int t = t0 + 16 * j + (l & 15), o = o0 + 16 * i + 4 * (l >> 4);
        if (t >= a.n_tok) continue;
        const float xs = a.x_scale[t];
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int oe = min(o + e, a.n_out - 1);
            v[e] = scaled(s[e], xs, a.w_scale[oe]);
            if (GATED) v[e] = silu_mul(v[e], scaled(s2[e], xs, a.w2_scale[oe]));
        }
        store_values<4>((uint8_t*)a.y + (int64_t)t * a.ldy * float_bytes(a.y_type), a.y_type, o, v, a.n_out, a.unit);
    }
}

// Many tokens: BM tokens x BN weight rows a work-group (GATED: BN / 2 outputs, their gate and their up rows), WM x WN waves,
// v_mfma_i32_16x16x64_i8 (a block's sums: lane l has weight rows 4 (l / 16) .. + 3 of token l % 16).  Steps of 128 bytes of
// every row go to LDS by DMA, into S buffers of token rows and S + 1 of weight rows.
//
// Bound by the matrix pipe together with what feeds it: a step of a 256 x 256 tile is 2,048 cycles of products, 1,024 of DMA
// issue (64 of 1 KB), and 1,280 of LDS (192 KB read at 256 bytes a cycle, 64 KB written at 128).  So the DMAs are spread over
// the step, one after every 16 products: the third buffer lets the weights' be asked for a step early, when the tokens' buffer
// is not free yet.  Fragments are read a stage (16 to 32 products) ahead, across the step's one barrier too.
// 4096 x 14336 x 4096: 183 us, 2,629 TOP/s; with two buffers of both and the 8 DMAs after the barrier 203.  Also measured there:
// 32 x 32 x 32 products 7% slower, steps of 64 bytes 15% (each 128-byte line is asked of the L2 twice), 4 waves of 128 x 128
// with a SIMD each 13%, two groups of waves taking turns at products and loads 10%.  The clock falls from 2.4 to 1.95 GHz under it,
// and the matrix pipe is busy 61% of those cycles.
template <int BM, int BN, int S>
constexpr int tile_lds() {
    return (S * BM + (S + 1) * BN) * 128;
}
template <int BM, int BN, int WM, int WN, int S, bool GATED>
__global__ __launch_bounds__(64 * WM * WN) void w8a8_tile_kernel(const W8Args a, const int m_tiles, const int n_tiles) {
    constexpr int NW = WM * WN, FM = BM / WM / 16, FN = BN / WN / 16, BK = 128;
    constexpr int NX = BM / 8 / NW, NB = BN / 8 / NW;   // a wave's DMAs a step: tokens', weights'
    constexpr int JH = FN < 4 ? FN : 4, NH = FN / JH;   // weight blocks a stage; stages a 64 bytes of k
    constexpr int NQ = 2 * NH;                          // stages a step
    // the wave's weight rows are permuted, so that a lane's sums of two blocks (JO of them where JO < 4) are neighbouring outputs
    // of its token; JO blocks are a group
    constexpr int JO = GATED ? (FN / 2 < 4 ? FN / 2 : 4) : JH, OB = 16 * JO, GW = FN / JO / (GATED ? 2 : 1);
    static_assert(NX * 8 * NW == BM && NB * 8 * NW == BN, "whole DMAs of tokens and of weights a wave");
    static_assert(FN % JH == 0 && (GATED ? FN / 2 : FN) % JO == 0 && NW % 2 == 0, "whole groups of blocks");
    extern __shared__ __align__(16) uint8_t lds[];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    int mt, nt;
    tile_of(blockIdx.x, m_tiles, n_tiles, mt, nt);
    const int t0 = mt * BM, o0 = nt * (GATED ? BN / 2 : BN);
    const int wm = wave / WN, wn = wave % WN, l15 = lane & 15, quad = lane >> 4;
    const int K = a.n_in, steps = (K + BK - 1) / BK, whole = K / BK;

    // the wave's DMAs of a step: 1 KB each, 8 rows of the tokens' or the weights' slab, from a uniform address and the lane's
    // 32-bit offset
    const int sub = lane >> 3, chunk = (lane & 7) ^ swz(8 * (wave & 1) + sub);   // (NW is even)
    const int8_t* const xbase = a.x + (int64_t)t0 * a.ldx;
    const int8_t* const wbase = a.w + (int64_t)o0 * a.ldw;
    const int8_t* const ubase = GATED ? a.w2 + (int64_t)o0 * a.ldw : nullptr;
    uint32_t xoff[NX], woff[NB];
    bool up[NB];   // whether the DMA's 8 rows are up rows; uniform
#pragma unroll
    for (int i = 0; i < NX; ++i) xoff[i] = 16u * chunk + (uint32_t)min((wave + NW * i) * 8 + sub, a.n_tok - 1 - t0) * (uint32_t)a.ldx;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        // LDS row b is row `in` of block j of a wave's rows; that is this output of the block group j / JO, the groups of up rows
        // after those of gate rows.  A lane's 8 neighbouring outputs are then 16 bytes, which with the other quads' fill 64
        // (32 a lane in two stores 32 bytes apart: 4096 x 7168 x 8192 199 us, 189 so).
        const int b = (wave + NW * i) * 8 + sub, w = b / (BN / WN), j = b % (BN / WN) / 16, in = b & 15, g = j / JO;
        const int o = (w * GW + g % GW) * OB + (in & 3) +
                      (JO == 4 ? 32 * (j % JO / 2) + 8 * (in >> 2) + 4 * (j & 1) : 4 * JO * (in >> 2) + 4 * (j % JO));
        up[i] = __builtin_amdgcn_readfirstlane(GATED && g >= GW);
        woff[i] = 16u * chunk + (uint32_t)min(o, a.n_out - 1 - o0) * (uint32_t)a.ldw;
    }
    const uint32_t lds0 = lds_offset(lds) + (uint32_t)wave * 1024u;
    // the row's last step: lanes whose 16 bytes are past the row read its start instead (their products are masked)
    auto from = [&](uint32_t off, int k) { return k + BK > K && k + 16 * chunk >= K ? off - 16u * chunk : off + (uint32_t)k; };
    auto fetch_x = [&](int s, int i) {
        dma16_at(xbase, from(xoff[i], s * BK), lds0 + (uint32_t)(s % S) * (BM * BK) + (uint32_t)(i * NW * 1024));
    };
    auto fetch_w = [&](int s, int i) {
        dma16_at(GATED && up[i] ? ubase : wbase, from(woff[i], s * BK),
                 lds0 + (uint32_t)(S * BM * BK) + (uint32_t)(s % (S + 1)) * (BN * BK) + (uint32_t)(i * NW * 1024));
    };
    v4i acc[FN][FM];
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int i = 0; i < FM; ++i) acc[j][i] = (v4i){0, 0, 0, 0};
    int at[2];   // a lane's byte in a 16-row block for each 64 bytes of k (blocks start at whole 16 rows: swz of l15)
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) at[kk] = l15 * BK + (((4 * kk + quad) ^ swz(l15)) << 4);
    const uint8_t* const lx = lds + wm * (BM / WM) * BK;
    const uint8_t* const lw = lds + (S * BM + wn * (BN / WN)) * BK;
    v4i x[2][FM], w[2][JH];
    auto read_x = [&](int s, int kk) {
#pragma unroll
        for (int i = 0; i < FM; ++i) x[kk][i] = *(const v4i*)(lx + (s % S) * (BM * BK) + at[kk] + i * 16 * BK);
    };
    auto read_w = [&](int s, int kk, int h, v4i (&to)[JH]) {
#pragma unroll
        for (int j = 0; j < JH; ++j) to[j] = *(const v4i*)(lw + (s % (S + 1)) * (BN * BK) + at[kk] + (h * JH + j) * 16 * BK);
    };
    // a stage's products of block row j
    auto multiply = [&](int kk, int h, int j, const v4i (&wj)[JH]) {
#pragma unroll
        for (int i = 0; i < FM; ++i)
            acc[h * JH + j][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wj[j], x[kk][i], acc[h * JH + j][i], 0, 0, 0);
    };
    // (tests/test_w8a8_schedule.py compiles the lines from here to the sums, and the ring's loop, for the host)
    // asked for in the order in which they are waited for: x 0, w 0, ... x S - 1, w S - 1, w S
#pragma unroll
    for (int s = 0; s <= S; ++s)
        if (s < steps) {
#pragma unroll
            for (int i = 0; i < NX; ++i)
                if (s < S) fetch_x(s, i);
#pragma unroll
            for (int i = 0; i < NB; ++i) fetch_w(s, i);
        }
    // A step is there for every wave: this wave's DMAs of it have landed, then the barrier.  The wave's reads of the step before
    // have returned as well, so that after the barrier that step's buffers may be filled again.
    auto arrive = [&] {
        lds_reads_done();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    if (steps > S)
        vm_left<(S - 1) * (NX + NB) + NB>();
    else
        vm_left<0>();
    arrive();
    if (whole > 0) {
        read_x(0, 0);
        read_w(0, 0, 0, w[0]);
    }
    for (int s = 0; s < whole; ++s) {
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
            // the next stage's fragments are read while this one's products run; those of the next step after its arrival, with
            // one stage of this step's products still to come
            const int n = q + 1, kk = q / NH, nk = n / NH & 1, nh = n % NH;
            if (n < NQ) {
                if (nh == 0) read_x(s, nk);
                read_w(s, nk, nh, w[n & 1]);
            } else {
                if (s + S < steps)   // (x of s + 2 .. s + S - 1 and w of s + 2 .. s + S may be on their way)
                    vm_left<(S - 2) * NX + (S - 1) * NB>();
                else
                    vm_left<0>();
                arrive();
                read_x(s + 1, 0);   // (past the last whole step: bytes that no product uses)
                read_w(s + 1, 0, 0, w[0]);
            }
#pragma unroll
            for (int j = 0; j < JH; ++j) {
                multiply(kk, q % NH, j, w[q & 1]);
                __builtin_amdgcn_sched_barrier(0);
                // in the first stage the weights of s + S (s 0: they are asked for above), whose buffer step s - 1 has left; in
                // the last, the tokens of s + S
                if (q == 0 && s > 0 && s + S < steps) {
#pragma unroll
                    for (int i = j; i < NB; i += JH) fetch_w(s + S, i);
                }
                if (q == NQ - 1 && s + S < steps) {
#pragma unroll
                    for (int i = j; i < NX; i += JH) fetch_x(s + S, i);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
    if (whole < steps) {   // the row's last bytes, those past it masked
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            read_x(whole, kk);
#pragma unroll
            for (int i = 0; i < FM; ++i) x[kk][i] = keep_bytes(x[kk][i], whole * BK + 64 * kk + 16 * quad, K);
#pragma unroll
            for (int h = 0; h < NH; ++h) {
                read_w(whole, kk, h, w[0]);
#pragma unroll
                for (int j = 0; j < JH; ++j) multiply(kk, h, j, w[0]);
            }
        }
    }
    // a lane's sums: NO neighbouring outputs of token l15 of each 16, NP times
    constexpr int NO = JO == 4 ? 8 : 4 * JO, NP = JO == 4 ? 2 : 1, JP = NO / 4;
    float xs[FM];
#pragma unroll
    for (int i = 0; i < FM; ++i) xs[i] = a.x_scale[min(t0 + wm * (BM / WM) + 16 * i + l15, a.n_tok - 1)];
#pragma unroll
    for (int gp = 0; gp < GW * NP; ++gp) {
        const int g = gp / NP, p = gp % NP, o = o0 + (wn * GW + g) * OB + 32 * p + NO * quad;
        float ws[NO], us[NO];
#pragma unroll
        for (int e = 0; e < NO; ++e) {
            ws[e] = a.w_scale[min(o + e, a.n_out - 1)];
            us[e] = GATED ? a.w2_scale[min(o + e, a.n_out - 1)] : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            const int t = t0 + wm * (BM / WM) + 16 * i + l15;
            float v[NO];
#pragma unroll
            for (int e = 0; e < NO; ++e) {
                v[e] = scaled(acc[g * JO + p * JP + e / 4][i][e % 4], xs[i], ws[e]);
                if (GATED) v[e] = silu_mul(v[e], scaled(acc[(GATED ? GW + g : 0) * JO + p * JP + e / 4][i][e % 4], xs[i], us[e]));
            }
            if (t < a.n_tok) store_values<NO>((uint8_t*)a.y + (int64_t)t * a.ldy * float_bytes(a.y_type), a.y_type, o, v, a.n_out, a.unit);
        }
    }
}

namespace {

template <typename K>
hipError_t allow_lds(K* kern, int bytes) {
    return bytes > 65536 ? hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) : hipSuccess;
}
template <int TT, int WT, int U, int NW, bool ONCE, bool GATED>
hipError_t launch_ring(const W8Args& a, hipStream_t s) {
    constexpr int kOut = GATED ? 8 * WT : 16 * WT, kLds = NW * U * (TT + WT) * 2048;
    auto* kern = &w8a8_ring_kernel<TT, WT, U, NW, ONCE, GATED>;
    if (const hipError_t e = allow_lds(kern, kLds)) return e;
    const dim3 grid((unsigned)((a.n_out + kOut - 1) / kOut), (unsigned)((a.n_tok + 16 * TT - 1) / (16 * TT)));
    hipLaunchKernelGGL(kern, grid, dim3(64 * NW), kLds, s, a);
    return hipGetLastError();
}
template <int BM, int BN, int WM, int WN, int S, bool GATED>
hipError_t launch_tiles(const W8Args& a, hipStream_t s) {
    constexpr int kOut = GATED ? BN / 2 : BN, kLds = tile_lds<BM, BN, S>();
    auto* kern = &w8a8_tile_kernel<BM, BN, WM, WN, S, GATED>;
    if (const hipError_t e = allow_lds(kern, kLds)) return e;
    const int m = (a.n_tok + BM - 1) / BM, n = (a.n_out + kOut - 1) / kOut;
    hipLaunchKernelGGL(kern, dim3((unsigned)(m * n)), dim3(64 * WM * WN), kLds, s, a, m, n);
    return hipGetLastError();
}
template <bool GATED>
hipError_t launch_w8a8(const W8Args& a, hipStream_t s) {
    switch (pick_shape(a.n_tok, a.n_in, a.n_out, GATED)) {
        case 0:
            if constexpr (GATED)
                return a.n_tok <= 16 ? launch_ring<1, 2, 2, 4, true, true>(a, s) : launch_ring<1, 2, 2, 4, false, true>(a, s);
            else
                return a.n_tok <= 16 ? launch_ring<1, 1, 2, 16, true, false>(a, s) : launch_ring<1, 1, 2, 16, false, false>(a, s);
        case 1: return launch_ring<2, 2, 2, 4, false, GATED>(a, s);
        case 2: return launch_ring<4, 2, 2, 4, false, GATED>(a, s);
        case 3: return launch_ring<4, 4, 1, 8, false, GATED>(a, s);
        case 4: return launch_tiles<64, 64, 2, 2, 4, GATED>(a, s);
        case 5: return launch_tiles<64, 128, 2, 4, 4, GATED>(a, s);
        case 6: return launch_tiles<128, 128, 2, 4, 2, GATED>(a, s);
        case 7: return launch_tiles<128, 256, 2, 4, 2, GATED>(a, s);
        case 8: return launch_tiles<256, 256, 4, 2, 2, GATED>(a, s);
    }
    return hipErrorInvalidValue;
}

// (row strides up to 8 MiB: 255 rows and a row's bytes stay within the tiles' 32-bit offsets)
constexpr int64_t kMaxIn = 65536, kMaxOut = 1 << 24, kMaxTok = 1 << 20, kMaxStride = 1 << 23;

int product_args(const char* what, const int8_t* x, int64_t ldx, const float* x_scale, const int8_t* w,
                 const float* w_scale, const int8_t* w2, const float* w2_scale, bool gated, int64_t ldw, void* y,
                 int y_type, int64_t ldy, int64_t n_tok, int64_t n_in, int64_t n_out, W8Args* a) {
    using namespace block;
    if (n_tok > kMaxTok || n_in < 1 || n_in > kMaxIn || n_out < 1 || n_out > kMaxOut)
        return fail(XS_EINVAL, "%s: %lld tokens, %lld x %lld weights (up to %lld tokens, 1 .. %lld inputs, 1 .. %lld outputs)",
                    what, (long long)n_tok, (long long)n_out, (long long)n_in, (long long)kMaxTok, (long long)kMaxIn,
                    (long long)kMaxOut);
    if (!aligned(x, 16) || !aligned(w, 16) || (gated && !aligned(w2, 16)) || !aligned(x_scale, 4) || !aligned(w_scale, 4) ||
        (gated && !aligned(w2_scale, 4)))
        return fail(XS_EINVAL, "%s: a span is missing or misaligned (codes 16 bytes, scales 4)", what);
    const int64_t need = (n_in + 15) / 16 * 16;
    if (ldx % 16 || ldw % 16 || ldx < need || ldw < need || ldx > kMaxStride || ldw > kMaxStride)
        return fail(XS_EINVAL, "%s: int8 rows of %lld values %lld and %lld bytes apart (multiples of 16, %lld .. %lld)", what,
                    (long long)n_in, (long long)ldx, (long long)ldw, (long long)need, (long long)kMaxStride);
    if (int r = check_rows(what, gated ? "h" : "y", y, y_type, ldy, n_out)) return r;
    const Span none{nullptr, 0};
    if (int r = check_overlap<1, 6>(what, {rows_span(y, n_tok, ldy, n_out, float_bytes(y_type))},
                                    {rows_span(x, n_tok, ldx, need, 1), Span{x_scale, 4 * (uint64_t)n_tok},
                                     rows_span(w, n_out, ldw, need, 1), Span{w_scale, 4 * (uint64_t)n_out},
                                     gated ? rows_span(w2, n_out, ldw, need, 1) : none,
                                     gated ? Span{w2_scale, 4 * (uint64_t)n_out} : none}))
        return r;
    int unit = 16;
    while (!vec_rows(y, ldy, float_bytes(y_type), unit)) unit /= 2;   // (down to the type's size at the least)
    *a = W8Args{x, x_scale, w, w_scale, w2, w2_scale, y, ldx, ldw, ldy, y_type, (int)n_tok, (int)n_in, (int)n_out,
                unit};
    return XS_OK;
}

}  // namespace
}  // namespace xs

using namespace xs;

extern "C" {

int xs_w8a8_gemm(const int8_t* x, int64_t ldx, const float* x_scale, const int8_t* w, int64_t ldw, const float* w_scale,
                 void* y, int y_type, int64_t ldy, int64_t n_tok, int64_t n_in, int64_t n_out, void* stream) {
    if (n_tok <= 0) return XS_OK;
    W8Args a;
    if (int r = product_args("w8a8_gemm", x, ldx, x_scale, w, w_scale, nullptr, nullptr, false, ldw, y, y_type, ldy, n_tok,
                             n_in, n_out, &a))
        return r;
    return block::finish(stream, launch_w8a8<false>(a, hip_stream(stream)), "w8a8_gemm");
}

int xs_w8a8_swiglu(const int8_t* x, int64_t ldx, const float* x_scale, const int8_t* w_gate, const float* gate_scale,
                   const int8_t* w_up, const float* up_scale, int64_t ldw, void* h, int h_type, int64_t ldh,
                   int64_t n_tok, int64_t n_in, int64_t n_ff, void* stream) {
    if (n_tok <= 0) return XS_OK;
    W8Args a;
    if (int r = product_args("w8a8_swiglu", x, ldx, x_scale, w_gate, gate_scale, w_up, up_scale, true, ldw, h, h_type, ldh,
                             n_tok, n_in, n_ff, &a))
        return r;
    return block::finish(stream, launch_w8a8<true>(a, hip_stream(stream)), "w8a8_swiglu");
}

}  // extern "C"
