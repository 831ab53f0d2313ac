// softmax_loss.hip - softmax cross entropy of a batch of rows against a whole catalogue of items, and its gradient, without
// ever keeping the n x n_items logits (gfx950, MI355X).
//
//   z_rv = scale x_r.w_v + b_v,   lse_r = log sum_v exp z_rv,   loss_r = lse_r - z_{r,t_r}
//   G_rv = g_r (exp(z_rv - lse_r) - [v = t_r]),   dX = scale G W,   dW = scale G^T X,   db = sum_r G_r
//
// One kernel shape does all the products (k_stream): a wave keeps 32 STATIONARY rows in registers and walks past tiles of
// STREAMED rows in LDS.  With streamed rows as MFMA rows and stationary rows as MFMA columns a lane ends up with 16 logits
// of ONE stationary row, so a row's reference and sum are private to two lanes, and the exponentials are, as they stand, the B
// operand of the second product (the order of the streamed rows inside an operand is free, and the other operand, read
// transposed from the same LDS tile, takes the same order).
//   planes   rows that are no operands as they are: split, padded, and cleared where they take no part (small batches do
//            that on the way instead)
//   pass 1   stationary x, streamed items:  a reference m, sum_v exp(z - m) and sum_v exp(z - m) w_v, in one walk
//   join     the parts of the items' axis: lse, loss, dX
//   pass 2   stationary items, streamed x:  the logits again, now with lse known:  dW, db, and a join if x is cut into parts
// 8 n d V operations, two of the logits, against the 6 that cannot be avoided: keeping the logits would move 2 n V elements
// to memory and back instead (4096 x 624961 in bf16: 10 GB, 2 ms, instead of 1.2 ms of products).
//
// What bounds it: power, then the vector unit.  4096 x 624961 x 256 bf16: 2.23 and 2.43 ms for the passes, 1180 and 1080
// TFLOP/s; the matrix cores are busy 70 % and 63 % of the cycles at the 1.6 GHz that the card keeps under this load (a library
// product of 8192 cubed: 1115 TFLOP/s).  8192 x 17770 x 128 fp32: 356 and 402 us, 1260 and 1110 TFLOP/s of bf16 products, busy
// 80 % and 76 %.  A loss without gradients has an exponential, a multiply-add and an add for 2 d operations: 5003 x 59047 x
// 100 bf16 97 us, vector unit 60 %, matrix cores 44 %.  LDS: no bank conflicts (swizzle, below), active 30 to 50 %.  A third
// tile in LDS, so that loads have two tiles' time, changed nothing.  Small problems wait: 12 us a launch to start, fetch and
// end, which decides the number of parts (parts_of).
//
// The target's own term stays out of the matrix products: pass 1 leaves it to the join, which adds it in fp32 from the rows
// themselves - 1 - p_t is then the other items' share, not a difference of rounded numbers, and a well-learnt row's gradient
// (p_t near 1) keeps its digits; pass 2 adds a bf16 target's x to its item in fp32.
//
// Types: bf16 rows are the operands as they are.  An fp32 row is split into three bf16 rows of 8 bits each (x = x0 + x1 + x2,
// exact to 2^-24), and a product is the six products of order up to 2 - the three left out are below 2^-24 of it.  Six bf16
// matrix instructions cost less than one fp32 instruction of the same shape (2.5 PFLOP/s against 157 TFLOP/s).  The
// exponentials, too, are rounded to bf16 for the second product (bf16 rows: once, by at most 2^-8 of a term, what the outputs themselves
// are rounded by; in three parts it took 30 % more time.  fp32 rows: three parts, exact to 2^-24).  The sum of the
// exponentials, lse, loss and 1 - p_t are of the unrounded ones.
#include <algorithm>
#include <math.h>
#include <type_traits>
#include "rows.h"

namespace {

#define LDS_AS __attribute__((address_space(3)))
#define GLB_AS __attribute__((address_space(1)))
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
// The reference of a row's exponentials is the largest logit of the first 32 items that are in the catalogue, and stays it
// while the row's sum is below this (log2 60): what counts is that nothing overflows, so no maximum is taken on the way.
constexpr float TOO_MUCH = 1.152921504606846976e18f;
constexpr float UNSET = 1e30f;          // the sum of a row that has no reference yet: too much, so that the next items set one

enum { LOSS = 0, LOSS_SUMS = 1, TABLE = 2 };   // pass 1 without / with the weighted sums, pass 2

struct Rows {                           // rows as the caller has them
    const void *p;
    int64_t stride;
    int32_t n;
};

struct StreamArgs {
    Rows st, sm;                        // stationary rows; streamed rows where they are converted on the way (CONV)
    const __bf16 *sm_planes;            // else: planes of the streamed rows, DP wide, zero padded
    int64_t planes_stride, plane;
    int32_t d, n_items;
    int32_t clear;                      // pass 1: sm_planes is the table itself, and items may be out of the catalogue
    const int32_t *targets;             // of the x rows
    const float *bias;                  // of the items, may be NULL
    float c, inv_scale;                 // scale log2(e), 1 / scale
    int32_t splits, row_tiles;
    float *part_m, *part_s;             // pass 1 [splits][rows]; pass 2: part_s = sums of G for the bias, NULL: not wanted
    float *part_o;                      // [splits][rows][DP]; pass 2, splits == 1: NULL, the result goes to out
    const float *row_init, *row_q, *row_g;   // pass 2: -lse / scale, g (1 - p_t), g (g: the row's weight, NULL: all 1)
    void *out;                          // pass 2: dW [n_items][d] of the rows' type, times out_f
    float *out_b;                       // and db, times weight
    float out_f, weight;
};

// 8 elements of a row from column c on, zero behind column d
template <typename T> struct Piece;
template <> struct Piece<float> { float v[8]; };
template <> struct Piece<__bf16> { uint32_t v[4]; };
__device__ __forceinline__ void load_piece(const float *row, int32_t c, int32_t d, Piece<float> &o)
{
    if (c + 8 <= d) load_vec<8>(row + c, o.v);
    else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float t = row[c + i < d ? c + i : 0];
            o.v[i] = c + i < d ? t : 0.f;
        }
    }
}
__device__ __forceinline__ void load_piece(const __bf16 *row, int32_t c, int32_t d, Piece<__bf16> &o)
{
    if (c + 8 <= d) {
        const words_of<8, __bf16> t = *(const words_of<8, __bf16> *)(row + c);
#pragma unroll
        for (int i = 0; i < 4; ++i) o.v[i] = t[i];
    } else {
        const uint16_t *bits = (const uint16_t *)row;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t lo = bits[c + 2 * i < d ? c + 2 * i : 0], hi = bits[c + 2 * i + 1 < d ? c + 2 * i + 1 : 0];
            o.v[i] = (c + 2 * i < d ? lo : 0) | (c + 2 * i + 1 < d ? hi << 16 : 0);
        }
    }
}
// ... as matrix operands: a bf16 piece as it is, an fp32 piece as three of which the sum is exact to 2^-24
__device__ __forceinline__ void split_piece(const Piece<__bf16> &in, bool live, bf16x8 (&out)[1])
{
    const uint4 u = live ? make_uint4(in.v[0], in.v[1], in.v[2], in.v[3]) : make_uint4(0, 0, 0, 0);
    out[0] = __builtin_bit_cast(bf16x8, u);
}
__device__ __forceinline__ void split_piece(const Piece<float> &in, bool live, bf16x8 (&out)[3])
{
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = live ? in.v[i] : 0.f;
#pragma unroll
    for (int p = 0; p < 3; ++p) {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            u[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
            v[2 * i] -= bf16_lo(u[i]);
            v[2 * i + 1] -= bf16_hi(u[i]);
        }
        out[p] = __builtin_bit_cast(bf16x8, *(const uint4 *)u);
    }
}

template <int DP, int PL, int MODE, bool CONV> struct Shape {
    // 32-row tiles of stationary rows a wave keeps.  Two halve the reads of LDS, which bound nothing but the loss of wide bf16
    // rows (4096 x 59047, d = 256: 122 us with two, 130 with one); elsewhere one leaves more waves a SIMD
    static constexpr int UT = PL == 1 && !CONV && MODE == LOSS && DP > 128 ? 2 : 1;
    static constexpr int ROWS = 128 * UT;                            // stationary rows a workgroup
    static constexpr int NB = DP == 256 && MODE != LOSS ? (PL == 1 ? 8 : 4) : 0;     // sixteenths of a stationary row that wait in LDS
    static constexpr int TB = ((PL == 3 || CONV) && DP > 32) || NB ? 32 : 64;      // streamed rows a tile
    static constexpr int CH = DP / 8;                                // 16-byte pieces of a row
    static constexpr int BUF = PL * TB * DP * 2;                     // bytes of a tile
    static constexpr int LDS = 2 * BUF + 2 * TB * 16 + NB * PL * 4096;
    static constexpr int HOLD = CONV ? TB * CH / 256 : 0;            // pieces a thread holds on their way to LDS
    // registers: the stationary rows, the sums, the logits and what is in flight
    static constexpr int REGS = UT * PL * (DP - 16 * NB) / 4 + (MODE == LOSS ? 0 : UT * DP / 2) + UT * 16 + HOLD * (PL == 3 ? 8 : 4) + (CONV ? 20 : 0) + 48;
    // waves a SIMD; at 256 (fp32 rows of 256, no gradients) two of them spill: 4096 x 17770 269 us, 220 with one
    static constexpr int WAVES = REGS <= 120 ? 4 : REGS <= 156 ? 3 : REGS < 256 ? 2 : 1;
    static constexpr int GROUPS = WAVES < 160 * 1024 / LDS ? WAVES : 160 * 1024 / LDS;           // workgroups a CU
};

// Piece c of row r lies at piece c ^ swizzle(r).  The logits' operand takes one piece of 16 consecutive rows at a time, the
// transposed operand four neighbouring pieces of 4 consecutive rows: either set has to cover the 64 banks once.
template <int CH> __device__ __forceinline__ int swizzle(int r)
{
    if constexpr (CH % 16 == 0) return ((r & 3) << 2) | ((r >> 2) & 3);
    else if constexpr (CH % 8 == 0) return ((r & 3) << 1) | ((r >> 2) & 1);
    else return (r & 2) | ((r >> 2) & 1);
}

template <typename T, int DP, int MODE, bool CONV>
__global__ __launch_bounds__(256, (Shape<DP, sizeof(T) == 4 ? 3 : 1, MODE, CONV>::WAVES)) void k_stream(const StreamArgs a)
{
    constexpr int PL = sizeof(T) == 4 ? 3 : 1;
    using S = Shape<DP, PL, MODE, CONV>;
    constexpr int UT = S::UT, TB = S::TB, CH = S::CH, BUF = S::BUF, KS = DP / 16, DT = DP / 32, PLANE = TB * DP * 2;
    constexpr int Q = BUF / 4096, HOLD = S::HOLD;
    constexpr int GA = PL == 3 ? 1 : 2;                 // operands of a group
    static_assert(BUF % 4096 == 0, "a tile is a whole number of 1 KB pieces per wave");
    extern __shared__ __attribute__((aligned(16))) char lds[];
    float *l_init = (float *)(lds + 2 * BUF);           // [2][TB]
    float *l_g = l_init + 2 * TB, *l_q = l_g + 2 * TB;
    int32_t *l_t = (int32_t *)(l_q + 2 * TB);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 31, kh = lane >> 5;

    // consecutive workgroups go round the 8 XCDs: the row tiles that walk the same part of the streamed axis share one's L2
    int split, rt;
    if (a.splits % 8 == 0) {
        const int j = blockIdx.x >> 3;
        split = (j / a.row_tiles) * 8 + (blockIdx.x & 7);
        rt = j % a.row_tiles;
    } else {
        split = blockIdx.x / a.row_tiles;
        rt = blockIdx.x % a.row_tiles;
    }
    const int32_t n_st = a.st.n, n_sm = a.sm.n;
    const int32_t st0 = (rt * 4 + wave) * (32 * UT);
    const bool busy = st0 < n_st;
    const int32_t tiles = (n_sm + TB - 1) / TB;
    const int32_t t0 = (int32_t)((int64_t)tiles * split / a.splits), t1 = (int32_t)((int64_t)tiles * (split + 1) / a.splits);

    // A tile goes straight from memory to LDS, 1 KB a wave and instruction; its place is the lane's, so the swizzle is in
    // which piece a lane asks for.  Where few workgroups read the streamed rows (CONV) they take them as they are and
    // convert them on the way, through registers.
    constexpr int STEP = 256 / CH;                      // rows an instruction of the whole workgroup covers
    constexpr bool EVEN = 256 % CH == 0;
    uint32_t from[2];                                   // a lane's byte offset in the rows of even and odd steps
#pragma unroll
    for (int v = 0; v < 2; ++v) from[v] = (uint32_t)(tid / CH) * (uint32_t)a.planes_stride * 2 + (uint32_t)((tid % CH) ^ swizzle<CH>(tid / CH + v * STEP)) * 16;
    Piece<T> hold[HOLD ? HOLD : 1];
    uint32_t held = 0;                                  // bit q: row of piece q takes part
    // What goes with a streamed row.  Asked for in front of the tile and put into LDS when the tile is there: to put it there at
    // once would wait for it, and with it for all that was asked for before.
    float p_init = 0.f, p_g = 0.f, p_q = 0.f;
    int32_t p_t = 0;
    auto stage = [&](int32_t t, int buf) {
        const int32_t last = std::min(TB, n_sm - t * TB) - 1;
        if (tid < TB) {
            const bool in = tid <= last;
            const int32_t row = t * TB + std::min(tid, last);
            if constexpr (MODE == TABLE) {
                p_init = in ? a.row_init[row] : -INFINITY;
                if (a.row_g) p_g = a.row_g[row];
                p_q = a.row_q[row];
                p_t = in ? a.targets[row] : -1;
            } else
                p_init = !in ? -INFINITY : a.bias ? a.bias[row] : 0.f;
        }
        if constexpr (CONV) {
            held = 0;
#pragma unroll
            for (int q = 0; q < HOLD; ++q) {
                const int slot = q * 256 + tid, r = slot / CH, c = (slot % CH) ^ swizzle<CH>(slot / CH);
                const int32_t row = t * TB + std::min(r, last);
                const bool live = MODE == TABLE ? (uint32_t)a.targets[row] < (uint32_t)a.n_items : !a.bias || a.bias[row] != -INFINITY;
                held |= (uint32_t)live << q;
                load_piece((const T *)a.sm.p + row * a.sm.stride, c * 8, a.d, hold[q]);
            }
        } else {
            const __bf16 *base = a.sm_planes + (int64_t)t * TB * a.planes_stride;
            if (EVEN && last == TB - 1) {
#pragma unroll
                for (int q = 0; q < Q; ++q) {
                    constexpr int PER = Q / PL;
                    const __bf16 *rows = base + (q / PER) * a.plane + (q % PER) * STEP * a.planes_stride;
                    __builtin_amdgcn_global_load_lds((const GLB_AS void *)((const char *)rows + from[q % PER % 2]),
                                                     (LDS_AS void *)(lds + buf * BUF + (q * 4 + wave) * 1024), 16, 0, 0);
                    __builtin_amdgcn_sched_barrier(0);
                }
            } else {                                    // rows behind the last one are the last one, masked below
#pragma unroll 1
                for (int q = 0; q < Q; ++q) {
                    const int slot = q * 256 + tid;
                    const int p = slot / (TB * CH), r = slot / CH % TB, c = (slot % CH) ^ swizzle<CH>(slot / CH % TB);
                    __builtin_amdgcn_global_load_lds((const GLB_AS void *)(base + p * a.plane + std::min(r, last) * a.planes_stride + c * 8),
                                                     (LDS_AS void *)(lds + buf * BUF + (q * 4 + wave) * 1024), 16, 0, 0);
                }
            }
        }
    };
    auto commit = [&](int buf) {                        // what stage() began is in LDS afterwards
        if constexpr (CONV) {
#pragma unroll
            for (int q = 0; q < HOLD; ++q) {
                bf16x8 v[PL];
                split_piece(hold[q], (held >> q) & 1, v);
#pragma unroll
                for (int p = 0; p < PL; ++p) *(bf16x8 *)(lds + buf * BUF + p * PLANE + (q * 256 + tid) * 16) = v[p];
            }
        } else
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if (tid < TB) {
            l_init[buf * TB + tid] = MODE == TABLE ? p_init : p_init * a.inv_scale;
            if constexpr (MODE == TABLE) {
                l_g[buf * TB + tid] = p_g;
                l_q[buf * TB + tid] = p_q;
                l_t[buf * TB + tid] = p_t;
            }
        }
        __syncthreads();
        if constexpr (MODE != TABLE && !CONV && PL == 1) {
            if (a.clear) {                              // rows of items that are out: whatever they hold, zero from here on
                const uint64_t out = __ballot(lane < TB && l_init[buf * TB + lane % TB] == -INFINITY);
                if (out) {                              // the same in all four waves
                    for (uint64_t h = out; h; h &= h - 1) {
                        const int r = __builtin_ctzll(h);
                        if ((r & 3) == wave && lane < CH) *(uint4 *)(lds + buf * BUF + r * DP * 2 + lane * 16) = make_uint4(0, 0, 0, 0);
                    }
                    __syncthreads();
                }
            }
        }
    };

    f32x16 o[UT][MODE == LOSS ? 1 : DT];
    float m[UT], neg_ref[UT], sum[UT];              // log2 reference, -reference as the exponent takes it, sum
#pragma unroll
    for (int u = 0; u < UT; ++u) {
        m[u] = -INFINITY;
        neg_ref[u] = 0.f;
        sum[u] = MODE == TABLE ? 0.f : UNSET;
#pragma unroll
        for (auto &v : o[u]) v = (f32x16)(0.f);
    }

    // LDS addresses of this lane, for the tile in work: the swizzle makes an operand's address no linear function of its
    // column, but one of 2, 4 or 8 registers and a constant
    constexpr int NA = CH % 16 == 0 ? 8 : CH % 8 == 0 ? 4 : 2, NT = NA / 2;
    const LDS_AS char *l3 = (const LDS_AS char *)lds;
    uint32_t at_a[NA], at_t[NT][2], at_i = 2 * BUF + 16 * kh;
    const int i16 = lane & 15, half = (lane >> 4) & 1, tr = 4 * kh + (i16 >> 2);
#pragma unroll
    for (int s = 0; s < NA; ++s) at_a[s] = col * DP * 2 + ((2 * s + kh) ^ swizzle<CH>(col)) * 16;
#pragma unroll
    for (int d = 0; d < NT; ++d)
#pragma unroll
        for (int h = 0; h < 2; ++h)
            at_t[d][h] = (tr + 8 * h) * DP * 2 + ((4 * d + 2 * half + ((i16 & 3) >> 1)) ^ swizzle<CH>(tr + 8 * h)) * 16 + (i16 & 1) * 8;

    // operands: 16 columns of 32 streamed rows for the logits, 32 columns of 16 streamed rows, transposed, for the sums
    auto load_a = [&](int buf, int sub, int s, bf16x8 (&x)[PL]) {
#pragma unroll
        for (int p = 0; p < PL; ++p) x[p] = *(const LDS_AS bf16x8 *)(l3 + at_a[s % NA] + (buf * BUF + sub * 32 * DP * 2 + p * PLANE + s / NA * NA * 32));
    };
    auto load_t = [&](int buf, int sub, int n, bf16x8 (&x)[PL]) {
        const int k = n / DT, dt = n % DT;
#pragma unroll
        for (int p = 0; p < PL; ++p) {
            const int imm = buf * BUF + (sub * 32 + 16 * k) * DP * 2 + p * PLANE + dt / NT * NT * 64;
            const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_AS i16x4 *)(l3 + at_t[dt % NT][0] + imm));
            const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_AS i16x4 *)(l3 + at_t[dt % NT][1] + imm));
            x[p] = __builtin_shufflevector(__builtin_bit_cast(bf16x4, lo), __builtin_bit_cast(bf16x4, hi), 0, 1, 2, 3, 4, 5, 6, 7);
        }
    };

    if (t0 < t1) stage(t0, 0);                          // in flight while the stationary rows are fetched and split

    constexpr int NB = S::NB, KR = KS - NB;
    bf16x8 b[UT][PL][KR];
    LDS_AS char *l_b = (LDS_AS char *)lds + 2 * BUF + 2 * TB * 16 + (wave * NB * PL * 64 + lane) * 16;
    int32_t target[UT];
    float b2[UT];
#pragma unroll
    for (int u = 0; u < UT; ++u) {
        const int32_t row = std::min(st0 + 32 * u + col, n_st - 1);
        target[u] = MODE == TABLE ? 0 : a.targets[row];
        b2[u] = (MODE == TABLE && a.bias) ? a.bias[row] * LOG2E : 0.f;
        // neither padding nor an item that is out of the catalogue is looked at
        const bool live = MODE == TABLE ? b2[u] != -INFINITY : (uint32_t)target[u] < (uint32_t)a.n_items;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            Piece<T> raw;
            bf16x8 v[PL];
            load_piece((const T *)a.st.p + row * a.st.stride, 16 * s + 8 * kh, a.d, raw);
            split_piece(raw, live, v);
#pragma unroll
            for (int p = 0; p < PL; ++p) {
                if (s < KR) b[u][p][s] = v[p];
                else *(LDS_AS bf16x8 *)(l_b + ((s - KR) * PL + p) * 1024) = v[p];       // read by the same lane only
            }
        }
    }

    commit(0);
    // one tile; which of the two places in LDS it has is known at compile time, so that every address is a register and a constant
    auto walk = [&](int32_t t, auto place) __attribute__((always_inline)) {
        constexpr int buf = decltype(place)::value;
        if (t + 1 < t1) stage(t + 1, buf ^ 1);
        bool hit_tile = false;                          // does any row's target lie in this tile?
        if constexpr (MODE != TABLE) {
#pragma unroll
            for (int u = 0; u < UT; ++u) hit_tile |= (uint32_t)(target[u] - t * TB) < (uint32_t)TB;
            hit_tile = __ballot(hit_tile) != 0;
        }
        if (CONV && !busy) { commit(buf ^ 1); return; }     // all its rows are behind the last one
#pragma unroll
        for (int sub = 0; sub < TB / 32; ++sub) {
            // logits (in units of scale) of 32 streamed rows: acc[u][j] is row 8 (j / 4) + 4 kh + j % 4 for stationary row `col`
            f32x16 acc[UT];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const f32x4 v = *(const LDS_AS f32x4 *)(l3 + at_i + (buf * TB + sub * 32 + 8 * j) * 4);
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[0][4 * j + i] = v[i];
            }
#pragma unroll
            for (int u = 1; u < UT; ++u) acc[u] = acc[0];
            // the wave that multiplies goes first: the others' exponentials fill its gaps (8192 x 17770 x 128 fp32: 786 -> 764 us)
            __builtin_amdgcn_s_setprio(1);
            // operands are read one group ahead of the products that take them
            bf16x8 x[2][GA][PL];
#pragma unroll
            for (int q = 0; q < GA; ++q) load_a(buf, sub, q, x[0][q]);
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                if (s % GA == 0) {
                    if (s) __builtin_amdgcn_sched_barrier(0);
                    if (s + GA < KS) {
#pragma unroll
                        for (int q = 0; q < GA; ++q) load_a(buf, sub, s + GA + q, x[(s / GA + 1) & 1][q]);
                    }
                }
                const bf16x8 (&y)[PL] = x[(s / GA) & 1][s % GA];
#pragma unroll
                for (int u = 0; u < UT; ++u) {
                    bf16x8 z[PL];
#pragma unroll
                    for (int p = 0; p < PL; ++p) z[p] = s < KR ? b[u][p][s < KR ? s : 0] : *(const LDS_AS bf16x8 *)(l_b + ((s - KR) * PL + p) * 1024);
                    if constexpr (PL == 3) {
                        acc[u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(y[2], z[0], acc[u], 0, 0, 0);
                        acc[u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(y[0], z[2], acc[u], 0, 0, 0);
                        acc[u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(y[1], z[1], acc[u], 0, 0, 0);
                        acc[u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(y[1], z[0], acc[u], 0, 0, 0);
                        acc[u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(y[0], z[1], acc[u], 0, 0, 0);
                    }
                    acc[u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(y[0], z[0], acc[u], 0, 0, 0);
                }
            }
            if constexpr (MODE != LOSS) {
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int q = 0; q < GA; ++q) load_t(buf, sub, q, x[0][q]);
            }
            __builtin_amdgcn_s_setprio(0);
            bf16x8 w[UT][2][PL];       // the exponentials as operands: j 0..7 and 8..15
            uint32_t hits = 0, at = 0;
            if constexpr (MODE == TABLE) {
                // rows of the tile whose target is one of this wave's items
                at = (uint32_t)(l_t[buf * TB + sub * 32 + col] - st0);
                hits = (uint32_t)__ballot(at < 32u * UT);
            }
#pragma unroll
            for (int u = 0; u < UT; ++u) {
                float e[16];
                if constexpr (MODE != TABLE) {
                    float add;
                    auto weigh = [&] {
#pragma unroll
                        for (int j = 0; j < 16; ++j) e[j] = __builtin_amdgcn_exp2f(fmaf(acc[u][j], a.c, neg_ref[u]));
                        if (hit_tile) {
                            int32_t own = target[u] - (t * TB + sub * 32) - 4 * kh;
                            asm volatile("" : "+v"(own));           // keeps the 16 comparisons inside the branch
#pragma unroll
                            for (int j = 0; j < 16; ++j) e[j] = own == 8 * (j / 4) + j % 4 ? 0.f : e[j];
                        }
                        float s4[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) s4[j] = (e[j] + e[j + 4]) + (e[j + 8] + e[j + 12]);
                        add = (s4[0] + s4[1]) + (s4[2] + s4[3]);
                    };
                    weigh();
                    bool rise = sum[u] + add > TOO_MUCH;
                    if (__ballot(rise)) {               // rare: a new reference, the same for both lanes of a row
                        rise |= (bool)__shfl_xor((int)rise, 32, 64);
                        if (m[u] == -INFINITY && sum[u] == UNSET) sum[u] = 0.f;
                        float top = acc[u][0];
#pragma unroll
                        for (int j = 1; j < 16; ++j) top = fmaxf(top, acc[u][j]);
                        top = fmaxf(top, __shfl_xor(top, 32, 64)) * a.c;
                        const float both = sum[u] + __shfl_xor(sum[u], 32, 64);
                        const float up = both > 1.f ? fmaxf(top, m[u] + __builtin_amdgcn_logf(both)) : fmaxf(top, m[u]);
                        const float f = rise && up > m[u] ? __builtin_amdgcn_exp2f(m[u] - up) : 1.f;     // the first time: exp2(-inf) = 0
                        if (rise) m[u] = up;
                        sum[u] *= f;
                        if constexpr (MODE == LOSS_SUMS) {
#pragma unroll
                            for (auto &v : o[u]) { v *= f; __builtin_amdgcn_sched_barrier(0); }
                        }
                        neg_ref[u] = m[u] == -INFINITY ? 0.f : -m[u];
                        weigh();
                        if (m[u] == -INFINITY && sum[u] == 0.f && add == 0.f) sum[u] = UNSET;     // still no item in the catalogue
                    }
                    sum[u] += add;
                } else {
#pragma unroll
                    for (int j = 0; j < 16; ++j) e[j] = __builtin_amdgcn_exp2f(fmaf(acc[u][j], a.c, b2[u]));
                    if (a.row_g) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const f32x4 v = *(const LDS_AS f32x4 *)(l3 + at_i + ((2 + buf) * TB + sub * 32 + 8 * j) * 4);
#pragma unroll
                            for (int i = 0; i < 4; ++i) e[4 * j + i] *= v[i];
                        }
                    }
                    // Rows whose target is one of these items: -g (1 - p_t) in the place of g p_t.  It outweighs all else in an
                    // item's gradient, so bf16 rows do not leave it to the matrix product, which would round it to 8 bits (the
                    // error of a weighted batch's dW rose by half): it is added to the item's sums in fp32, row by row - one
                    // row in n_items / 32 tiles.
                    if (hits) {
                        uint32_t mine = 0;  // rows of the 32 whose target is this lane's item
                        for (uint32_t h = hits; h; h &= h - 1) {
                            const int r = __builtin_ctz(h);
                            const bool own = __builtin_amdgcn_readlane((int)at, r) == 32 * u + col;
                            mine |= (uint32_t)own << r;
                            if constexpr (PL == 1) {
                                const int row = sub * 32 + r, sw = swizzle<CH>(row);
                                const float q = own ? -l_q[buf * TB + row] : 0.f;
                                sum[u] += kh ? 0.f : q;
#pragma unroll
                                for (int c = 0; c < 4 * DT; ++c) {
                                    const uint2 x = *(const uint2 *)(lds + buf * BUF + row * DP * 2 + (c ^ sw) * 16 + kh * 8);
                                    f32x16 &v = o[u][c / 4];
                                    const int j = c % 4 * 4;
                                    v[j] = fmaf(q, bf16_lo(x.x), v[j]);
                                    v[j + 1] = fmaf(q, bf16_hi(x.x), v[j + 1]);
                                    v[j + 2] = fmaf(q, bf16_lo(x.y), v[j + 2]);
                                    v[j + 3] = fmaf(q, bf16_hi(x.y), v[j + 3]);
                                    __builtin_amdgcn_sched_barrier(0);
                                }
                            }
                        }
                        mine >>= 4 * kh;
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            f32x4 v = {0.f, 0.f, 0.f, 0.f};
                            if constexpr (PL == 3) v = *(const LDS_AS f32x4 *)(l3 + at_i + ((4 + buf) * TB + sub * 32 + 8 * j) * 4);
#pragma unroll
                            for (int i = 0; i < 4; ++i) e[4 * j + i] = (mine >> (8 * j + i)) & 1 ? -v[i] : e[4 * j + i];
                        }
                    }
                }
                if (MODE == TABLE && a.part_s) {
                    float s4[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) s4[j] = (e[j] + e[j + 4]) + (e[j + 8] + e[j + 12]);
                    sum[u] += (s4[0] + s4[1]) + (s4[2] + s4[3]);
                }
                if constexpr (MODE != LOSS) {
#pragma unroll
                    for (int p = 0; p < PL; ++p)
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            uint32_t v[4];
#pragma unroll
                            for (int q = 0; q < 4; ++q) {
                                v[q] = pack_bf16(e[8 * k + 2 * q], e[8 * k + 2 * q + 1]);
                                if (p + 1 < PL) { e[8 * k + 2 * q] -= bf16_lo(v[q]); e[8 * k + 2 * q + 1] -= bf16_hi(v[q]); }
                            }
                            w[u][k][p] = __builtin_bit_cast(bf16x8, *(const uint4 *)v);
                        }
                }
            }
            if constexpr (MODE != LOSS) {
                // o[u][dt][j] += sum over the 32 streamed rows of their column 32 dt + 8 (j / 4) + 4 kh + j % 4 times e
#pragma unroll
                for (int n = 0; n < 2 * DT; ++n) {
                    if (n % GA == 0) {
                        if (n) __builtin_amdgcn_sched_barrier(0);
                        if (n + GA < 2 * DT) {
#pragma unroll
                            for (int q = 0; q < GA; ++q) load_t(buf, sub, n + GA + q, x[(n / GA + 1) & 1][q]);
                        }
                    }
                    const bf16x8 (&y)[PL] = x[(n / GA) & 1][n % GA];
                    const int k = n / DT, dt = n % DT;
#pragma unroll
                    for (int u = 0; u < UT; ++u) {
                        if constexpr (PL == 3) {
                            o[u][dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(y[2], w[u][k][0], o[u][dt], 0, 0, 0);
                            o[u][dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(y[0], w[u][k][2], o[u][dt], 0, 0, 0);
                            o[u][dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(y[1], w[u][k][1], o[u][dt], 0, 0, 0);
                            o[u][dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(y[1], w[u][k][0], o[u][dt], 0, 0, 0);
                            o[u][dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(y[0], w[u][k][1], o[u][dt], 0, 0, 0);
                        }
                        o[u][dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(y[0], w[u][k][0], o[u][dt], 0, 0, 0);
                    }
                }
            }
        }
        commit(buf ^ 1);
    };
    for (int32_t t = t0; t < t1; t += 2) {
        walk(t, std::integral_constant<int, 0>());
        if (t + 1 < t1) walk(t + 1, std::integral_constant<int, 1>());
    }

#pragma unroll
    for (int u = 0; u < UT; ++u) {
        const int32_t row = st0 + 32 * u + col;
        if (MODE != TABLE && sum[u] == UNSET) sum[u] = 0.f;
        const float both = sum[u] + __shfl_xor(sum[u], 32, 64);
        if (row >= n_st) continue;
        const int64_t out = (int64_t)split * n_st + row;
        if (kh == 0) {
            if constexpr (MODE != TABLE) {
                a.part_m[out] = m[u];
                a.part_s[out] = both;
            } else if (a.part_s) {
                if (a.part_o) a.part_s[out] = both;
                else a.out_b[row] = both * a.weight;
            }
        }
        if constexpr (MODE != LOSS) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int c = 32 * dt + 8 * j + 4 * kh;
                    if (MODE == LOSS_SUMS || a.part_o) {
                        f32x4 v;
#pragma unroll
                        for (int i = 0; i < 4; ++i) v[i] = o[u][dt][4 * j + i];
                        *(f32x4 *)(a.part_o + out * DP + c) = v;
                    } else if (c < a.d) {
                        T *dst = (T *)a.out + (int64_t)row * a.d + c;
                        float v[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) v[i] = o[u][dt][4 * j + i] * a.out_f;
                        if (c + 4 <= a.d) store_vec<4>(dst, v);
                        else {
#pragma unroll
                            for (int i = 0; i < 4; ++i) if (c + i < a.d) store_f32(dst + i, v[i]);
                        }
                    }
                }
        }
    }
}

// rows -> planes of bf16, dp wide, columns from d on zero; the x rows that take no part (targets) and the items that are out of
// the catalogue (bias) are zero, whatever they hold.  Both sides in one launch (1000 x 3706 x 40 step: 49 -> 47 us).  Bound by memory:
// 59047 rows of 100 bf16, 27 MB: 9 us.
struct PlaneJob {
    Rows src;
    const int32_t *targets;             // of x rows, else NULL
    const float *bias;                  // of items, may be NULL
    __bf16 *dst;
};
template <typename T, int PL>
__global__ __launch_bounds__(256) void k_planes(const PlaneJob x, const PlaneJob w, int64_t x_groups, int32_t n_items, int32_t d, int32_t dp)
{
    const bool is_x = group_id() < x_groups;
    const PlaneJob &job = is_x ? x : w;
    const int32_t per = dp / 8, n = job.src.n;
    const int64_t p = (group_id() - (is_x ? 0 : x_groups)) * 256 + threadIdx.x;
    if (p >= (int64_t)n * per) return;
    const int64_t r = p / per;
    const int32_t c = (int32_t)(p - r * per) * 8;
    const bool live = is_x ? (uint32_t)job.targets[r] < (uint32_t)n_items : !job.bias || job.bias[r] != -INFINITY;
    Piece<T> raw;
    bf16x8 v[PL];
    load_piece((const T *)job.src.p + r * job.src.stride, c, d, raw);
    split_piece(raw, live, v);
#pragma unroll
    for (int q = 0; q < PL; ++q) *(bf16x8 *)(job.dst + (int64_t)q * n * dp + r * dp + c) = v[q];
}

struct JoinArgs {
    int64_t n, n_items, x_stride, w_stride;
    int32_t d, dp, splits;
    float scale, weight;
    const int32_t *targets;
    const float *bias, *weights, *part_m, *part_s, *part_o;
    float *loss, *lse, *row_init, *row_q, *row_g;     // row_init NULL: no gradients
};

// W waves a row (one, or four where there are many parts): joins the parts of the items' axis, adds the target's own term and
// writes loss, lse, the row's dX and what pass 2 needs of the row.  Bound by the parts' bytes where there are many rows (4096 rows
// of 256, 8 parts: 18 us), by a chain of loads where there are few (1000 rows of 40 in 32 parts: 7 us).
template <typename T, int W>
__global__ __launch_bounds__(64 * W) void k_join_rows(const JoinArgs a, const T *__restrict__ x, const T *__restrict__ w, T *__restrict__ dx)
{
    __shared__ float sums[W][256];
    const int64_t r = group_id();
    if (r >= a.n) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int32_t t = a.targets[r];
    const bool in = (uint32_t)t < (uint64_t)a.n_items;
    if (!in) {
        if (wave) return;
        if (lane == 0) {
            a.loss[r] = a.lse[r] = t < 0 ? 0.f : NAN;
            if (a.row_init) { a.row_init[r] = -INFINITY; a.row_q[r] = 0.f; if (a.row_g) a.row_g[r] = 0.f; }
        }
        if (dx) for (int c = lane; c < a.d; c += 64) store_f32(dx + r * a.d + c, 0.f);
        return;
    }
    const float bias = a.bias ? a.bias[t] : 0.f;
    float z = -INFINITY;                                       // the target's logit, log2
    const bool out = bias * LOG2E == -INFINITY;                // the target is out of the catalogue
    if (!out) {
        float dot = 0.f;
        for (int c = lane; c < a.d; c += 64) dot = fmaf(load_f32(x + r * a.x_stride + c), load_f32(w + (int64_t)t * a.w_stride + c), dot);
        z = (wave_sum(dot) * a.scale + bias) * LOG2E;
        if (z == INFINITY) z = NAN;                            // inf - inf: pass 1, which leaves the target out, does not show it
    }
    // The largest part's sum, log2.  Not the largest of the parts' references: a sum may stand 2^60 above its own
    float m = -INFINITY;
    bool bad = false;
    for (int s = lane; s < a.splits; s += 64) {
        const float v = a.part_s[(int64_t)s * a.n + r];
        m = fmaxf(m, a.part_m[(int64_t)s * a.n + r] + __builtin_amdgcn_logf(v));
        bad |= !(v >= 0.f);                                    // not a number
    }
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) m = fmaxf(m, __shfl_xor(m, k, 64));
    const float top = fmaxf(m, z);
    const bool none = out && !__ballot(bad);                   // no gradient
    const bool empty = none && m == -INFINITY;
    // Everything relative to the largest of the target's exponential and the parts' sums: a part's sum and its weighted sums are
    // then multiplied by no more than what makes that sum at most 1.  Where it is the target's the loss is log1p(others), with no
    // difference of nearly equal numbers in it; elsewhere it is a sum of two numbers of one sign
    const bool near = z > m;
    const float ref = near ? z : (top == -INFINITY ? 0.f : top);
    float sum = 0.f;
    for (int s = lane; s < a.splits; s += 64) sum += a.part_s[(int64_t)s * a.n + r] * __builtin_amdgcn_exp2f(a.part_m[(int64_t)s * a.n + r] - ref);
    const float others = wave_sum(sum), own = __builtin_amdgcn_exp2f(z - ref), all = others + own;
    const float log_all = near ? log1pf(others) : logf(all);
    const float loss = none ? INFINITY : (near ? log_all : log_all + (ref - z) * LN2);
    const float q = none ? 0.f : others / all;                 // 1 - p_t
    if (lane == 0 && wave == 0) {
        a.loss[r] = loss;
        a.lse[r] = empty ? -INFINITY : log_all + ref * LN2;
    }
    if (!a.row_init) return;
    const float g = a.weights ? a.weights[r] : 1.f;
    if (lane == 0 && wave == 0) {
        a.row_init[r] = none ? -INFINITY : -((log_all + ref * LN2) / a.scale);
        a.row_q[r] = none ? 0.f : q * g;
        if (a.row_g) a.row_g[r] = none ? 0.f : g;
    }
    // four columns a lane, the parts dealt to 64 / lanes groups of lanes
    const float f = g * a.weight * a.scale;
    const int lanes = a.dp > 128 ? 64 : a.dp > 64 ? 32 : a.dp > 32 ? 16 : 8;        // dp = 192: 48 of 64 busy
    const int c = lane % lanes * 4, step = 64 / lanes;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (c < a.dp) {
#pragma unroll 8
        for (int s = wave * step + lane / lanes; s < a.splits; s += W * step) {
            const float w2 = __builtin_amdgcn_exp2f(a.part_m[(int64_t)s * a.n + r] - ref);
            const f32x4 p = *(const f32x4 *)(a.part_o + ((int64_t)s * a.n + r) * a.dp + c);
            v += p * w2;
        }
    }
    for (int k = lanes; k < 64; k <<= 1)
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += __shfl_xor(v[i], k, 64);
    if constexpr (W > 1) {
        if (lane < lanes && c < a.dp) *(f32x4 *)(sums[wave] + c) = v;
        __syncthreads();
        if (wave) return;
        if (lane < lanes && c < a.dp)
#pragma unroll
            for (int k = 1; k < W; ++k) v += *(const f32x4 *)(sums[k] + c);
    }
    if (lane < lanes)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (c + i < a.d) {
                const float out = none ? 0.f : f * (v[i] / all - q * load_f32(w + (int64_t)t * a.w_stride + c + i));
                store_f32(dx + r * a.d + c + i, out);
            }
}

// the parts of the rows' axis of pass 2, summed in order: dW and db.  Four columns a thread.
template <typename T>
__global__ __launch_bounds__(256) void k_join_items(const float *__restrict__ part_o, const float *__restrict__ part_s, int32_t splits,
                                                    int64_t n_items, int32_t d, int32_t dp, float f, float weight, T *__restrict__ dw,
                                                    float *__restrict__ db)
{
    const int32_t per = (d + 3) / 4;
    const int64_t p = group_id() * 256 + threadIdx.x;
    if (p >= n_items * per) return;
    const int64_t v = p / per;
    const int32_t c = (int32_t)(p - v * per) * 4;
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int k = 0; k < splits; ++k) s += *(const f32x4 *)(part_o + ((int64_t)k * n_items + v) * dp + c);
    float o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = s[i] * f;
    if (c + 4 <= d) store_vec<4>(dw + v * d + c, o);
    else
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (c + i < d) store_f32(dw + v * d + c + i, o[i]);
    if (db && c == 0) {
        float t = 0.f;
        for (int k = 0; k < splits; ++k) t += part_s[(int64_t)k * n_items + v];
        db[v] = t * weight;
    }
}

// Workgroups of a pass at once on the chip, stationary rows a workgroup and streamed rows a tile, by the kernel's shape
struct PassShape { int groups, rows, tile; };
template <int PL, int MODE, bool CONV>
PassShape pass_shape_d(int dp)
{
#define MF_SHAPE(DP_) case DP_: { using S = Shape<DP_, PL, MODE, CONV>; return {256 * S::GROUPS, S::ROWS, S::TB}; }
    switch (dp) { MF_SHAPE(32) MF_SHAPE(64) MF_SHAPE(128) MF_SHAPE(192) default: MF_SHAPE(256) }
#undef MF_SHAPE
}
template <int PL>
PassShape pass_shape(int dp, int mode, bool conv)
{
    if (mode == LOSS) return conv ? pass_shape_d<PL, LOSS, true>(dp) : pass_shape_d<PL, LOSS, false>(dp);
    if (mode == LOSS_SUMS) return conv ? pass_shape_d<PL, LOSS_SUMS, true>(dp) : pass_shape_d<PL, LOSS_SUMS, false>(dp);
    return conv ? pass_shape_d<PL, TABLE, true>(dp) : pass_shape_d<PL, TABLE, false>(dp);
}

// Parts the streamed axis is cut into: the number with the least time by this reckoning.  A workgroup takes 12 us to start and
// end.  Of a tile it takes alone_us where it has its share of a full CU; with q workgroups a CU that is alone_us sqrt(q^2 + c^2),
// as measured with one to three of them: fp32 rows (c = 1) keep the matrix cores busy with one, bf16 rows (c = 3), with one
// product an operand, wait for LDS and memory.  A part's sums are written and read again at 8 TB/s; pass 2 joins its parts in a
// launch of its own.
int parts_of(int64_t n_sm, int64_t n_st, int64_t row_tiles, const PassShape &s, int dp, int products, bool sums, bool pass2)
{
    static const int counts[] = {1, 2, 3, 4, 5, 6, 7, 8, 16, 24, 32, 48, 64, 96, 128, 192, 256, 384, 512, 768, 1024};
    const double alone_us = 2.0 * s.rows * s.tile * dp * products / 4.2e6, c = products >= 6 ? 1.0 : 3.0;
    const double part_us = (sums ? n_st * (double)dp * 8 / 8e6 : 0.0) + 0.015;
    const int64_t tiles = (n_sm + s.tile - 1) / s.tile;
    int best = 1;
    double least = 1e300;
    for (int k : counts) {
        if (k > tiles) break;
        const double rounds = (double)((row_tiles * k + s.groups - 1) / s.groups);
        const double q = std::min(row_tiles * k / 256.0, s.groups / 256.0);
        const double us = rounds * ((double)((tiles + k - 1) / k) * alone_us * sqrt(q * q + c * c) + 12.0) + (k > 1 ? k * part_us + 5.0 * pass2 : 0.0);
        if (us < least) { least = us; best = k; }
    }
    return best;
}

struct LossPlan {
    int dp, planes, splits1, rt1, splits2, rt2;
    bool conv, as_is;
    int64_t xp, wp, m1, s1, o1, init, q, g, s2, o2, bytes;
};

// Rows that start at multiples of 16 bytes, near enough for the tiles' 32-bit offsets
bool rows_aligned(const void *p, int64_t stride) { return (uintptr_t)p % 16 == 0 && stride % 8 == 0 && stride < (1 << 20); }

// aligned: the table's rows are (rows_aligned)
LossPlan loss_plan(int64_t n, int64_t n_items, int32_t d, int32_t dtype, bool grads, bool aligned)
{
    LossPlan p = {};
    n = std::max<int64_t>(n, 1);
    p.dp = d <= 32 ? 32 : d <= 64 ? 64 : d <= 128 ? 128 : d <= 192 ? 192 : 256;
    p.planes = dtype == MFSGD_F32 ? 3 : 1;
    p.as_is = p.planes == 1 && d == p.dp && aligned;           // a bf16 table whose rows are dp wide is the operand as it is
    const int mode1 = grads ? LOSS_SUMS : LOSS;
    auto shape = [&](int mode, bool conv) { return p.planes == 3 ? pass_shape<3>(p.dp, mode, conv) : pass_shape<1>(p.dp, mode, conv); };
    // Few row tiles convert the rows they stream on the way: a launch and a round trip to memory less (200 x 162541 x 64 fp32
    // step: 150 -> 143 us; with 8 row tiles nothing is gained, with more it costs).  fp32 rows of 256 with gradients leave no
    // registers for it.
    p.conv = n <= 4 * shape(mode1, true).rows && !(p.planes == 3 && p.dp == 256 && grads);
    const PassShape s1 = shape(mode1, p.conv), s2 = shape(TABLE, p.conv);
    p.rt1 = (int)((n + s1.rows - 1) / s1.rows);
    const int six = p.planes == 3 ? 6 : 1;
    p.splits1 = parts_of(n_items, n, p.rt1, s1, p.dp, six * (grads ? 2 : 1), grads, false);
    p.rt2 = (int)((n_items + s2.rows - 1) / s2.rows);
    p.splits2 = parts_of(n, n_items, p.rt2, s2, p.dp, six * 2, true, true);
    int64_t at = 0;
    auto take = [&](int64_t bytes) { const int64_t o = at; at += align_up(bytes, 256); return o; };
    if (!p.conv) {
        if (grads) p.xp = take((int64_t)p.planes * n * p.dp * 2);
        if (!p.as_is) p.wp = take((int64_t)p.planes * n_items * p.dp * 2);
    }
    p.m1 = take((int64_t)p.splits1 * n * 4);
    p.s1 = take((int64_t)p.splits1 * n * 4);
    if (grads) {
        p.o1 = take((int64_t)p.splits1 * n * p.dp * 4);
        p.init = take(n * 4); p.q = take(n * 4); p.g = take(n * 4);
        if (p.splits2 > 1) {
            p.s2 = take((int64_t)p.splits2 * n_items * 4);
            p.o2 = take((int64_t)p.splits2 * n_items * p.dp * 4);
        }
    }
    p.bytes = std::max<int64_t>(at, 256);
    return p;
}

template <typename T, int DP, int MODE, bool CONV>
int launch_stream(const StreamArgs &a, hipStream_t st)
{
    auto kern = k_stream<T, DP, MODE, CONV>;
    constexpr int bytes = Shape<DP, sizeof(T) == 4 ? 3 : 1, MODE, CONV>::LDS;
    static_assert(bytes <= 160 * 1024, "a CU's LDS");
    if (bytes > 64 * 1024) MF_HIP(hipFuncSetAttribute((const void *)kern, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
    hipLaunchKernelGGL(kern, dim3((unsigned)(a.splits * a.row_tiles)), dim3(256), bytes, st, a);
    MF_LAUNCH_CHECK();
    return MFSGD_OK;
}

template <typename T, int MODE>
int launch_stream_d(int dp, bool conv, const StreamArgs &a, hipStream_t st)
{
#define MF_STREAM(DP_) case DP_: return conv ? launch_stream<T, DP_, MODE, true>(a, st) : launch_stream<T, DP_, MODE, false>(a, st);
    switch (dp) { MF_STREAM(32) MF_STREAM(64) MF_STREAM(128) MF_STREAM(192) }
#undef MF_STREAM
    if constexpr (sizeof(T) == 2 || MODE == LOSS) if (conv) return launch_stream<T, 256, MODE, true>(a, st);
    return launch_stream<T, 256, MODE, false>(a, st);
}

template <typename T>
int loss_impl(const T *x, int64_t xs, const T *w, int64_t ws_, const int32_t *targets, const float *bias, const float *weights, float weight,
              int64_t n, int64_t n_items, int32_t d, float scale, float *loss, float *lse, T *dx, T *dw, float *db, bool grads, char *ws,
              hipStream_t st)
{
    constexpr int PL = sizeof(T) == 4 ? 3 : 1;
    const LossPlan p = loss_plan(n, n_items, d, PL == 3 ? MFSGD_F32 : MFSGD_BF16, grads, rows_aligned(w, ws_));
    const Rows xr = {x, xs, (int32_t)n}, wr = {w, ws_, (int32_t)n_items};
    __bf16 *xp = (__bf16 *)(ws + p.xp), *wp = (__bf16 *)(ws + p.wp);
    if (!p.conv) {
        auto groups = [&](int64_t rows) { return (rows * (p.dp / 8) + 255) / 256; };
        const PlaneJob jx = {xr, targets, nullptr, xp}, jw = {wr, nullptr, bias, wp};
        const int64_t gx = grads ? groups(n) : 0, gw = p.as_is ? 0 : groups(n_items);
        if (gx + gw) hipLaunchKernelGGL((k_planes<T, PL>), grid_of(gx + gw), dim3(256), 0, st, jx, jw, gx, (int32_t)n_items, d, p.dp);
        MF_LAUNCH_CHECK();
    }

    StreamArgs a = {};
    a.d = d;
    a.n_items = (int32_t)n_items;
    a.targets = targets;
    a.bias = bias;
    a.c = scale * LOG2E;
    a.inv_scale = 1.f / scale;
    a.st = xr;
    a.sm = wr;
    a.sm_planes = p.as_is ? (const __bf16 *)w : wp;
    a.planes_stride = p.as_is ? ws_ : p.dp;
    a.plane = n_items * p.dp;
    a.clear = p.as_is && bias;
    a.splits = p.splits1; a.row_tiles = p.rt1;
    a.part_m = (float *)(ws + p.m1); a.part_s = (float *)(ws + p.s1); a.part_o = (float *)(ws + p.o1);
    if (const int rc = grads ? launch_stream_d<T, LOSS_SUMS>(p.dp, p.conv, a, st) : launch_stream_d<T, LOSS>(p.dp, p.conv, a, st)) return rc;

    JoinArgs j = {};
    j.n = n; j.n_items = n_items; j.x_stride = xs; j.w_stride = ws_; j.d = d; j.dp = p.dp; j.splits = p.splits1;
    j.scale = scale; j.weight = weight; j.targets = targets; j.bias = bias; j.weights = weights;
    j.part_m = a.part_m; j.part_s = a.part_s; j.part_o = a.part_o; j.loss = loss; j.lse = lse;
    if (grads) {
        j.row_init = (float *)(ws + p.init); j.row_q = (float *)(ws + p.q);
        j.row_g = weights ? (float *)(ws + p.g) : nullptr;
    }
    // four waves a row: 192 parts of one row 12 -> 5 us; one wave where the rows fill the chip
    if (grads && p.splits1 >= 32) hipLaunchKernelGGL((k_join_rows<T, 4>), grid_of(n), dim3(256), 0, st, j, x, w, dx);
    else hipLaunchKernelGGL((k_join_rows<T, 1>), grid_of(n), dim3(64), 0, st, j, x, w, dx);
    MF_LAUNCH_CHECK();
    if (!grads) return MFSGD_OK;

    a.st = wr;
    a.sm = xr;
    a.sm_planes = xp;
    a.planes_stride = p.dp;
    a.plane = n * p.dp;
    a.splits = p.splits2; a.row_tiles = p.rt2;
    a.part_m = nullptr;
    a.part_s = db ? (float *)(ws + p.s2) : nullptr;
    a.part_o = p.splits2 > 1 ? (float *)(ws + p.o2) : nullptr;
    a.row_init = j.row_init; a.row_q = j.row_q; a.row_g = j.row_g;
    a.out = dw; a.out_b = db; a.out_f = scale * weight; a.weight = weight;
    if (const int rc = launch_stream_d<T, TABLE>(p.dp, p.conv, a, st)) return rc;
    if (p.splits2 > 1) {
        hipLaunchKernelGGL((k_join_items<T>), grid_of((n_items * ((d + 3) / 4) + 255) / 256), dim3(256), 0, st, a.part_o, a.part_s, p.splits2, n_items,
                           d, p.dp, scale * weight, weight, dw, db);
        MF_LAUNCH_CHECK();
    }
    return MFSGD_OK;
}

int check_loss(const char *who, const void *x, int64_t xs, const void *w, int64_t ws_, const int32_t *targets, int64_t n, int64_t n_items,
               int32_t d, float scale, int32_t dtype, const float *loss, const float *lse, void *ws, int64_t ws_bytes, bool grads)
{
    MF_ARG(n >= 0 && n <= INT32_MAX / 4 && n_items >= 1 && n_items <= INT32_MAX / 4 && d >= 1 && d <= 256 && xs >= d && ws_ >= d,
           "%s: bad shape (1 <= d <= 256, at least one item, rows and items below 2^29)", who);
    MF_ARG(dtype == MFSGD_F32 || dtype == MFSGD_BF16, "%s: unknown dtype %d", who, dtype);
    MF_ARG(scale >= 1e-20f && scale <= 1e20f, "%s: scale must be from 1e-20 to 1e20", who);
    if (n == 0 && !grads) return MFSGD_OK;
    MF_ARG(w && (n == 0 || (x && targets && loss && lse)), "%s: null pointer", who);
    const int64_t need = loss_plan(n, n_items, d, dtype, grads, rows_aligned(w, ws_)).bytes;
    MF_ARG(ws && (uintptr_t)ws % 16 == 0 && ws_bytes >= need, "%s: needs a 16-byte aligned workspace of %lld bytes", who, (long long)need);
    return MFSGD_OK;
}

template <typename T>
__global__ __launch_bounds__(256) void k_zero(T *__restrict__ p, int64_t n)
{
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) store_f32(p + i, 0.f);
}

}  // namespace

extern "C" {

int64_t mfsgd_softmax_loss_workspace(int64_t n, int64_t n_items, int32_t d, int32_t dtype, int32_t flags)
{
    if (n < 0 || n > INT32_MAX / 4 || n_items < 1 || n_items > INT32_MAX / 4 || d < 1 || d > 256 || (dtype != MFSGD_F32 && dtype != MFSGD_BF16))
        return -1;
    return loss_plan(n, n_items, d, dtype, flags & MFSGD_WITH_GRADS, flags & MFSGD_TABLE_ALIGNED).bytes;
}

int mfsgd_hip_softmax_loss(const void *x, int64_t x_stride, const void *table, int64_t table_stride, const int32_t *targets, const float *bias,
                           int64_t n, int64_t n_items, int32_t d, float scale, int32_t dtype, float *loss, float *lse, void *workspace,
                           int64_t workspace_bytes, void *stream)
{
    if (const int rc = check_loss("softmax_loss", x, x_stride, table, table_stride, targets, n, n_items, d, scale, dtype, loss, lse, workspace,
                                  workspace_bytes, false)) return rc;
    if (n == 0) return MFSGD_OK;
    if (dtype == MFSGD_F32)
        return loss_impl<float>((const float *)x, x_stride, (const float *)table, table_stride, targets, bias, nullptr, 1.f, n, n_items, d, scale,
                                   loss, lse, nullptr, nullptr, nullptr, false, (char *)workspace, as_stream(stream));
    return loss_impl<__bf16>((const __bf16 *)x, x_stride, (const __bf16 *)table, table_stride, targets, bias, nullptr, 1.f, n, n_items, d, scale,
                                loss, lse, nullptr, nullptr, nullptr, false, (char *)workspace, as_stream(stream));
}

int mfsgd_hip_softmax_loss_grads(const void *x, int64_t x_stride, const void *table, int64_t table_stride, const int32_t *targets,
                                 const float *bias, const float *weights, float weight, int64_t n, int64_t n_items, int32_t d, float scale,
                                 int32_t dtype, float *loss, float *lse, void *dx, void *dtable, float *dbias, void *workspace,
                                 int64_t workspace_bytes, void *stream)
{
    if (const int rc = check_loss("softmax_loss_grads", x, x_stride, table, table_stride, targets, n, n_items, d, scale, dtype, loss, lse, workspace,
                                  workspace_bytes, true)) return rc;
    MF_ARG(dtable && (n == 0 || dx), "softmax_loss_grads: null pointer");
    hipStream_t st = as_stream(stream);
    if (n == 0) {       // no rows: the table's gradients are zero
        const unsigned grid = (unsigned)std::min<int64_t>((n_items * d + 255) / 256, 4096);
        if (dtype == MFSGD_F32) hipLaunchKernelGGL((k_zero<float>), dim3(grid), dim3(256), 0, st, (float *)dtable, n_items * d);
        else hipLaunchKernelGGL((k_zero<__bf16>), dim3(grid), dim3(256), 0, st, (__bf16 *)dtable, n_items * d);
        if (dbias) hipLaunchKernelGGL((k_zero<float>), dim3(grid), dim3(256), 0, st, dbias, n_items);
        MF_LAUNCH_CHECK();
        return MFSGD_OK;
    }
    if (dtype == MFSGD_F32)
        return loss_impl<float>((const float *)x, x_stride, (const float *)table, table_stride, targets, bias, weights, weight, n, n_items, d,
                                   scale, loss, lse, (float *)dx, (float *)dtable, dbias, true, (char *)workspace, st);
    return loss_impl<__bf16>((const __bf16 *)x, x_stride, (const __bf16 *)table, table_stride, targets, bias, weights, weight, n, n_items, d,
                                scale, loss, lse, (__bf16 *)dx, (__bf16 *)dtable, dbias, true, (char *)workspace, st);
}

}  // extern "C"
