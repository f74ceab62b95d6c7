// Attention over key ranges, forward and backward, head_dim 64 / 128, shared key heads.
//
// Row i of batch entry b sees the keys of [a_lo, a_hi) and [b_lo, b_hi).  With z = q.k scale, c = cap tanh(z / cap) (or z),
// t = c + bias[h][clamp(j - pos_i)]:
//     forward    P = exp(t - lse), lse = log sum over visible keys of exp t, O = P V
//     backward   dV = P^T dO, dP = dO V^T, dT = P (dP - delta), delta = sum_c dO O, dbias = sum of dT by distance,
//                dZ = dT (1 - (c / cap)^2), dQ = scale dZ K, dK = scale dZ^T Q
// Scores live in base 2 (t log2 e), maxima and sums in 32 bits; P and dZ are rounded to bf16 once, as operands of the next
// matrix product (at most 2^-8 of each weight, like the rounding of the result itself).
//
// All products are 32 x 32 x 16 MFMAs in the "swapped" form: the result of the first product has the long axis of the second
// one's contraction in its registers (rows 4 (l / 32) + 8 (r / 4) + r % 4 of lane l, register r), which is how the second
// product wants its B operand if its A operand is read with the same permutation -- ds_read_b64_tr_b16 on the row-major LDS
// tile does that.  So P and dZ never leave the registers.  Tiles arrive by 16-byte LDS-DMA into a layout whose 16-byte chunks
// are XOR-swizzled by row so that both kinds of reads hit all banks (swz below).
//
// A hidden key must not reach a row's result even as 0 x inf: the matrix products cannot tell, so a result row that came out
// non-finite although some of the row's keys were hidden (by a range or by the bias) is recomputed by a plain loop over its
// visible keys (exact_*), which ends early where every channel is NaN anyway.
#include <type_traits>
#include "common.h"
#include "pyflow_hip.h"
#include "rows_view.h"

int pf_set_err(const char* m);

namespace {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f, HIDDEN = -1.0e30f;
constexpr float DEFER = 6.0f;          // the running maximum follows when a row outgrows it by 2^6: P stays below 64
constexpr int MAX_RADIUS = 512;        // the bias table and four accumulators of its gradient share LDS with the tiles

typedef short s4_t __attribute__((ext_vector_type(4)));
typedef short s8_t __attribute__((ext_vector_type(8)));

struct View { bf16_t* p; long long bs, ld, hs; };

struct RArgs {
    View q, k, v, o, dO, dq, dk, dv;
    float* lse;
    const int* a_lo; const int* a_hi; const int* b_lo; const int* b_hi; long long range_bs;
    const int* q_pos; long long pos_bs;
    const float* bias; int R;
    // z = q.k.  Scores in base 2 are x zs + shift with x = z (uncapped), x = cap_u(z zc) (cap) or x = tanh(z zc) (SERIES);
    // the shift is left out wherever only differences of scores count
    float zs, zc, shift, cap2;
    float zn, shift_n;                 // zs and shift in natural units
    float scale, dscale;               // dQ, dK = dscale times the products of dZ (4 scale with cap_u's slope)
    int series;
    int D, B, H, Hk, G, Lq, Lk;
    int nqt, nkt, nrb, nsplit;
    int key_wgs, key_pad;              // backward: workgroups for the key gradients, the first of those for the row gradients
    float* parts;                      // split forward: [unit][split][32][D + 2]
    float* stat;                       // backward: [B][H][nq64][4][64] lse log2 e - shift, -delta, position, the tile's positions
    int* vis;                          // backward: [B][nq64][4][64] the rows' ranges (Vis)
    int* tiles;                        // backward: [B][nq64][8] bounds of 64-row tiles
    int nq64;
    float* kv_parts; int kv_split;     // backward: [part][B][Hk][Lk][2][D] unscaled dK, dV of a part of the rows
    float* dbias_parts; float* dbias;  // backward: [B][H][nqt][2 R + 1]
};

// ---------------------------------------------------------------------------------------------- visibility
struct Vis { int alo, na, blo, nb; };          // keys [alo, alo + na) and [blo, blo + nb), inside [0, Lk)

PF_DEVICE Vis load_vis(const RArgs& p, int b, int row) {
    Vis v = {0, 0, 0, 0};
    if (row >= p.Lq) return v;
    if (!p.a_lo) {
        v.na = p.Lk;
        return v;
    }
    const long long at = b * p.range_bs + row;
    const auto inside = [&](int x) { return min(max(x, 0), p.Lk); };          // any integers: clipped before they are subtracted
    v.alo = inside(p.a_lo[at]);
    v.na = max(inside(p.a_hi[at]) - v.alo, 0);
    if (v.na == 0) v.alo = 0;
    if (p.b_lo) {
        v.blo = inside(p.b_lo[at]);
        v.nb = max(inside(p.b_hi[at]) - v.blo, 0);
        if (v.nb == 0) v.blo = 0;
    }
    return v;
}
PF_DEVICE bool sees(const Vis& v, int key) {
    return (unsigned)(key - v.alo) < (unsigned)v.na || (unsigned)(key - v.blo) < (unsigned)v.nb;
}

// over the wave, as a scalar: four cross-lane moves inside each row of 16 lanes, then one lane of each row (64-lane butterflies
// through LDS are 6 round trips each, and a workgroup starts with eight of these)
template <int CTRL>
PF_DEVICE int dpp(int x) { return __builtin_amdgcn_update_dpp(x, x, CTRL, 0xf, 0xf, false); }
template <typename F>
PF_DEVICE int wave_fold(int x, F f) {
    x = f(x, dpp<0xB1>(x));                    // lanes 1 0 3 2
    x = f(x, dpp<0x4E>(x));                    // lanes 2 3 0 1
    x = f(x, dpp<0x141>(x));                   // halves of 8 mirrored
    x = f(x, dpp<0x140>(x));                   // 16 mirrored
    auto at = [&](int lane) { return __builtin_amdgcn_readlane(x, lane); };
    return f(f(at(0), at(16)), f(at(32), at(48)));
}
PF_DEVICE int wave_min(int x) { return wave_fold(x, [](int a, int b) { return min(a, b); }); }
PF_DEVICE int wave_max(int x) { return wave_fold(x, [](int a, int b) { return max(a, b); }); }
PF_DEVICE float wave_add(float x) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) x += __shfl_xor(x, o);
    return x;
}

// the rows of memory that a tile may be filled from: [a0, a1) and [b0, b1) (an empty one: 0, 0)
struct Cover {
    int a0, a1, b0, b1;
    PF_DEVICE bool has(int j) const { return (unsigned)(j - a0) < (unsigned)(a1 - a0) || (unsigned)(j - b0) < (unsigned)(b1 - b0); }
    PF_DEVICE bool whole(int j0, int j1) const { return (a0 <= j0 && a1 >= j1) || (b0 <= j0 && b1 >= j1); }
    PF_DEVICE int some(int j0, int j1) const { return max(j0, a0 < j1 && a1 > j0 ? a0 : b0); }      // one of them in [j0, j1), which has one
};
PF_DEVICE Cover scalar(const Cover& c) {       // the same in every lane
    auto one = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
    return {one(c.a0), one(c.a1), one(c.b0), one(c.b1)};
}
// the key tiles (of KB keys) that a set of rows needs: the union of its two key ranges' tiles, each tile once
struct TileList {
    int s0, n0, s1, n;                         // tiles s0 .. s0 + n0 - 1, then s1 .. ; n in all
    Cover keys;
    PF_DEVICE int at(int i) const { return i < n0 ? s0 + i : s1 + (i - n0); }
    // at no end of a run: all of its keys are in the cover, which the loops then need not keep in registers
    PF_DEVICE bool inner(int i) const { return i > 0 && i < n - 1 && (unsigned)(i + 1 - n0) > 1u; }
};
template <int KB>
PF_DEVICE TileList tile_list(int amin, int amax, int bmin, int bmax) {
    int as = 0, ae = 0, bs = 0, be = 0;
    Cover keys = {0, 0, 0, 0};
    if (amax > amin) { as = amin / KB; ae = (amax + KB - 1) / KB; keys.a0 = amin; keys.a1 = amax; }
    if (bmax > bmin) { bs = bmin / KB; be = (bmax + KB - 1) / KB; keys.b0 = bmin; keys.b1 = bmax; }
    if (ae == as) { as = bs; ae = be; bs = be = 0; }
    if (be > bs) {
        if (bs < as) { int t = as; as = bs; bs = t; t = ae; ae = be; be = t; }
        bs = max(bs, ae);
        be = max(be, bs);
    }
    return {as, ae - as, bs, (ae - as) + (be - bs), keys};
}

template <int D, int KS>
constexpr int FWD_KB = D == 64 || KS == 2 ? 64 : 32;     // keys of a forward tile
// waves per SIMD the registers are cut for: latency is what is left over (D = 128, 16 heads of 8000 rows: 3 waves and two tiles
// in LDS 576 us, 2 waves 624 us, 2 waves and three tiles 613 us)
template <int D, int KS>
constexpr int FWD_WAVES = D == 64 ? 4 : KS == 1 ? 3 : 2;

// ---------------------------------------------------------------------------------------------- LDS tiles
// Row-major bf16 rows of D channels, 16-byte chunk c of row r at c ^ swz(r).  A row read (ds_read_b128, one chunk of 16
// consecutive rows per 256 bytes) needs swz to differ over 16 rows modulo the row pitch; a transposed read
// (ds_read_b64_tr_b16: four chunks of four consecutive rows) needs swz to move those four rows to different quarters.
template <int D>
PF_DEVICE int swz(int r) {
    if constexpr (D == 64) return ((r & 2) << 1) | ((r & 4) >> 1) | ((r & 8) >> 3);
    else return ((r & 3) << 2) | ((r >> 2) & 3);
}

// Rows [row0, row0 + ROWS) of a head -> LDS, by the NW waves that share the tile.  A lane's 32-bit byte offsets inside a tile are
// fixed, the tile's base is wave-uniform: no vector arithmetic per tile (64-bit addresses per piece were a sixth of the forward
// kernel's vector instructions).  Rows outside the cover repeat one inside it (hidden later): what a cache holds in slots that nobody
// sees does not even arrive, so that infinities and NaN there cost nothing (NaN behind the last key, the same times as with zeros there,
// and before, when they were read and rows computed again: 16 rows over 30000 keys of 32 / 8 heads of 128 340 us, 13.5 ms; 2 x 512 rows
// over 470 keys of 64 heads of 64 22 us, 2.2 ms.  The tests of a tile's place cost 1 % of 15488 rows of 30 heads of 64).  Row strides
// are below 2^25 elements (host check).
template <int D, int ROWS, int NW>
struct Stager {
    static constexpr int LPR = D / 8, RPP = 64 / LPR, N = ROWS / RPP / NW;     // lanes per row, rows per 1-KiB piece
    static_assert(N >= 1 && N * RPP * NW == ROWS, "the tile is a whole number of pieces per wave");
    unsigned off[N];
    PF_DEVICE Stager(long long ld, int wid, int lane) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int r = (wid * N + j) * RPP + lane / LPR;
            off[j] = (unsigned)r * (unsigned)(2 * ld) + (unsigned)(((lane % LPR) ^ swz<D>(r)) * 16);
        }
    }
    PF_DEVICE void whole(const bf16_t* head, long long ld, int row0, char* lds, int wid) const {
        const char* base = (const char*)(head + row0 * ld);
#pragma unroll
        for (int j = 0; j < N; ++j) glds16(base + off[j], lds + (wid * N + j) * 1024);
    }
    PF_DEVICE void part(const bf16_t* head, long long ld, int row0, const Cover& rows, char* lds, int wid, int lane) const {
        const char* base = (const char*)(head + row0 * ld);
        const int spare = rows.some(row0, row0 + ROWS) - row0;
        asm volatile("" : "+v"(lane));         // what follows from it is worked out here, not kept in registers through the caller's loop
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int r = (wid * N + j) * RPP + lane / LPR, from = rows.has(row0 + r) ? r : spare;
            const unsigned o = (unsigned)from * (unsigned)(2 * ld) + (unsigned)(((lane % LPR) ^ swz<D>(r)) * 16);
            glds16(base + o, lds + (wid * N + j) * 1024);
        }
    }
    // rows up to `last`, which those behind it repeat
    PF_DEVICE void upto(const bf16_t* head, long long ld, int row0, int last, char* lds, int wid, int lane) const {
        if (row0 + ROWS - 1 <= last) return whole(head, ld, row0, lds, wid);
        const char* base = (const char*)(head + row0 * ld);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int r = (wid * N + j) * RPP + lane / LPR;
            const unsigned o = (unsigned)min(r, last - row0) * (unsigned)(2 * ld) + (unsigned)(((lane % LPR) ^ swz<D>(r)) * 16);
            glds16(base + o, lds + (wid * N + j) * 1024);
        }
    }
};

// Wave-uniform bounds of the ranges of a wave's rows: any key of [j0, j1) seen by some row; all of them by every row (a
// sufficient test: rows that cover it by different ranges count as partial)
struct Bounds {
    int amin, amax, bmin, bmax;                // over the ranges that are not empty
    int alo, ahi, blo, bhi;                    // largest start, smallest end over all rows (an empty range: none)
    PF_DEVICE bool any(int j0, int j1) const { return (amin < j1 && amax > j0) || (bmin < j1 && bmax > j0); }
    PF_DEVICE bool full(int j0, int j1) const { return (alo <= j0 && ahi >= j1) || (blo <= j0 && bhi >= j1); }
};
PF_DEVICE Bounds wave_bounds(const Vis& v) {
    constexpr int BIG = 0x7fffffff;
    return {wave_min(v.na ? v.alo : BIG), wave_max(v.na ? v.alo + v.na : 0), wave_min(v.nb ? v.blo : BIG), wave_max(v.nb ? v.blo + v.nb : 0),
            wave_max(v.na ? v.alo : BIG), wave_min(v.na ? v.alo + v.na : 0), wave_max(v.nb ? v.blo : BIG), wave_min(v.nb ? v.blo + v.nb : 0)};
}
// the key tiles of a workgroup of 4 waves (`red`: 16 ints of LDS, read behind a barrier; `cover`: 4 for all waves to leave the same in)
template <int KB>
PF_DEVICE TileList workgroup_tiles(const Bounds& w, int* red, Cover* cover, int wid, int lane) {
    if (lane == 0) { red[4 * wid] = w.amin; red[4 * wid + 1] = w.amax; red[4 * wid + 2] = w.bmin; red[4 * wid + 3] = w.bmax; }
    __syncthreads();
    int x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[i] = red[i];
#pragma unroll
        for (int u = 1; u < 4; ++u) x[i] = (i & 1) ? max(x[i], red[4 * u + i]) : min(x[i], red[4 * u + i]);
        x[i] = __builtin_amdgcn_readfirstlane(x[i]);
    }
    const TileList t = tile_list<KB>(x[0], x[1], x[2], x[3]);
    *cover = t.keys;
    return t;
}

// A operand of a product over channels: row lane % 32 (+ 32 i), channels 16 ks + 8 (lane / 32) ..
template <int D>
PF_DEVICE unsigned row_offset(int lane) {
    const int r = lane & 31, hi = lane >> 5;
    return (unsigned)(r * (2 * D) + ((hi ^ swz<D>(r)) << 4));
}
template <int D>
PF_DEVICE bf16x8_t row_frag(const char* tile, unsigned off, int i, int ks) {
    return *(const bf16x8_t*)(tile + i * (64 * D) + (off ^ (unsigned)(ks << 5)));
}
// A operand of a product over rows: channel lane % 32 (+ 32 c), rows 16 g + 4 (lane / 32) + {0..3} and + 8
template <int D>
PF_DEVICE unsigned tr_offset(int lane, int plus) {
    const int r = 4 * (lane >> 5) + ((lane & 15) >> 2) + plus;
    const int c = ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
    return (unsigned)(r * (2 * D) + ((c ^ swz<D>(r)) << 4) + 8 * (lane & 1));
}
template <int D>
PF_DEVICE bf16x8_t tr_frag(const char* tile, unsigned off0, unsigned off8, int c, int g) {
    const char* t = tile + g * (32 * D);
    const s4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4_t*)(t + (off0 ^ (unsigned)(c << 6))));
    const s4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4_t*)(t + (off8 ^ (unsigned)(c << 6))));
    return __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

// LDS-DMA is not ordered by the compiler's own counts: everything issued so far has landed, every LDS read has returned
PF_DEVICE void drain() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory"); }
PF_DEVICE void drain_barrier() {
    drain();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

PF_DEVICE f32x16_t mfma(bf16x8_t a, bf16x8_t b, f32x16_t c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
PF_DEVICE f32x16_t zero16() {
    f32x16_t z;
#pragma unroll
    for (int r = 0; r < 16; ++r) z[r] = 0.f;
    return z;
}
PF_DEVICE bf16x8_t half_of(const f32x16_t& s, int g) {
    bf16x8_t v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (bf16_t)s[8 * g + e];
    return v;
}
PF_DEVICE constexpr int reg_row(int r) { return (r & 3) + 8 * (r >> 2); }      // + 4 (lane / 32)

PF_DEVICE float other_half(float x) {
    const auto w = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return (threadIdx.x & 32) ? __uint_as_float(w[0]) : __uint_as_float(w[1]);
}

// ---------------------------------------------------------------------------------------------- scores
// cap tanh(z / cap) = cap (1 + 2 u) with u = -1 / (1 + 2^(z zc)), zc = 2 scale log2 e / cap: the kernels keep u where an uncapped
// score would be (its factor is 2 cap log2 e), and the slope 1 - tanh^2 = -4 (u + u^2).  That leaves up to 3 x 2^-23 of the CAP in the
// score: nothing that a weight in bf16 shows for caps up to 64, but a 32-bit log-sum-exp does (one visible key, cap 64: 3e-6 rms, where
// tanh leaves 2e-7; 30 keys, cap 30: 7e-7 and 4e-7).  SERIES (larger caps, the bias's gradient, and whoever asks for it) takes tanh
// itself, below |x| = 0.3 by its odd series (next term 0.0089 x^10: 5e-8): 158 instead of 128 us at 16 heads of 128 channels and 8000
// packed rows, 295 instead of 286 for 16 tokens over 32768 keys, so not in every call.
PF_DEVICE float cap_u(float x) { return __builtin_amdgcn_rcpf(-1.f - __builtin_amdgcn_exp2f(x)); }
PF_DEVICE float tanh_f(float x) {
    const float y = x * x;
    const float near = x * __builtin_fmaf(y, __builtin_fmaf(y, __builtin_fmaf(y, __builtin_fmaf(y, 62.f / 2835.f, -17.f / 315.f), 2.f / 15.f), -1.f / 3.f), 1.f);
    const float e = __builtin_amdgcn_exp2f(-2.f * LOG2E * fabsf(x)), d = 1.f + e;
    float r = __builtin_amdgcn_rcpf(d);
    r = __builtin_fmaf(__builtin_fmaf(-d, r, 1.f), r, r);
    return fabsf(x) < 0.3f ? near : copysignf((1.f - e) * r, x);
}
// x of one product and the slope of the cap (a quarter of it with cap_u)
template <int MODE>
PF_DEVICE float capped(const RArgs& p, float z, float& slope) {
    if constexpr ((MODE & 1) == 0) {
        return z;
    } else if constexpr ((MODE & 4) != 0) {
        const float y = tanh_f(z * p.zc);
        slope = __builtin_fmaf(-y, y, 1.f);
        return y;
    } else {
        const float u = cap_u(z * p.zc);
        slope = __builtin_fmaf(-u, u, -u);
        return u;
    }
}
PF_DEVICE float bias2(float b) { return b <= HIDDEN ? -__builtin_inff() : b * LOG2E; }
// a hidden distance hides a score that is not finite, too
PF_DEVICE float with_bias(float t, float b) { return b == -__builtin_inff() ? b : t + b; }

// base-2 score of one pair from global memory (exact_* and nothing else)
PF_DEVICE float score2(const RArgs& p, float z, int h, int dist, float& slope) {
    slope = 1.f;
    const float x = p.cap2 == 0.f ? z : p.series ? capped<5>(p, z, slope) : capped<1>(p, z, slope);
    const float t = __builtin_fmaf(x, p.zs, p.shift);
    return p.bias ? with_bias(t, bias2(p.bias[(long long)h * (2 * p.R + 1) + min(max(dist, -p.R), p.R) + p.R])) : t;
}
// positions in front of or behind every key by more than any radius count alike: differences stay inside 32 bits
PF_DEVICE int row_pos(const RArgs& p, int b, int row) {
    return p.q_pos ? min(max(p.q_pos[b * p.pos_bs + row], 4096 - (1 << 30)), (1 << 30) + 4096) : row + p.Lk - p.Lq;
}

template <int D>
PF_DEVICE float dot_row(const bf16_t* a, const bf16_t* b) {
    float s = 0.f;
#pragma unroll 2
    for (int c = 0; c < D; c += 8) {
        float x[8], y[8];
        unpack8(*(const u32x4_t*)(a + c), x);
        unpack8(*(const u32x4_t*)(b + c), y);
#pragma unroll
        for (int e = 0; e < 8; ++e) s = __builtin_fmaf(x[e], y[e], s);
    }
    return s;
}

// acc (channels lane D / 64 ..) += w(lane t) row(j0 + t) over the lanes with `use`
template <int D>
PF_DEVICE void add_rows(const bf16_t* base, long long ld, int j0, unsigned long long use, float w, float* acc) {
    const int lane = threadIdx.x & 63;
    while (use) {
        const int t = __builtin_ctzll(use);
        use &= use - 1;
        const float wt = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), t));
        const bf16_t* r = base + (long long)(j0 + t) * ld + lane * (D / 64);
#pragma unroll
        for (int c = 0; c < D / 64; ++c) acc[c] = __builtin_fmaf(wt, (float)r[c], acc[c]);
    }
}
// a NaN stays one: nothing that is added later changes the row any more
template <int D>
PF_DEVICE bool all_nan(const float* acc) {
    bool nan = acc[0] != acc[0];
    if (D == 128) nan = nan && acc[1] != acc[1];
    return __builtin_amdgcn_ballot_w64(!nan) == 0;
}
template <int D>
PF_DEVICE void store_row(bf16_t* row, const float* acc) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int c = 0; c < D / 64; ++c) row[lane * (D / 64) + c] = (bf16_t)acc[c];
}

// one whole wave: O of row i of head h from its visible keys alone (m: base-2 reference, l: sum of 2^(t - m - e))
template <int D>
PF_DEVICE void exact_o(const RArgs& p, int b, int h, int i, float m, float l, float e = 0.f) {
    const int lane = threadIdx.x & 63, hk = h / p.G;
    const Vis v = load_vis(p, b, i);
    const int pos = row_pos(p, b, i);
    const bf16_t* q = p.q.p + b * p.q.bs + i * p.q.ld + h * p.q.hs;
    const bf16_t* K = p.k.p + b * p.k.bs + hk * p.k.hs;
    const bf16_t* V = p.v.p + b * p.v.bs + hk * p.v.hs;
    float acc[2] = {0.f, 0.f};
    for (int j0 = 0; j0 < p.Lk; j0 += 64) {
        const int j = j0 + lane;
        bool use = j < p.Lk && sees(v, j);
        if (__builtin_amdgcn_ballot_w64(use) == 0) continue;
        float w = 0.f, slope;
        if (use) {
            const float t = score2(p, dot_row<D>(q, K + j * p.k.ld), h, j - pos, slope);
            use = t != -__builtin_inff();
            w = __builtin_amdgcn_exp2f((t - m) - e) / l;
        }
        add_rows<D>(V, p.v.ld, j0, __builtin_amdgcn_ballot_w64(use), w, acc);
        if (all_nan<D>(acc)) break;
    }
    store_row<D>(p.o.p + b * p.o.bs + i * p.o.ld + h * p.o.hs, acc);
}

// P and dZ of one visible pair, from global memory
template <int D>
PF_DEVICE bool exact_pair(const RArgs& p, int b, int h, int hk, int i, int j, float& P, float& dz) {
    float slope;
    const float z = dot_row<D>(p.q.p + b * p.q.bs + i * p.q.ld + h * p.q.hs, p.k.p + b * p.k.bs + j * p.k.ld + hk * p.k.hs);
    const float t = score2(p, z, h, j - row_pos(p, b, i), slope);
    if (t == -__builtin_inff()) return false;
    const float* st = p.stat + (((long long)b * p.H + h) * p.nq64 + (i >> 6)) * 256 + (i & 63);
    P = __builtin_amdgcn_exp2f(t - p.shift - st[0]);
    const float dp = dot_row<D>(p.dO.p + b * p.dO.bs + i * p.dO.ld + h * p.dO.hs, p.v.p + b * p.v.bs + j * p.v.ld + hk * p.v.hs);
    dz = P * (dp + st[64]) * slope;
    return true;
}
template <int D>
PF_DEVICE void exact_dq(const RArgs& p, int b, int h, int i) {
    const int lane = threadIdx.x & 63, hk = h / p.G;
    const Vis v = load_vis(p, b, i);
    float acc[2] = {0.f, 0.f};
    for (int j0 = 0; j0 < p.Lk; j0 += 64) {
        const int j = j0 + lane;
        bool use = j < p.Lk && sees(v, j);
        if (__builtin_amdgcn_ballot_w64(use) == 0) continue;
        float P = 0.f, dz = 0.f;
        if (use) use = exact_pair<D>(p, b, h, hk, i, j, P, dz);
        add_rows<D>(p.k.p + b * p.k.bs + hk * p.k.hs, p.k.ld, j0, __builtin_amdgcn_ballot_w64(use), dz * p.dscale, acc);
        if (all_nan<D>(acc)) break;
    }
    store_row<D>(p.dq.p + b * p.dq.bs + i * p.dq.ld + h * p.dq.hs, acc);
}
template <int D>
PF_DEVICE void exact_dkv(const RArgs& p, int b, int hk, int j) {
    const int lane = threadIdx.x & 63;
    float ak[2] = {0.f, 0.f}, av[2] = {0.f, 0.f};
    bool nan_k = false, nan_v = false;
    for (int h = hk * p.G; h < (hk + 1) * p.G && !(nan_k && nan_v); ++h)
        for (int i0 = 0; i0 < p.Lq && !(nan_k && nan_v); i0 += 64) {
            const int i = i0 + lane;
            bool use = i < p.Lq && sees(load_vis(p, b, i), j);
            if (__builtin_amdgcn_ballot_w64(use) == 0) continue;
            float P = 0.f, dz = 0.f;
            if (use) use = exact_pair<D>(p, b, h, hk, i, j, P, dz);
            const unsigned long long m = __builtin_amdgcn_ballot_w64(use);
            if (!nan_k) add_rows<D>(p.q.p + b * p.q.bs + h * p.q.hs, p.q.ld, i0, m, dz * p.dscale, ak);
            if (!nan_v) add_rows<D>(p.dO.p + b * p.dO.bs + h * p.dO.hs, p.dO.ld, i0, m, P, av);
            nan_k = nan_k || all_nan<D>(ak);
            nan_v = nan_v || all_nan<D>(av);
        }
    store_row<D>(p.dk.p + b * p.dk.bs + j * p.dk.ld + hk * p.dk.hs, ak);
    store_row<D>(p.dv.p + b * p.dv.bs + j * p.dv.ld + hk * p.dv.hs, av);
}

// One whole wave: whether the sums of keys w0 .. w0 + 31 may hold what does not belong there -- a row that shares a tile with them does
// not see one of them, a bias hides some distance, or the last row, which a short tile repeats with weights of 0, is not finite.
// Where none of this is so, a result that is not finite is right as it is: one infinite entry of dout costs nothing (16 heads of 64
// over 4 key heads, 2048 rows, nothing hidden: 106 us with and 112 without it, 2320 when all keys were computed again).
template <int D, bool BIAS>
PF_DEVICE bool strangers(const RArgs& p, int b, int hk, int w0) {
    int lane = threadIdx.x & 63;
    // nothing of this is worked out early and kept in registers through the caller's loop (4 x 3000 causal rows of 32 heads of 128 with a
    // bias 1611 instead of 1677 us; without a bias there is no such gain)
    if (BIAS) asm volatile("" : "+v"(lane));
    const int w1 = min(w0 + 32, p.Lk), rest = p.Lq & 63;
    const int* const tiles = p.tiles + (long long)b * p.nq64 * 8;
    bool bad = false;
    if (BIAS && p.bias)
        for (long long i = (long long)hk * p.G * (2 * p.R + 1) + lane; i < (long long)(hk + 1) * p.G * (2 * p.R + 1); i += 64) bad = bad || p.bias[i] <= HIDDEN;
    for (int n = lane; n < p.nq64 - (rest ? 1 : 0); n += 64) {
        const int* x = tiles + n * 8LL;
        const bool some = (x[0] < w1 && x[1] > w0) || (x[2] < w1 && x[3] > w0);
        bad = bad || (some && !((x[4] <= w0 && x[5] >= w1) || (x[6] <= w0 && x[7] >= w1)));
    }
    if (rest) {                                    // row by row: the rows behind the last one see nothing
        const int* x = tiles + (p.nq64 - 1) * 8LL;
        const int* v = p.vis + ((long long)b * p.nq64 + p.nq64 - 1) * 256 + lane;
        const int alo = v[0], ahi = alo + v[64], blo = v[128], bhi = blo + v[192];
        const bool all = (alo <= w0 && ahi >= w1) || (blo <= w0 && bhi >= w1);
        if ((x[0] < w1 && x[1] > w0) || (x[2] < w1 && x[3] > w0)) {
            bad = bad || (lane < rest && !all);
            const long long last = p.Lq - 1;
            for (int h = hk * p.G; h < (hk + 1) * p.G; ++h)
#pragma unroll
                for (int c = 0; c < D / 64; ++c) {
                    const int at = lane * (D / 64) + c;
                    bad = bad || !(fabsf((float)p.q.p[b * p.q.bs + last * p.q.ld + h * p.q.hs + at]) < __builtin_inff()) ||
                          !(fabsf((float)p.dO.p[b * p.dO.bs + last * p.dO.ld + h * p.dO.hs + at]) < __builtin_inff());
                }
        }
    }
    return __builtin_amdgcn_ballot_w64(bad) != 0;
}

// lane l holds column l % 32 of a [D][32] result, channels reg_row(r) + 4 (l / 32) + 32 c: 8-byte stores into its row
template <int D>
PF_DEVICE void store_cols(bf16_t* row, const f32x16_t* o, float f) {
    const int hi = (threadIdx.x >> 5) & 1;
#pragma unroll
    for (int c = 0; c < D / 32; ++c)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
            u32x2_t w;
            w[0] = pack2(o[c][4 * q4] * f, o[c][4 * q4 + 1] * f);
            w[1] = pack2(o[c][4 * q4 + 2] * f, o[c][4 * q4 + 3] * f);
            *(u32x2_t*)(row + c * 32 + q4 * 8 + 4 * hi) = w;
        }
}
template <int N>
PF_DEVICE bool any_nonfinite(const f32x16_t* o) {
    float t = 0.f;                                     // 0 x finite = 0; 0 x (inf | NaN) = NaN
#pragma unroll
    for (int c = 0; c < N; ++c)
#pragma unroll
        for (int r = 0; r < 16; ++r) t = __builtin_fmaf(o[c][r], 0.f, t);
    return t != t;
}

// The bias table of head h in LDS, base 2 (or times `unit`), continued by PAD entries of its end values on both sides: a 32 x 64
// block of consecutive rows whose distances are not all behind an end stays inside it, so its entries lie at fixed offsets from one
// address per lane (a subtraction, a clamp and an address per score otherwise).  Returned: the entry of distance 0.
constexpr int PAD = 96;
constexpr int table_floats(int R) { return 2 * R + 1 + 2 * PAD; }
PF_DEVICE const float* load_table(const RArgs& p, int h, float* tab, float unit = LOG2E) {
    for (int i = threadIdx.x; i < table_floats(p.R); i += 256) {
        const float b = p.bias[(long long)h * (2 * p.R + 1) + min(max(i - PAD, 0), 2 * p.R)];
        tab[i] = b <= HIDDEN ? -__builtin_inff() : b * unit;
    }
    return tab + PAD + p.R;
}
// how a block with distances lo .. hi (wave-uniform) reads it
enum Reach { NEAR, FAR, MIXED };
PF_DEVICE Reach reach(int R, int lo, int hi) {
    return (hi <= -R || lo >= R) ? FAR : (lo >= -R - PAD && hi <= R + PAD) ? NEAR : MIXED;
}

// products -> x (see RArgs)
template <int MODE>
PF_DEVICE void cap_only(const RArgs& p, f32x16_t& s) {
    if constexpr ((MODE & 1) != 0) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            float slope;
            s[r] = capped<MODE>(p, s[r], slope);
        }
    }
}
// x -> x zs + bias (a NaN stays one even where the bias hides it: what comes out of it is not finite, and is done again with care); d0 = distance of this lane's register 0 (SIGN 1: registers are keys, -1: rows), lo, hi = of the block
template <int SIGN>
PF_DEVICE void add_bias(const RArgs& p, f32x16_t& s, float zs, const float* tab, int d0, int lo, int hi) {
    const Reach how = reach(p.R, lo, hi);
    if (how == NEAR) {
        const float* at = tab + d0;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = __builtin_fmaf(s[r], zs, at[SIGN * reg_row(r)]);
    } else if (how == FAR) {
        const float c = tab[hi <= -p.R ? -p.R : p.R];
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = __builtin_fmaf(s[r], zs, c);
    } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = __builtin_fmaf(s[r], zs, tab[min(max(d0 + SIGN * reg_row(r), -p.R), p.R)]);
    }
}

// Which (head, tile) a workgroup takes.  Every XCD has a contiguous run of heads (their K and V stay in its L2), walks the first
// half of each head's tiles -- the ones that causal and frame-wise masks make long -- for all of its heads and then the second
// halves: the launch ends on short workgroups.  Tile numbers here count from the heavy end.  (Against head after
// head, at the time: 1308 instead of 1415 us for 30 heads of the 15488-row video sequence, today 1222 .. 1330 by the card; gradients at
// 7808 rows 1333 instead of 1500, today 1260 .. 1325.)
//
// `resident` > 0: the first workgroups of an XCD go to its 32 compute units in turn, so those that start together on one unit are 32
// apart; every other 32 come in reverse, which pairs long ones with short ones.
struct Place { int head, rank; };
PF_DEVICE Place heavy_first(int block, int n, int nwg, int resident = 0) {
    const int q = nwg >> 3, r = nwg & 7, xcd = block & 7;
    int i = block >> 3;
    if (((i >> 5) & 1) && (i >> 5) < resident && (i | 31) < q) i ^= 31;
    const int c0 = xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q, c1 = c0 + q + (xcd < r ? 1 : 0);
    const int nh = (n + 1) / 2, nl = n - nh;
    auto heavy_below = [&](int c) { const int w = c / n; return w * nh + min(c - w * n, nh); };
    const int h0 = heavy_below(c0), hn = heavy_below(c1) - h0;
    const bool heavy = i < hn;
    const int k = heavy ? h0 + i : (c0 - h0) + (i - hn), m = heavy ? nh : nl, w = k / m;
    return {w, k - w * m + (heavy ? 0 : nh)};
}

// whether the row tiles of a forward launch of nwg workgroups, `resident` to a compute unit, start in falling order of their keys
constexpr int SORTED_TILES = 256;
__host__ __device__ constexpr bool sorted_launch(int nwg, int resident) { return nwg > 256 * resident && nwg <= 768 * resident; }

// The row tile (of ROWS rows) that comes at place `rank` when a head's tiles start in falling order of their keys: `sort` and at most
// 256 tiles.  One thread per tile takes the larger count of its first and last row and counts the tiles before it, the same in every
// workgroup of the batch entry.  Otherwise the tiles come from the sequence's end on.  `mem`: 1028 bytes of LDS, free again behind
// the caller's next barrier.  Sorted where a launch is one to three rounds of workgroups: with fewer all start at once, with more the
// unevenness fades and the sorting costs 1 % (16 heads of 128, 8000 rows packed of 5 documents: 127 instead of 137 us, of 12: 63
// instead of 79 us).
template <int ROWS>
PF_DEVICE int ranked_tile(const RArgs& p, int b, int rank, bool sort, int* mem) {
    if (!sort || !p.a_lo || p.nqt > SORTED_TILES) return p.nqt - 1 - rank;
    const int t = threadIdx.x;
    int mine = -1;
    if (t < p.nqt) {
        const Vis x = load_vis(p, b, t * ROWS), y = load_vis(p, b, min(t * ROWS + ROWS, p.Lq) - 1);
        mine = min(max(x.na + x.nb, y.na + y.nb) >> 2, (1 << 23) - 1) << 8 | t;
    }
    mem[t] = mine;
    __syncthreads();
    int before = 0;
    for (int i = 0; i < (p.nqt + 3) / 4; ++i) {
        const u32x4_t k = *(const u32x4_t*)(mem + 4 * i);
#pragma unroll
        for (int e = 0; e < 4; ++e) before += (int)k[e] > mine;
    }
    if (t < p.nqt && before == rank) mem[256] = t;
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(mem[256]);
}

// ---------------------------------------------------------------------------------------------- forward, many rows
// One workgroup of 4 waves = 128 rows of one head, or with KS = 2 64 rows whose two halves of every key tile go to different waves
// (their results meet in LDS at the end): the shorter chain for problems with few row tiles.  Key tiles of KB, two in flight.
// MODE bits: 1 cap, 2 bias (scores are formed before the maximum; without one the exponent's multiply-add scales them), 4 SERIES.
//
// Bound: vector issue (per 32 rows x 64 keys 512 cycles of matrix pipe at D = 64 against 32 multiply-adds, 32 exponentials at
// 8 cycles, 32 adds, 16 conversions).  So the first pass keeps no running maximum: a row's reference is the maximum of the first
// tile in which it sees a key; a weight may then grow to 2^127 before anything overflows and its rounding to bf16 is relative,
// so the result is the same.  If a sum or a result of the workgroup came out non-finite, it runs again with the running maximum
// (CAREFUL), and rows that are still non-finite and had hidden keys are recomputed from their visible keys (exact_o).
template <int D, int MODE, int KS>
__global__ __launch_bounds__(256, (FWD_WAVES<D, KS>)) void range_fwd_kernel(const RArgs p) {
    constexpr bool BIAS = MODE & 2;
    constexpr int KB = FWD_KB<D, KS>, NI = KB / 32 / KS, TILE = KB * 2 * D, BUF = 2 * TILE, RW = 4 / KS;
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    int* const red = (int*)(smem + 2 * BUF);
    int* const redo_flag = red + 16;
    Cover* const cover = (Cover*)(red + 20);
    float* const meet = (float*)(smem + 2 * BUF + 96);           // KS = 2: [row wave][3][64] reference, sum, its exponent and `whole`
    float* const tab_ = meet + (KS == 2 ? RW * 192 : 0);
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), rw = wid % RW, kw = wid / RW;
    constexpr int RESIDENT = FWD_WAVES<D, KS>;       // workgroups of a compute unit
    const int nwg = p.nqt * p.H * p.B;
    const Place at = heavy_first(blockIdx.x, p.nqt, nwg, RESIDENT);
    const int bh = at.head, b = bh / p.H, h = bh - b * p.H, hk = h / p.G;
    const int qt = ranked_tile<32 * RW>(p, b, at.rank, sorted_launch(nwg, RESIDENT), (int*)smem);
    const int hi = lane >> 5, row0 = (qt * RW + rw) * 32, row = row0 + (lane & 31);
    const Vis vis = load_vis(p, b, row);
    const int pos = BIAS ? row_pos(p, b, min(row, p.Lq - 1)) : 0;
    const int pmin = BIAS ? wave_min(pos) : 0, pmax = BIAS ? wave_max(pos) : 0;
    const Bounds wb = wave_bounds(vis);
    if (threadIdx.x == 0) *redo_flag = 0;
    const TileList tl = workgroup_tiles<KB>(wb, red, cover, wid, lane);
    const bf16_t* const K = p.k.p + b * p.k.bs + hk * p.k.hs;
    const bf16_t* const V = p.v.p + b * p.v.bs + hk * p.v.hs;
    const Stager<D, KB, 4> sk_(p.k.ld, wid, lane), sv_(p.v.ld, wid, lane);
    const unsigned roff = row_offset<D>(lane), t0 = tr_offset<D>(lane, 0), t8 = tr_offset<D>(lane, 8);
    f32x16_t o[D / 32];
    float m, l;
    bool whole;                                    // wave-uniform: no row of the wave had a hidden key in any tile (a bias may hide some)
    auto issue = [&](int n, bool begin = false) {
        const int j0 = tl.at(n) * KB;
        char* buf = smem + (n & 1) * BUF;
        if (begin ? tl.keys.whole(j0, j0 + KB) : tl.inner(n)) {
            sk_.whole(K, p.k.ld, j0, buf, wid);
            sv_.whole(V, p.v.ld, j0, buf + TILE, wid);
        } else {
            const Cover c = begin ? tl.keys : scalar(*cover);
            sk_.part(K, p.k.ld, j0, c, buf, wid, lane);
            sv_.part(V, p.v.ld, j0, c, buf + TILE, wid, lane);
        }
    };
    if (tl.n > 0) issue(0, true);                  // the first tile is on its way before the rows are read
    const float* const tab = BIAS ? load_table(p, h, tab_) : nullptr;
    bf16x8_t qf[D / 16];
    {
        const bf16_t* q = p.q.p + b * p.q.bs + (long long)min(row, p.Lq - 1) * p.q.ld + h * p.q.hs + hi * 8;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) qf[ks] = *(const bf16x8_t*)(q + ks * 16);
    }
    auto pass = [&](auto careful) {
        constexpr bool CAREFUL = decltype(careful)::value;
        const float zs = BIAS ? 1.f : p.zs;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) o[c] = zero16();
        m = -__builtin_inff();
        l = 0.f;
        whole = !BIAS;
        unsigned long long fresh = __builtin_amdgcn_ballot_w64(vis.na + vis.nb > 0);     // rows without a reference yet
        if (CAREFUL) {
            drain_barrier();                       // nobody reads the first pass's tiles any more
            if (tl.n > 0) issue(0);
        }
        for (int n = 0; n < tl.n; ++n) {
            drain_barrier();
            if (n + 1 < tl.n) issue(n + 1);
            const int j0 = tl.at(n) * KB + kw * 32 * NI;             // this wave's keys of the tile
            const char* sk = smem + (n & 1) * BUF + kw * NI * 64 * D;
            const char* sv = sk + TILE;
            const bool full = wb.full(j0, j0 + 32 * NI);
            if (!full) {
                whole = false;
                if (!wb.any(j0, j0 + 32 * NI)) continue;
            }
            f32x16_t s[NI];
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                s[i] = zero16();
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks) s[i] = mfma(row_frag<D>(sk, roff, i, ks), qf[ks], s[i]);
            }
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                cap_only<MODE>(p, s[i]);
                if (BIAS) add_bias<1>(p, s[i], p.zs, tab, j0 + 32 * i + 4 * hi - pos, j0 + 32 * i - pmax, j0 + 32 * i + 31 - pmin);
            }
            if (CAREFUL && BIAS) {                 // NaN + -inf: hidden
#pragma unroll
                for (int i = 0; i < NI; ++i)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const float b = tab[min(max(j0 + 32 * i + 4 * hi + reg_row(r) - pos, -p.R), p.R)];
                        s[i][r] = b == -__builtin_inff() ? b : s[i][r];
                    }
            }
            if (!full) {
#pragma unroll
                for (int i = 0; i < NI; ++i)
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[i][r] = sees(vis, j0 + 32 * i + 4 * hi + reg_row(r)) ? s[i][r] : -__builtin_inff();
            }
            if (CAREFUL || fresh != 0) {           // wave-uniform
                float mt = s[0][0];
#pragma unroll
                for (int i = 0; i < NI; ++i)
#pragma unroll
                    for (int r = 0; r < 16; ++r) mt = fmaxf(mt, s[i][r]);
                mt = fmaxf(mt, other_half(mt)) * zs;
                if (CAREFUL) {
                    if (__builtin_amdgcn_ballot_w64(mt > m + DEFER) != 0) {
                        const float mn = fmaxf(m, mt);
                        const float alpha = mn == m ? 1.f : __builtin_amdgcn_exp2f(m - mn);
                        m = mn;
                        l *= alpha;
#pragma unroll
                        for (int c = 0; c < D / 32; ++c)
#pragma unroll
                            for (int r = 0; r < 16; ++r) o[c][r] *= alpha;
                    }
                } else {
                    m = m == -__builtin_inff() ? mt : m;
                    fresh &= __builtin_amdgcn_ballot_w64(m == -__builtin_inff());
                }
            }
            const float ms = m == -__builtin_inff() ? 0.f : m;
            float ps[2] = {0.f, 0.f};
#pragma unroll
            for (int i = 0; i < NI; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i][r], zs, -ms));
                    s[i][r] = e;
                    ps[r & 1] += e;
                }
            l += ps[0] + ps[1];
            // the second product goes first: its operands are ready, the other waves' exponentials fill in behind it (15488 rows, 30
            // heads of 64: 1252 instead of 1283 us; at D = 128 no gain)
            if (D == 64) __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int g = 0; g < 2 * NI; ++g) {
                const bf16x8_t pf = half_of(s[g >> 1], g & 1);
#pragma unroll
                for (int c = 0; c < D / 32; ++c) o[c] = mfma(tr_frag<D>(sv, t0, t8, c, g), pf, o[c]);
            }
            if (D == 64) __builtin_amdgcn_s_setprio(0);
        }
        l += other_half(l);
    };
    pass(std::false_type{});
    if (__builtin_amdgcn_ballot_w64(!(l < __builtin_inff()) || any_nonfinite<D / 32>(o)) != 0 && lane == 0) *redo_flag = 1;
    __syncthreads();
    if (*redo_flag != 0) pass(std::true_type{});   // workgroup-uniform: the passes share tiles and barriers
    float le = 0.f;                                // the row's sum is l 2^(m + le)
    if constexpr (KS == 2) {
        // The halves' references are the maxima of their first tiles, not of their rows: a half's sum may lie 2^127 above its own.  So
        // both are brought to sums in [1/2, 1) first (exact), and the powers of two that were taken out go into the halves' distance:
        // what is then below 2^-126 of the other half counts for nothing, and no sum can overflow.
        float* const acc = (float*)smem + rw * (D / 32) * 16 * 64;   // the tiles' memory: [row wave][register][lane]
        const int e1 = __builtin_amdgcn_frexp_expf(l);               // 0 where the half saw no key, or l is not finite
        l = __builtin_amdgcn_ldexpf(l, -e1);
#pragma unroll
        for (int c = 0; c < D / 32; ++c)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[c][r] = __builtin_amdgcn_ldexpf(o[c][r], -e1);
        __syncthreads();
        if (kw == 1) {
#pragma unroll
            for (int c = 0; c < D / 32; ++c)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[(c * 16 + r) * 64 + lane] = o[c][r];
            meet[rw * 192 + lane] = m;
            meet[rw * 192 + 64 + lane] = l;
            meet[rw * 192 + 128 + lane] = (float)(2 * e1 + (whole ? 1 : 0));
        }
        __syncthreads();
        if (kw == 1) return;
        const float m2 = meet[rw * 192 + lane], l2 = meet[rw * 192 + 64 + lane];
        const int w2 = (int)meet[rw * 192 + 128 + lane], e2 = w2 >> 1;
        whole = whole && (__builtin_amdgcn_readfirstlane(w2) & 1) != 0;
        const bool one = m2 == -__builtin_inff(), two = m == -__builtin_inff();       // only one half saw a key
        const float x = (m - m2) + (float)(e1 - e2);                 // log2 of the halves' ratio, but for a factor of two
        const bool first = one || x >= 0.f;                          // the half whose scale the row keeps
        const float f = two ? 0.f : first ? 1.f : __builtin_amdgcn_exp2f(x), f2 = one ? 0.f : first ? __builtin_amdgcn_exp2f(-x) : 1.f;
        // a half without a key holds zeros (or 0 x inf of hidden keys, which exact_o sees); a NaN sum has its reference at -inf
        l = (two && l == 0.f ? 0.f : two ? l : f * l) + (one ? l2 : f2 * l2);
#pragma unroll
        for (int c = 0; c < D / 32; ++c)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[c][r] = f * o[c][r] + f2 * acc[(c * 16 + r) * 64 + lane];
        m = first ? m : m2;
        le = (float)(first ? e1 : e2);
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const bool bad = any_nonfinite<D / 32>(o) && !whole && l == l && row < p.Lq;
    unsigned long long redo = __builtin_amdgcn_ballot_w64(bad);
    redo = (redo | (redo >> 32)) & 0xffffffffull;
    const bool mine = (redo >> (lane & 31)) & 1;
    if (row < p.Lq) {
        if (!mine) store_cols<D>(p.o.p + b * p.o.bs + row * p.o.ld + h * p.o.hs, o, inv);
        if (p.lse && hi == 0) p.lse[((long long)b * p.H + h) * p.Lq + row] = l == 0.f ? -__builtin_inff() : (m + p.shift + (le + __builtin_amdgcn_logf(l))) * LN2;
    }
    while (redo) {
        const int i = __builtin_ctzll(redo);
        redo &= redo - 1;
        exact_o<D>(p, b, h, row0 + i, __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(m), i)) + p.shift,
                   __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(l), i)), __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(le), i)));
    }
}

// ---------------------------------------------------------------------------------------------- forward, few rows
// One workgroup = 32 (row, head) pairs that share a key head, one part of the keys; its 4 waves take every fourth 32-key tile of
// the part and meet in LDS at the end.  Tiles are private to a wave: no barrier in the loop, the next tile is in flight while the
// current one is used.  nsplit > 1: parts go to the workspace, range_join_kernel adds them.
template <int D, int MODE>
__global__ __launch_bounds__(256, 1) void range_split_kernel(const RArgs p) {
    constexpr bool CAP = MODE & 1, BIAS = MODE & 2;
    constexpr int TILE = 32 * 2 * D, BUF = 2 * TILE, WAVE = 2 * BUF, NP = 2 * 32 / (512 / D);
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int unit = blockIdx.x / p.nsplit, part = blockIdx.x - unit * p.nsplit;
    const int bk = unit / p.nrb, rb = unit - bk * p.nrb;
    const int b = bk / p.Hk, hk = bk - b * p.Hk;
    const int hi = lane >> 5;
    const int rho = rb * 32 + (lane & 31);                          // row rho / G of head hk G + rho % G
    const bool valid = rho < p.Lq * p.G;
    const int row = valid ? rho / p.G : p.Lq - 1, h = hk * p.G + (valid ? rho % p.G : 0);
    Vis vis = load_vis(p, b, row);
    if (!valid) vis.na = vis.nb = 0;
    const int pos = BIAS ? row_pos(p, b, row) : 0;
    const float* const bias = BIAS ? p.bias + (long long)h * (2 * p.R + 1) + p.R : nullptr;
    const float far_below = BIAS ? bias2(bias[-p.R]) : 0.f, far_above = BIAS ? bias2(bias[p.R]) : 0.f;
    const int pmin = BIAS ? wave_min(pos) : 0, pmax = BIAS ? wave_max(pos) : 0;
    const int amin = wave_min(vis.na ? vis.alo : 0x7fffffff), amax = wave_max(vis.na ? vis.alo + vis.na : 0);
    const int bmin = wave_min(vis.nb ? vis.blo : 0x7fffffff), bmax = wave_max(vis.nb ? vis.blo + vis.nb : 0);
    const TileList tl = tile_list<32>(amin, amax, bmin, bmax);
    Cover* const cover = (Cover*)(smem + 4 * WAVE) + wid;
    *cover = tl.keys;
    const int n0 = (int)((long long)tl.n * part / p.nsplit), n1 = (int)((long long)tl.n * (part + 1) / p.nsplit);
    const bf16_t* const K = p.k.p + b * p.k.bs + hk * p.k.hs;
    const bf16_t* const V = p.v.p + b * p.v.bs + hk * p.v.hs;
    bf16x8_t qf[D / 16];
    {
        const bf16_t* q = p.q.p + b * p.q.bs + row * p.q.ld + h * p.q.hs + hi * 8;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) qf[ks] = *(const bf16x8_t*)(q + ks * 16);
    }
    const unsigned roff = row_offset<D>(lane), t0 = tr_offset<D>(lane, 0), t8 = tr_offset<D>(lane, 8);
    f32x16_t o[D / 32];
#pragma unroll
    for (int c = 0; c < D / 32; ++c) o[c] = zero16();
    float m = -__builtin_inff(), l = 0.f;
    char* const mem = smem + wid * WAVE;
    drain();                                                        // the counted waits below see tile pieces only
    const Stager<D, 32, 1> sk_(p.k.ld, 0, lane), sv_(p.v.ld, 0, lane);
    auto issue = [&](int n, int buf, bool begin = false) {
        const int j0 = tl.at(n) * 32;
        char* to = mem + buf * BUF;
        if (begin ? tl.keys.whole(j0, j0 + 32) : tl.inner(n)) {
            sk_.whole(K, p.k.ld, j0, to, 0);
            sv_.whole(V, p.v.ld, j0, to + TILE, 0);
        } else {
            const Cover c = begin ? tl.keys : scalar(*cover);
            sk_.part(K, p.k.ld, j0, c, to, 0, lane);
            sv_.part(V, p.v.ld, j0, c, to + TILE, 0, lane);
        }
    };
    if (n0 + wid < n1) issue(n0 + wid, 0, true);
    int buf = 0;
    for (int n = n0 + wid; n < n1; n += 4, buf ^= 1) {
        if (n + 4 < n1) {
            issue(n + 4, buf ^ 1);
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NP) : "memory");
        } else {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        const int j0 = tl.at(n) * 32;
        const char* sk = mem + buf * BUF;
        const char* sv = sk + TILE;
        f32x16_t s = zero16();
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) s = mfma(row_frag<D>(sk, roff, 0, ks), qf[ks], s);
        const int k0 = j0 + 4 * hi;
        // the gather from global memory waits for the tile in flight too: only where the distances are inside the table
        const bool far = BIAS && reach(p.R, j0 - pmax, j0 + 31 - pmin) == FAR;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            float slope;
            float t = capped<MODE>(p, s[r], slope) * p.zs;
            if (BIAS) t = with_bias(t, far ? (j0 + 31 - pmin <= -p.R ? far_below : far_above) : bias2(bias[min(max(k0 + reg_row(r) - pos, -p.R), p.R)]));
            s[r] = sees(vis, k0 + reg_row(r)) ? t : -__builtin_inff();
        }
        float mt = s[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) mt = fmaxf(mt, s[r]);
        mt = fmaxf(mt, other_half(mt));
        const float mn = fmaxf(m, mt);
        const float alpha = mn == m ? 1.f : __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        const float ms = m == -__builtin_inff() ? 0.f : m;
        float ps = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s[r] = __builtin_amdgcn_exp2f(s[r] - ms);
            ps += s[r];
        }
        l = l * alpha + ps;
#pragma unroll
        for (int c = 0; c < D / 32; ++c)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[c][r] *= alpha;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            const bf16x8_t pf = half_of(s, g);
#pragma unroll
            for (int c = 0; c < D / 32; ++c) o[c] = mfma(tr_frag<D>(sv, t0, t8, c, g), pf, o[c]);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");           // the tile is read: its buffer may be refilled
    }
    l += other_half(l);
    // ---- the four waves meet: [wave][32][D + 4] fp32 (O, m, l), a row per lane pair
    constexpr int PITCH = D + 4;
    __syncthreads();
    float* const acc = (float*)smem;
    {
        float* r = acc + (wid * 32 + (lane & 31)) * PITCH;
#pragma unroll
        for (int c = 0; c < D / 32; ++c)
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4) {
                f32x4_t w;
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = o[c][4 * q4 + e];
                *(f32x4_t*)(r + 32 * c + 8 * q4 + 4 * hi) = w;
            }
        if (hi == 0) { r[D] = m; r[D + 1] = l; }
    }
    __syncthreads();
    const int rows = min(32, p.Lq * p.G - rb * 32);
    for (int r = wid; r < rows; r += 4) {                           // one row per wave: lanes over channels
        float mm = -__builtin_inff(), f[4], ll = 0.f, v[2] = {0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; ++w) mm = fmaxf(mm, acc[(w * 32 + r) * PITCH + D]);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float* a = acc + (w * 32 + r) * PITCH;
            f[w] = a[D] == mm ? (mm == -__builtin_inff() ? 0.f : 1.f) : __builtin_amdgcn_exp2f(a[D] - mm);
            ll += f[w] == 0.f && a[D + 1] == 0.f ? 0.f : f[w] * a[D + 1];
#pragma unroll
            for (int c = 0; c < D / 64; ++c) v[c] += f[w] == 0.f && a[D + 1] == 0.f ? 0.f : f[w] * a[lane * (D / 64) + c];
        }
        const int pr = rb * 32 + r, i = pr / p.G, hh = hk * p.G + pr % p.G;
        if (p.nsplit > 1) {
            float* out = p.parts + (((long long)unit * p.nsplit + part) * 32 + r) * (D + 2);
#pragma unroll
            for (int c = 0; c < D / 64; ++c) out[lane * (D / 64) + c] = v[c];
            if (lane == 0) { out[D] = mm; out[D + 1] = ll; }
            continue;
        }
        bool bad = false;
#pragma unroll
        for (int c = 0; c < D / 64; ++c) bad = bad || !(fabsf(v[c]) < __builtin_inff());
        if (__builtin_amdgcn_ballot_w64(bad) != 0 && ll == ll) {
            exact_o<D>(p, b, hh, i, mm + p.shift, ll);
        } else {
            const float inv = ll == 0.f ? 0.f : 1.f / ll;
#pragma unroll
            for (int c = 0; c < D / 64; ++c) v[c] *= inv;
            store_row<D>(p.o.p + b * p.o.bs + i * p.o.ld + hh * p.o.hs, v);
        }
        if (p.lse && lane == 0) p.lse[((long long)b * p.H + hh) * p.Lq + i] = ll == 0.f ? -__builtin_inff() : (mm + p.shift + __builtin_amdgcn_logf(ll)) * LN2;
    }
}

// one wave per (row, head): the parts' maxima, then the weighted sums, in part order
template <int D>
__global__ __launch_bounds__(256) void range_join_kernel(const RArgs p) {
    const int lane = threadIdx.x & 63;
    const long long w = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int per = p.Lq * p.G;
    if (w >= (long long)p.B * p.Hk * per) return;
    const int bk = (int)(w / per), pr = (int)(w - (long long)bk * per);
    const int b = bk / p.Hk, hk = bk - b * p.Hk, i = pr / p.G, h = hk * p.G + pr % p.G;
    const float* base = p.parts + (((long long)bk * p.nrb + pr / 32) * p.nsplit * 32 + pr % 32) * (D + 2);
    const long long step = 32 * (D + 2);
    float m = -__builtin_inff();
    for (int s = lane; s < p.nsplit; s += 64) m = fmaxf(m, base[s * step + D]);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) m = fmaxf(m, __shfl_xor(m, o));
    float l = 0.f, v[2] = {0.f, 0.f};
    for (int s = 0; s < p.nsplit; ++s) {
        const float* a = base + s * step;
        const float ls = a[D + 1];
        if (ls == 0.f) continue;                                     // the part saw no key
        const float f = a[D] == m ? 1.f : __builtin_amdgcn_exp2f(a[D] - m);
        l += f * ls;
#pragma unroll
        for (int c = 0; c < D / 64; ++c) v[c] += f * a[lane * (D / 64) + c];
    }
    bool bad = false;
#pragma unroll
    for (int c = 0; c < D / 64; ++c) bad = bad || !(fabsf(v[c]) < __builtin_inff());
    if (__builtin_amdgcn_ballot_w64(bad) != 0 && l == l) {
        exact_o<D>(p, b, h, i, m + p.shift, l);
    } else {
        const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
        for (int c = 0; c < D / 64; ++c) v[c] *= inv;
        store_row<D>(p.o.p + b * p.o.bs + i * p.o.ld + h * p.o.hs, v);
    }
    if (p.lse && lane == 0) p.lse[((long long)b * p.H + h) * p.Lq + i] = l == 0.f ? -__builtin_inff() : (m + p.shift + __builtin_amdgcn_logf(l)) * LN2;
}

// ---------------------------------------------------------------------------------------------- backward
// What both gradient kernels need of a row, in 1-KiB pieces of 64 rows that the LDS-DMA can take as they are: log-sum-exp (base 2,
// less the scores' shift) and -delta = -sum_c dO O per head, the ranges per batch entry; and for each such tile the bounds of its
// ranges: 0..3 the smallest start and largest end of the a and b ranges that are not empty, 4..7 the largest start and smallest
// end over ALL its rows.
template <int D>
__global__ __launch_bounds__(256) void range_prep_kernel(const RArgs p) {
    const int qt = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
    const int r = threadIdx.x >> 2, row = qt * 64 + r, sub = threadIdx.x & 3;
    float s = 0.f;
    if (row < p.Lq) {
        const bf16_t* x = p.dO.p + b * p.dO.bs + row * p.dO.ld + h * p.dO.hs + sub * (D / 4);
        const bf16_t* y = p.o.p + b * p.o.bs + row * p.o.ld + h * p.o.hs + sub * (D / 4);
        s = dot_row<D / 4>(x, y);
    }
    s += __shfl_xor(s, 1);
    s += __shfl_xor(s, 2);
    float* st = p.stat + (((long long)b * p.H + h) * p.nq64 + qt) * 256 + r;
    const bool on = row < p.Lq;
    if (sub == 0) st[0] = on ? p.lse[((long long)b * p.H + h) * p.Lq + row] * LOG2E - p.shift : 0.f;
    if (sub == 1) st[64] = on ? -s : 0.f;
    if (sub == 2) ((int*)st)[128] = on ? row_pos(p, b, row) : 0;
    if (threadIdx.x < 64) {                                         // the tile's positions: smallest, largest, whether they follow one another
        const int at = row_pos(p, b, min(qt * 64 + (int)threadIdx.x, p.Lq - 1)), first = __builtin_amdgcn_readfirstlane(at);
        const bool line = __builtin_amdgcn_ballot_w64(qt * 64 + (int)threadIdx.x < p.Lq && at != first + (int)threadIdx.x) == 0;
        const int lo = line ? first : wave_min(at), hi = line ? first + 63 : wave_max(at);
        int* x = (int*)(p.stat + (((long long)b * p.H + h) * p.nq64 + qt) * 256) + 192;
        x[threadIdx.x] = threadIdx.x == 0 ? lo : threadIdx.x == 1 ? hi : threadIdx.x == 2 ? (int)line : 0;
    }
    if (h == 0 && threadIdx.x < 64) {
        const Vis v = load_vis(p, b, qt * 64 + threadIdx.x);
        const long long tile = (long long)b * p.nq64 + qt;
        int* vp = p.vis + tile * 256 + threadIdx.x;
        vp[0] = v.alo; vp[64] = v.na; vp[128] = v.blo; vp[192] = v.nb;
        int x[8] = {v.na ? v.alo : 0x7fffffff, v.na ? v.alo + v.na : 0, v.nb ? v.blo : 0x7fffffff, v.nb ? v.blo + v.nb : 0,
                    v.na ? v.alo : 0x7fffffff, v.na ? v.alo + v.na : 0, v.nb ? v.blo : 0x7fffffff, v.nb ? v.blo + v.nb : 0};
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = (i == 0 || i == 2 || i == 5 || i == 7) ? wave_min(x[i]) : wave_max(x[i]);
        if (threadIdx.x == 0) {
#pragma unroll
            for (int i = 0; i < 8; ++i) p.tiles[tile * 8 + i] = x[i];
        }
    }
}

// one wave per key: the parts' dK and dV, added in part order
template <int D>
__global__ __launch_bounds__(256) void range_kvjoin_kernel(const RArgs p) {
    const int lane = threadIdx.x & 63;
    const long long w = (long long)blockIdx.x * 4 + (threadIdx.x >> 6), keys = (long long)p.B * p.Hk * p.Lk;
    if (w >= keys) return;
    const int bk = (int)(w / p.Lk), j = (int)(w - (long long)bk * p.Lk), b = bk / p.Hk, hk = bk - b * p.Hk;
    float k[2] = {0.f, 0.f}, v[2] = {0.f, 0.f};
    for (int s = 0; s < p.kv_split; ++s) {
        const float* a = p.kv_parts + (s * keys + w) * (2 * D) + lane * (D / 64);
#pragma unroll
        for (int c = 0; c < D / 64; ++c) { k[c] += a[c]; v[c] += a[D + c]; }
    }
    bool bad = false;
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
        bad = bad || !(fabsf(k[c]) < __builtin_inff()) || !(fabsf(v[c]) < __builtin_inff());
        k[c] *= p.dscale;
    }
    if (__builtin_amdgcn_ballot_w64(bad) != 0 && strangers<D, true>(p, b, hk, j & ~31)) {
        exact_dkv<D>(p, b, hk, j);
        return;
    }
    store_row<D>(p.dk.p + b * p.dk.bs + j * p.dk.ld + hk * p.dk.hs, k);
    store_row<D>(p.dv.p + b * p.dv.bs + j * p.dv.ld + hk * p.dv.hs, v);
}

// Adds the 32 x 32 block dT (lane: row lane % 32, keys in registers) to the wave's table of distances.  Rows that follow one another
// make every distance a diagonal: 16 rows at a time go to LDS with 32 columns of zeros between them, and lane l sums diagonal
// l - 15 without a test.  d0 = distance of key 0 of the block from row 0.  (One LDS float add per pair instead: about 200 cycles per
// instruction, 57 us for the query gradients of 2 x 12 heads x 301 rows instead of 30.)
constexpr int SKEW = 16 * 64 + 64;                          // floats per wave
PF_DEVICE void add_diagonals(const f32x16_t& dt, float* skew, float* hist, int R, int d0, float& below, float& above) {
    const int lane = threadIdx.x & 63, hi = lane >> 5, r = lane & 15;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        if (((lane >> 4) & 1) == half) {
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4) {
                f32x4_t w;
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = dt[4 * q4 + e];
                *(f32x4_t*)(skew + 32 + 64 * r + 8 * q4 + 4 * hi) = w;
            }
        }
        __builtin_amdgcn_wave_barrier();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (lane < 47) {
            float a = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) a += skew[32 + 65 * i + lane - 15];
            const int d = d0 - 16 * half + lane - 15;
            if (d <= -R) below += a;
            else if (d >= R) above += a;
            else hist[d + R] += a;
        }
        __builtin_amdgcn_wave_barrier();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
}

// The same for rows at any positions: a row's distances differ, so row after row the lanes (keys now) add to distinct entries.
PF_DEVICE void add_rowwise(const f32x16_t& dt, float* skew, float* hist, int R, int key0, int pos, float& below, float& above) {
    const int lane = threadIdx.x & 63, hi = lane >> 5, r = lane & 15;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        if (((lane >> 4) & 1) == half) {
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4) {
                f32x4_t w;
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = dt[4 * q4 + e];
                *(f32x4_t*)(skew + 32 + 64 * r + 8 * q4 + 4 * hi) = w;
            }
        }
        __builtin_amdgcn_wave_barrier();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        for (int i = 0; i < 16; ++i) {
            const int d = key0 + lane - __builtin_amdgcn_readlane(pos, 16 * half + i);
            if (lane < 32) {
                const float a = skew[32 + 64 * i + lane];
                if (d <= -R) below += a;
                else if (d >= R) above += a;
                else hist[d + R] += a;
            }
            __builtin_amdgcn_wave_barrier();
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
    }
}

// dQ of 128 rows of one head (a wave's 32 rows held in registers; KS = 2: 64 rows, as in the forward kernel) over its key tiles, and
// this workgroup's part of dbias: every wave adds dT of its pairs into a table of its own (pairs behind the table's ends are summed
// in registers), the tables are added in wave order: no atomics, the same bits every time.
// Keys of a tile.  D = 128 with a bias: with 64 of them the distance tables leave one workgroup per compute unit, 32 let two in (the
// whole gradient of 4 x 3000 causal rows of 32 heads: 1620 instead of 2160 us).  KS = 2 needs 64, so it takes all registers instead.
template <int D, int MODE, int KS>
constexpr int DQ_KB = D == 128 && (MODE & 2) && KS == 1 ? 32 : 64;
template <int D, int MODE, int KS>
PF_DEVICE void row_gradients(const RArgs& p, int block) {
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    constexpr bool CAP = MODE & 1, BIAS = MODE & 2;
    constexpr int KB = DQ_KB<D, MODE, KS>, TILE = KB * 2 * D, BUF = 2 * TILE, RW = 4 / KS, NI = KB / 32 / KS;
    int* const red = (int*)(smem + 2 * BUF);
    Cover* const cover = (Cover*)(red + 16);
    float* const meet = (float*)(red + 20);                         // KS = 2: [row wave] whole
    float* const tab_ = meet + 4;
    const int NB = 2 * p.R + 1, TS = (table_floats(p.R) + 3) / 4 * 4;
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), rw = wid % RW, kw = wid / RW;
    float* const hists = tab_ + TS;
    float* const hist = hists + wid * NB;
    float* const skew = hists + (4 * NB + 3) / 4 * 4 + wid * SKEW;
    const Place at = heavy_first(block, p.nqt, p.nqt * p.H * p.B);
    const int bh = at.head, b = bh / p.H, h = bh - b * p.H, hk = h / p.G;
    const int qt = p.nqt - 1 - at.rank;
    const int hi = lane >> 5, row0 = (qt * RW + rw) * 32, row = row0 + (lane & 31), rc = min(row, p.Lq - 1);
    const Vis vis = load_vis(p, b, row);
    const int pos = BIAS ? row_pos(p, b, rc) : 0;
    const Bounds wb = wave_bounds(vis);
    const TileList tl = workgroup_tiles<KB>(wb, red, cover, wid, lane);
    const Stager<D, KB, 4> sk_(p.k.ld, wid, lane), sv_(p.v.ld, wid, lane);
    const bf16_t* const K = p.k.p + b * p.k.bs + hk * p.k.hs;
    const bf16_t* const V = p.v.p + b * p.v.bs + hk * p.v.hs;
    auto issue = [&](int n, bool begin = false) {
        const int j0 = tl.at(n) * KB;
        char* buf = smem + (n & 1) * BUF;
        if (begin ? tl.keys.whole(j0, j0 + KB) : tl.inner(n)) {
            sk_.whole(K, p.k.ld, j0, buf, wid);
            sv_.whole(V, p.v.ld, j0, buf + TILE, wid);
        } else {
            const Cover c = begin ? tl.keys : scalar(*cover);
            sk_.part(K, p.k.ld, j0, c, buf, wid, lane);
            sv_.part(V, p.v.ld, j0, c, buf + TILE, wid, lane);
        }
    };
    if (tl.n > 0) issue(0, true);                  // the first tile is on its way before the rows are read
    const float* const tab = BIAS ? load_table(p, h, tab_, 1.f) : nullptr;
    if (BIAS && p.dbias) {
        for (int i = lane; i < NB; i += 64) hist[i] = 0.f;
        for (int i = lane; i < SKEW; i += 64) skew[i] = 0.f;
    }
    bf16x8_t qf[D / 16], of[D / 16];
    {
        const bf16_t* q = p.q.p + b * p.q.bs + rc * p.q.ld + h * p.q.hs + hi * 8;
        const bf16_t* g = p.dO.p + b * p.dO.bs + rc * p.dO.ld + h * p.dO.hs + hi * 8;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
            qf[ks] = *(const bf16x8_t*)(q + ks * 16);
            of[ks] = *(const bf16x8_t*)(g + ks * 16);
        }
    }
    const float* const st = p.stat + (((long long)b * p.H + h) * p.nq64 + (rc >> 6)) * 256 + (rc & 63);
    const float ls = st[0], de = st[64];                            // log-sum-exp (base 2, less the shift), -delta
    // dbias is a 32-bit result: with a bias the scores stay in natural units here, so that only their difference from the row's lse
    // is rounded again by the change of base (lse, cap and bias times log2 e leave 5e-7 each, the same for whole rows and distances)
    const float lse = BIAS ? p.lse[((long long)b * p.H + h) * p.Lq + rc] - p.shift_n : 0.f;
    const unsigned roff = row_offset<D>(lane), t0 = tr_offset<D>(lane, 0), t8 = tr_offset<D>(lane, 8);
    f32x16_t dq[D / 32];
#pragma unroll
    for (int c = 0; c < D / 32; ++c) dq[c] = zero16();
    float below = 0.f, above = 0.f;                 // dbias of distances <= -R and >= R
    const int pmin = BIAS ? wave_min(pos) : 0, pmax = BIAS ? wave_max(pos) : 0;
    const int pos0 = __builtin_amdgcn_readfirstlane(pos);
    const bool in_line = __builtin_amdgcn_ballot_w64(row < p.Lq && pos != pos0 + (lane & 31)) == 0;
    bool whole = !BIAS;                             // as in the forward kernel
    for (int n = 0; n < tl.n; ++n) {
        drain_barrier();
        if (n + 1 < tl.n) issue(n + 1);
        const int j0 = tl.at(n) * KB + kw * 32 * NI;                // this wave's keys of the tile
        const char* sk = smem + (n & 1) * BUF + kw * NI * 64 * D;
        const char* sv = sk + TILE;
        const bool full = wb.full(j0, j0 + 32 * NI);
        if (!full) {
            whole = false;
            if (!wb.any(j0, j0 + 32 * NI)) continue;
        }
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            f32x16_t s = zero16(), dp;
#pragma unroll
            for (int r = 0; r < 16; ++r) dp[r] = de;
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks) {
                s = mfma(row_frag<D>(sk, roff, i, ks), qf[ks], s);
                dp = mfma(row_frag<D>(sv, roff, i, ks), of[ks], dp);
            }
            const int k0 = j0 + 32 * i + 4 * hi;
            f32x16_t fac;                                           // dbias wants dT without the slope
            if (CAP) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    float slope;
                    s[r] = capped<MODE>(p, s[r], slope);
                    if (BIAS) fac[r] = slope;
                    else dp[r] *= slope;
                }
            }
            if (BIAS) add_bias<1>(p, s, p.zn, tab, k0 - pos, j0 + 32 * i - pmax, j0 + 32 * i + 31 - pmin);
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                if (BIAS) s[r] = s[r] == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f((s[r] - lse) * LOG2E) * dp[r];
                else s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], p.zs, -ls)) * dp[r];
            }
            if (!full) {
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = sees(vis, k0 + reg_row(r)) ? s[r] : 0.f;
            }
            if (BIAS && p.dbias) {
                const int lo = j0 + 32 * i - pmax, hi_ = j0 + 32 * i + 31 - pmin;     // distances of this block, wave-uniform
                if (hi_ <= -p.R || lo >= p.R) {
                    float a = 0.f;
#pragma unroll
                    for (int r = 0; r < 16; ++r) a += s[r];
                    if (lo >= p.R) above += a;
                    else below += a;
                } else if (in_line) {
                    add_diagonals(s, skew, hist, p.R, j0 + 32 * i - pos0, below, above);
                } else {
                    add_rowwise(s, skew, hist, p.R, j0 + 32 * i, pos, below, above);
                }
            }
            if (CAP && BIAS) {
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] *= fac[r];
            }
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const bf16x8_t zf = half_of(s, g);
#pragma unroll
                for (int c = 0; c < D / 32; ++c) dq[c] = mfma(tr_frag<D>(sk, t0, t8, c, 2 * i + g), zf, dq[c]);
            }
        }
    }
    if constexpr (KS == 2) {
        float* const acc = (float*)smem + rw * (D / 32) * 16 * 64;
        __syncthreads();
        if (kw == 1) {
#pragma unroll
            for (int c = 0; c < D / 32; ++c)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[(c * 16 + r) * 64 + lane] = dq[c][r];
            if (lane == 0) meet[rw] = whole ? 1.f : 0.f;
        }
        __syncthreads();
        if (kw == 0) {
            whole = whole && meet[rw] != 0.f;
#pragma unroll
            for (int c = 0; c < D / 32; ++c)
#pragma unroll
                for (int r = 0; r < 16; ++r) dq[c][r] += acc[(c * 16 + r) * 64 + lane];
        }
    }
    const bool store = row < p.Lq && kw == 0;
    const bool bad = any_nonfinite<D / 32>(dq) && !whole && store;
    unsigned long long redo = __builtin_amdgcn_ballot_w64(bad);
    redo = (redo | (redo >> 32)) & 0xffffffffull;
    if (store && !((redo >> (lane & 31)) & 1)) store_cols<D>(p.dq.p + b * p.dq.bs + row * p.dq.ld + h * p.dq.hs, dq, p.dscale);
    while (redo) {
        const int i = __builtin_ctzll(redo);
        redo &= redo - 1;
        exact_dq<D>(p, b, h, row0 + i);
    }
    if (BIAS && p.dbias) {
        below = wave_add(below);
        above = wave_add(above);
        if (lane == 0) {
            hist[0] = below;
            hist[2 * p.R] = p.R == 0 ? below + above : above;
        }
        __syncthreads();
        float* out = p.dbias_parts + ((long long)bh * p.nqt + qt) * NB;
        for (int i = threadIdx.x; i < NB; i += 256) out[i] = (hists[i] + hists[NB + i]) + (hists[2 * NB + i] + hists[3 * NB + i]);
    }
}

template <int D, int MODE, int KS>
__global__ __launch_bounds__(256, D == 128 && (MODE & 2) && KS == 2 ? 1 : 2) void range_dq_kernel(const RArgs p) { row_gradients<D, MODE, KS>(p, blockIdx.x); }

// dK, dV of 128 keys of one key head: 4 waves x 32 keys, looping over the row tiles (of every query head that shares the key head)
// that see any of them.  The bounds of 64 tiles are tested at once (one lane each); the next tile is in flight while one is used.
// -delta enters through the C operand of the dP product.  kv_split > 1: this workgroup takes an even part of the (head, tile)
// pairs that the keys need and leaves 32-bit sums for range_kvjoin_kernel.
//
// D = 64: 64-row tiles, K and both results in registers, V in LDS: three waves per SIMD (when it was built 1370 us for the whole gradient of 30
// heads of the 7808-row video sequence; V in registers and two waves 1430 us; with a bias table the third wave spills: 53 instead of
// 48 us at 2 x 12 heads of 301 rows).  D = 128 has twice the results (128 registers): 32-row tiles and V in LDS leave room for
// a second workgroup (with V in registers and 64-row tiles one wave per SIMD ran everything in series, 8400 cycles per tile,
// 800 of its instructions register moves).
//
// Neither gradient needs the other: small problems run both in this launch (BOTH), where the row workgroups fill what the key
// workgroups leave of the chip; the number of key workgroups is padded to the XCDs, so that a block's place tells its XCD in both.
template <int D, int MODE>
constexpr bool KV_V_LDS = D == 128 || !(MODE & 2);
template <int D, int MODE, bool BOTH>
__global__ __launch_bounds__(256, D == 64 && !(MODE & 2) ? 3 : 2) void range_dkv_kernel(const RArgs p) {
    if constexpr (BOTH) {
        if ((int)blockIdx.x >= p.key_pad) return row_gradients<D, MODE, 2>(p, blockIdx.x - p.key_pad);
        if ((int)blockIdx.x >= p.key_wgs) return;
    }
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    constexpr bool CAP = MODE & 1, BIAS = MODE & 2, VLDS = KV_V_LDS<D, MODE>;
    constexpr int RT = D == 64 ? 64 : 32, HALVES = 64 / RT, TILE = RT * 2 * D, BUF = 2 * TILE + 2048, VTILE = VLDS ? 32 * 2 * D : 0;
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    char* const vtile = smem + 2 * BUF + wid * VTILE;
    float* const tab_ = (float*)(smem + 2 * BUF + 4 * VTILE);
    const float* tab = nullptr;
    const Place at = heavy_first(blockIdx.x, p.nkt * p.kv_split, p.nkt * p.kv_split * p.Hk * p.B);
    const int bk = at.head, kt = at.rank / p.kv_split, part = at.rank - kt * p.kv_split;
    const int b = bk / p.Hk, hk = bk - b * p.Hk;
    const int hi = lane >> 5;
    const int w0 = kt * 128 + wid * 32, key = w0 + (lane & 31);
    const int nq = p.nq64;
    const int* const tiles = p.tiles + (long long)b * nq * 8;
    bf16x8_t kf[D / 16], vf[VLDS ? 1 : D / 16];
    {
        const long long kr = min(key, p.Lk - 1);
        const bf16_t* k = p.k.p + b * p.k.bs + kr * p.k.ld + hk * p.k.hs + hi * 8;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) kf[ks] = *(const bf16x8_t*)(k + ks * 16);
        if constexpr (VLDS) {
            const Stager<D, 32, 1> s(p.v.ld, 0, lane);
            s.upto(p.v.p + b * p.v.bs + hk * p.v.hs, p.v.ld, min(w0, p.Lk - 1), p.Lk - 1, vtile, 0, lane);
        } else {
            const bf16_t* v = p.v.p + b * p.v.bs + kr * p.v.ld + hk * p.v.hs + hi * 8;
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks) vf[ks] = *(const bf16x8_t*)(v + ks * 16);
        }
    }
    const unsigned roff = row_offset<D>(lane), t0 = tr_offset<D>(lane, 0), t8 = tr_offset<D>(lane, 8);
    f32x16_t dk[D / 32], dv[D / 32];
#pragma unroll
    for (int c = 0; c < D / 32; ++c) dk[c] = dv[c] = zero16();
    const int wg0 = kt * 128, wg1 = min(wg0 + 128, p.Lk);
    const Stager<D, RT, 4> sq_(p.q.ld, wid, lane), so_(p.dO.ld, wid, lane);

    // ---- the (head g, 64-row tile) pairs of this part, 64 tiles at a time: which the workgroup needs, which this wave sees at all,
    //      which it sees whole
    unsigned long long need = 0, some = 0, all = 0;
    auto test = [&](int base) {
        const int n = base + lane;
        int x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (n < nq) {
            const u32x4_t u = *(const u32x4_t*)(tiles + n * 8LL), v = *(const u32x4_t*)(tiles + n * 8LL + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) { x[i] = (int)u[i]; x[4 + i] = (int)v[i]; }
        }
        need = __builtin_amdgcn_ballot_w64((x[0] < wg1 && x[1] > wg0) || (x[2] < wg1 && x[3] > wg0));
        some = __builtin_amdgcn_ballot_w64((x[0] < w0 + 32 && x[1] > w0) || (x[2] < w0 + 32 && x[3] > w0));
        all = __builtin_amdgcn_ballot_w64((x[4] <= w0 && x[5] >= w0 + 32) || (x[6] <= w0 && x[7] >= w0 + 32));
    };
    int g = 0, base = 0, skip = 0, left = 0x7fffffff, group_g = 0, group_base = 0;
    if (p.kv_split > 1) {
        int per_head = 0;
        for (int n = 0; n < nq; n += 64) {
            test(n);
            per_head += __builtin_popcountll(need);
        }
        need = 0;
        const long long pairs = (long long)per_head * p.G, from = pairs * part / p.kv_split;
        left = (int)(pairs * (part + 1) / p.kv_split - from);
        g = per_head ? (int)(from / per_head) : p.G;
        skip = (int)(from - (long long)g * per_head);
    }
    struct Item { int g, qt, half; bool any, full; };
    auto pop = [&]() -> Item {
        while (need == 0) {
            if (left == 0 || g >= p.G || nq == 0) return {-1, 0, 0, false, false};
            test(base);
            group_g = g;
            group_base = base;
            base += 64;
            if (base >= nq) { base = 0; ++g; }
            while (skip > 0 && need != 0) { need &= need - 1; --skip; }
        }
        if (left == 0) return {-1, 0, 0, false, false};
        const int i = __builtin_ctzll(need);
        need &= need - 1;
        --left;
        return {group_g, group_base + i, 0, ((some >> i) & 1) != 0, ((all >> i) & 1) != 0};
    };
    auto follow = [&](const Item& c) -> Item {                      // the other half of a tile, if it has rows, or the next tile
        if (HALVES == 2 && c.half == 0 && c.qt * 64 + RT < p.Lq) return {c.g, c.qt, 1, c.any, c.full};
        return pop();
    };
    auto issue = [&](const Item& n, int buf) {
        const int h = hk * p.G + n.g, r0 = n.qt * 64 + n.half * RT;
        char* dst = smem + buf * BUF;
        sq_.upto(p.q.p + b * p.q.bs + h * p.q.hs, p.q.ld, r0, p.Lq - 1, dst, wid, lane);
        so_.upto(p.dO.p + b * p.dO.bs + h * p.dO.hs, p.dO.ld, r0, p.Lq - 1, dst + TILE, wid, lane);
        if (wid == 0) glds16(p.stat + (((long long)b * p.H + h) * nq + n.qt) * 256 + lane * 4, dst + 2 * TILE);
        if (wid == 1) glds16(p.vis + ((long long)b * nq + n.qt) * 256 + lane * 4, dst + 2 * TILE + 1024);
    };
    Item cur = pop();
    int buf = 0, table_of = -1;
    if (cur.g >= 0) issue(cur, 0);
    while (cur.g >= 0) {
        drain_barrier();
        if (BIAS && cur.g != table_of) {                            // uniform: another head, another bias table
            table_of = cur.g;
            tab = load_table(p, hk * p.G + table_of, tab_);
            drain_barrier();
        }
        const Item nxt = follow(cur);
        if (nxt.g >= 0) issue(nxt, buf ^ 1);
        if (cur.any) {
            const char* sq = smem + buf * BUF;
            const char* so = sq + TILE;
            const float* st = (const float*)(sq + 2 * TILE) + cur.half * RT;
            const int* vi = (const int*)(sq + 2 * TILE + 1024) + cur.half * RT;
#pragma unroll
            for (int qb = 0; qb < RT / 32; ++qb) {
                f32x16_t s = zero16(), dp;
#pragma unroll
                for (int q4 = 0; q4 < 4; ++q4) {
                    const f32x4_t de = *(const f32x4_t*)(st + 64 + qb * 32 + 8 * q4 + 4 * hi);
#pragma unroll
                    for (int e = 0; e < 4; ++e) dp[4 * q4 + e] = de[e];
                }
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks) {
                    s = mfma(row_frag<D>(sq, roff, qb, ks), kf[ks], s);
                    dp = mfma(row_frag<D>(so, roff, qb, ks), VLDS ? row_frag<D>(vtile, roff, 0, ks) : vf[VLDS ? 0 : ks], dp);
                }
                if (CAP) {                                          // the slope goes to dP at once: P dP slope is all that follows
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        float slope;
                        s[r] = capped<MODE>(p, s[r], slope);
                        dp[r] *= slope;
                    }
                }
                if (BIAS) {
                    const int* of_tile = (const int*)(sq + 2 * TILE) + 192;
                    const int lo = __builtin_amdgcn_readfirstlane(of_tile[0]), hi_ = __builtin_amdgcn_readfirstlane(of_tile[1]);
                    if (__builtin_amdgcn_readfirstlane(of_tile[2]) != 0) {        // consecutive rows
                        const int p0 = lo + cur.half * RT + qb * 32;
                        add_bias<-1>(p, s, p.zs, tab, key - p0 - 4 * hi, w0 - p0 - 31, w0 + 31 - p0);
                    } else if (reach(p.R, w0 - hi_, w0 + 31 - lo) == FAR) {
                        add_bias<-1>(p, s, p.zs, tab, 0, w0 - hi_, w0 + 31 - lo);
                    } else {
#pragma unroll
                        for (int q4 = 0; q4 < 4; ++q4) {
                            const u32x4_t pos = *(const u32x4_t*)((const int*)st + 128 + qb * 32 + 8 * q4 + 4 * hi);
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const int r = 4 * q4 + e;
                                s[r] = __builtin_fmaf(s[r], p.zs, tab[min(max(key - (int)pos[e], -p.R), p.R)]);
                            }
                        }
                    }
                }
#pragma unroll
                for (int q4 = 0; q4 < 4; ++q4) {
                    const int r0 = qb * 32 + 8 * q4 + 4 * hi;
                    const f32x4_t ls = *(const f32x4_t*)(st + r0);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int r = 4 * q4 + e;
                        if (BIAS) s[r] = s[r] == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(s[r] - ls[e]);
                        else s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], p.zs, -ls[e]));
                        dp[r] *= s[r];
                    }
                }
                if (!cur.full) {
#pragma unroll
                    for (int q4 = 0; q4 < 4; ++q4) {
                        const int* v = vi + qb * 32 + 8 * q4 + 4 * hi;
                        const u32x4_t alo = *(const u32x4_t*)v, na = *(const u32x4_t*)(v + 64), blo = *(const u32x4_t*)(v + 128), nb = *(const u32x4_t*)(v + 192);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const bool ok = (unsigned)key - alo[e] < na[e] || (unsigned)key - blo[e] < nb[e];
                            s[4 * q4 + e] = ok ? s[4 * q4 + e] : 0.f;
                            dp[4 * q4 + e] = ok ? dp[4 * q4 + e] : 0.f;
                        }
                    }
                }
                // as in the forward kernel (2 x 2500 rows of 16 / 4 heads: 338 -> 329 us for the whole gradient; D = 64: 3 % slower)
                if (D == 128) __builtin_amdgcn_s_setprio(1);
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    const bf16x8_t pf = half_of(s, g), zf = half_of(dp, g);
#pragma unroll
                    for (int c = 0; c < D / 32; ++c) {
                        dv[c] = mfma(tr_frag<D>(so, t0, t8, c, 2 * qb + g), pf, dv[c]);
                        dk[c] = mfma(tr_frag<D>(sq, t0, t8, c, 2 * qb + g), zf, dk[c]);
                    }
                }
                if (D == 128) __builtin_amdgcn_s_setprio(0);
            }
        }
        cur = nxt;
        buf ^= 1;
    }
    if (p.kv_split > 1) {
        if (key < p.Lk) {
            float* out = p.kv_parts + (((long long)part * p.B * p.Hk + bk) * p.Lk + key) * (2 * D) + 4 * hi;
#pragma unroll
            for (int c = 0; c < D / 32; ++c)
#pragma unroll
                for (int q4 = 0; q4 < 4; ++q4) {
                    f32x4_t x, y;
#pragma unroll
                    for (int e = 0; e < 4; ++e) { x[e] = dk[c][4 * q4 + e]; y[e] = dv[c][4 * q4 + e]; }
                    *(f32x4_t*)(out + 32 * c + 8 * q4) = x;
                    *(f32x4_t*)(out + D + 32 * c + 8 * q4) = y;
                }
        }
        return;
    }
    const bool bad = key < p.Lk && (any_nonfinite<D / 32>(dk) || any_nonfinite<D / 32>(dv));
    unsigned long long redo = __builtin_amdgcn_ballot_w64(bad);
    if (redo != 0 && !strangers<D, BIAS>(p, b, hk, w0)) redo = 0;
    redo = (redo | (redo >> 32)) & 0xffffffffull;
    if (key < p.Lk && !((redo >> (lane & 31)) & 1)) {
        store_cols<D>(p.dk.p + b * p.dk.bs + key * p.dk.ld + hk * p.dk.hs, dk, p.dscale);
        store_cols<D>(p.dv.p + b * p.dv.bs + key * p.dv.ld + hk * p.dv.hs, dv, 1.f);
    }
    while (redo) {
        const int j = __builtin_ctzll(redo);
        redo &= redo - 1;
        exact_dkv<D>(p, b, hk, w0 + j);
    }
}

// dbias[h][i] = sum over batch entries and row tiles of the parts, in order: 64 entries per workgroup, 4 groups of parts.  A hidden
// distance has none, whatever keys that are not finite left there.
__global__ __launch_bounds__(256) void range_dbias_kernel(const RArgs p) {
    __shared__ float red[4][64];
    const int NB = 2 * p.R + 1, i = blockIdx.x * 64 + (threadIdx.x & 63), h = blockIdx.y, grp = threadIdx.x >> 6;
    float a = 0.f;
    if (i < NB)
        for (int u = grp; u < p.B * p.nqt; u += 4) a += p.dbias_parts[(((long long)(u / p.nqt) * p.H + h) * p.nqt + u % p.nqt) * NB + i];
    red[grp][threadIdx.x & 63] = a;
    __syncthreads();
    if (grp == 0 && i < NB) p.dbias[(long long)h * NB + i] = p.bias[(long long)h * NB + i] <= HIDDEN ? 0.f : (red[0][threadIdx.x] + red[1][threadIdx.x]) + (red[2][threadIdx.x] + red[3][threadIdx.x]);
}

// ---------------------------------------------------------------------------------------------- host side
bool bad_view(const pf_rows_view& v) {
    return !v.p || ((uintptr_t)v.p & 15) || v.batch < 0 || v.row < 0 || v.head < 0 || ((v.batch | v.row | v.head) & 7) || v.row >= (1 << 25);
}
View view(const pf_rows_view& v) { return {(bf16_t*)v.p, v.batch, v.row, v.head}; }

const char* check_ranges(const pf_attn_ranges_desc* d, bool grad) {
    if (!d) return "pf_attention_ranges: null descriptor";
    if (d->D != 64 && d->D != 128) return "pf_attention_ranges: head_dim must be 64 or 128";
    if (d->B < 0 || d->H < 0 || d->Hkv < 0 || d->Lq < 0 || d->Lk < 0) return "pf_attention_ranges: negative size";
    if ((d->H == 0) != (d->Hkv == 0) || (d->H && d->H % d->Hkv)) return "pf_attention_ranges: the number of heads must be a multiple of the key heads";
    if (d->Lq > (1 << 30) || d->Lk > (1 << 30)) return "pf_attention_ranges: more than 2^30 rows or keys";
    if (!(d->scale - d->scale == 0.f) || d->scale <= 0.f) return "pf_attention_ranges: scale must be positive and finite";
    if (!(d->cap >= 0.f) || d->cap > 1e30f) return "pf_attention_ranges: cap must be 0 (none) or positive and finite";
    if (d->cap > 0.f && !(d->scale / d->cap < 1e30f)) return "pf_attention_ranges: cap too small for this scale";
    if ((d->a_lo == nullptr) != (d->a_hi == nullptr) || (d->b_lo == nullptr) != (d->b_hi == nullptr) || (d->b_lo && !d->a_lo))
        return "pf_attention_ranges: a range needs its start and its end, the second one the first";
    if (d->range_batch < 0 || d->q_pos_batch < 0) return "pf_attention_ranges: negative stride";
    if (d->bias && (d->bias_radius < 0 || d->bias_radius > MAX_RADIUS)) return "pf_attention_ranges: bias_radius must be in 0..512";
    if (d->dbias && !d->bias) return "pf_attention_ranges: a bias gradient without a bias";
    const bool rows = d->B && d->H && d->Lq, keys = d->B && d->H && d->Lk;
    const char* const bad = "pf_attention_ranges: tensors must be 16-byte aligned with strides that are multiples of 8 elements, rows less than 2^25 elements apart";
    if ((rows && (bad_view(d->Q) || bad_view(d->O))) || (keys && (bad_view(d->K) || bad_view(d->V)))) return bad;
    if (grad) {
        if ((rows && (bad_view(d->dO) || bad_view(d->dQ))) || (keys && (bad_view(d->dK) || bad_view(d->dV)))) return bad;
        if (rows && !d->LSE) return "pf_attention_ranges_bwd: null LSE";
    }
    return nullptr;
}

// outputs share no element with an input or each other; O may be Q, element for element
const char* check_overlap(const pf_attn_ranges_desc* d, bool grad) {
    struct One { const pf_rows_view* v; int L, H; };
    const One q = {&d->Q, d->Lq, d->H}, k = {&d->K, d->Lk, d->Hkv}, v = {&d->V, d->Lk, d->Hkv}, o = {&d->O, d->Lq, d->H};
    const One dO = {&d->dO, d->Lq, d->H}, dq = {&d->dQ, d->Lq, d->H}, dk = {&d->dK, d->Lk, d->Hkv}, dv = {&d->dV, d->Lk, d->Hkv};
    const int B = d->B, D = d->D;
    auto share = [&](const One& x, const One& y) { return rows_share(*x.v, B, x.L, x.H, *y.v, B, y.L, y.H, D); };
    auto folded = [&](const One& x) { return rows_folded(*x.v, B, x.L, x.H, D); };
    if (!grad) {
        if (folded(o)) return "pf_attention_ranges_bf16: the output overlaps itself";
        if (share(o, k) || share(o, v)) return "pf_attention_ranges_bf16: the output overlaps the keys or values";
        if (!rows_same(d->O, d->Q, B, d->Lq, d->H) && share(o, q)) return "pf_attention_ranges_bf16: the output overlaps the queries and is not them";
        return nullptr;
    }
    const One out[3] = {dq, dk, dv}, in[5] = {q, k, v, o, dO};
    for (int x = 0; x < 3; ++x) {
        if (folded(out[x])) return "pf_attention_ranges_bwd: a gradient overlaps itself";
        for (const One& y : in)
            if (share(out[x], y)) return "pf_attention_ranges_bwd: a gradient overlaps an input";
        for (int y = 0; y < x; ++y)
            if (share(out[x], out[y])) return "pf_attention_ranges_bwd: two gradients overlap";
    }
    return nullptr;
}

constexpr long long MOST_WGS = (1 << 24) - 1;          // of 256 threads: 2^32 threads of a launch wrap around without an error

// the form with 32 (row, head) pairs per workgroup and the keys split: where even 64-row workgroups would be few (1 x 700 rows over 1400
// keys of 32 heads of 128, 192 in the count below: 87 us, rows 43; 64 rows over 8000 keys of 16 heads of 64, 16: 25 us, rows 82), and
// where one block of 32 pairs holds all rows that share a key head (each key is then read once, not once per query head)
bool few_rows(const pf_attn_ranges_desc* d) {
    return (long long)((d->Lq + 127) / 128) * d->H * d->B < 64 || (long long)d->Lq * (d->H / d->Hkv) <= 32;
}
// 64-row workgroups (KS = 2) instead of 128-row ones where those would be few: half the chain per wave for twice the tile traffic.
// Forward: 21.5 instead of 22 us at 2 x 64 heads of 512 rows of 64; 55 instead of 67 us with 128-row workgroups at 16 x 16 heads of
// 500 rows of 128.  dQ: 48 instead of 55 us for the whole gradient of 2 x 12 heads of 301 rows of 64, 240 instead of 263 us for that
// of 16 heads of 4001 rows of 128.
bool small_fwd(int D, long long Lq, long long H, long long B) { return (Lq + 127) / 128 * H * B < (D == 64 ? 1024 : 512); }
bool small_dq(int D, long long Lq, long long H, long long B) { return (Lq + 127) / 128 * H * B < (D == 64 ? 1024 : 2048); }
int row_groups(int Lq, bool small) { return small ? (Lq + 63) / 64 : (Lq + 127) / 128; }
// SERIES also where the bias's gradient is wanted: it is a 32-bit result, and what cap_u leaves of the cap would be all of its error; and
// where the caller asks for it
bool series(const pf_attn_ranges_desc* d) { return d->cap > 64.f || (d->cap > 0.f && (d->dbias || d->precise)); }
int mode(const pf_attn_ranges_desc* d) { return (d->cap > 0.f ? 1 : 0) + (d->bias ? 2 : 0) + (series(d) ? 4 : 0); }
int row_blocks(const pf_attn_ranges_desc* d) { return (int)(((long long)d->Lq * (d->H / d->Hkv) + 31) / 32); }
int splits(const pf_attn_ranges_desc* d) {
    const long long units = (long long)row_blocks(d) * d->Hkv * d->B, tiles = (d->Lk + 31) / 32;
    long long n = 512 / units;
    if (n > tiles / 32) n = tiles / 32;                   // eight tiles per wave at least: the join is a launch of its own
    return (int)(n < 1 ? 1 : n);
}
long long fwd_bytes(const pf_attn_ranges_desc* d) {
    if (!d->B || !d->H || !d->Lq || !few_rows(d)) return 0;
    const int s = splits(d);
    return s > 1 ? (long long)row_blocks(d) * d->Hkv * d->B * s * 32 * (d->D + 2) * 4 : 0;
}
long long up16(long long n) { return (n + 15) / 16 * 16; }
// The (head, row tile) list of a key block in n parts: the longest chain shrinks as tiles / n (0.8 .. 1.3 us per tile), the parts'
// traffic grows as n units (128 keys, 8 D bytes each way: 26 .. 52 ns), so n = sqrt(25 tiles / units).  Whole gradients at 8 heads
// of 2000 rows over 2 key heads of 128: n = 8 96 us, 16 126 us; 12 heads over 3 of 4 x 300 rows of 64: n = 1 78 us, 2 53 us, 5 40 us;
// 16 heads of 2 x 1000 rows of 64: n = 1 52 us, 2 58 us, 3 66 us.
int kv_splits(const pf_attn_ranges_desc* d) {
    if (!d->B || !d->H || !d->Lk || !d->Lq) return 1;
    const long long units = (long long)((d->Lk + 127) / 128) * d->Hkv * d->B, tiles = (long long)((d->Lq + 63) / 64) * (d->H / d->Hkv);
    long long n = 1, most = 768 / units < 32 ? 768 / units : 32;
    while (n < most && (2 * n + 1) * (2 * n + 1) * units <= 100 * tiles) ++n;      // rounded
    return (int)n;
}
struct BwdSizes { long long stat, vis, tiles, parts, kv; long long all() const { return stat + vis + tiles + parts + kv; } };
BwdSizes bwd_sizes(const pf_attn_ranges_desc* d) {
    BwdSizes s;
    const long long nq = (d->Lq + 63) / 64;
    s.stat = (long long)d->B * d->H * nq * 1024;
    s.vis = (long long)d->B * nq * 1024;
    s.tiles = up16((long long)d->B * nq * 32);
    s.parts = d->dbias ? up16((long long)d->B * d->H * row_groups(d->Lq, small_dq(d->D, d->Lq, d->H, d->B)) * (2 * d->bias_radius + 1) * 4) : 0;
    const int n = kv_splits(d);
    s.kv = n > 1 ? (long long)n * d->B * d->Hkv * d->Lk * 2 * d->D * 4 : 0;
    return s;
}

RArgs range_args(const pf_attn_ranges_desc* d) {
    RArgs a{};
    a.q = view(d->Q); a.k = view(d->K); a.v = view(d->V); a.o = view(d->O);
    a.dO = view(d->dO); a.dq = view(d->dQ); a.dk = view(d->dK); a.dv = view(d->dV);
    a.lse = d->LSE;
    a.a_lo = d->a_lo; a.a_hi = d->a_hi; a.b_lo = d->b_lo; a.b_hi = d->b_hi; a.range_bs = d->range_batch;
    a.q_pos = d->q_pos; a.pos_bs = d->q_pos_batch;
    a.bias = d->bias; a.R = d->bias ? d->bias_radius : 0;
    a.scale = d->scale;
    a.cap2 = d->cap * LOG2E;
    a.series = series(d);
    const bool fast = d->cap > 0.f && !a.series;
    a.zc = d->cap > 0.f ? d->scale / d->cap * (fast ? 2.f * LOG2E : 1.f) : 0.f;
    a.zs = fast ? 2.f * a.cap2 : a.series ? a.cap2 : d->scale * LOG2E;
    a.shift = fast ? a.cap2 : 0.f;
    a.zn = fast ? 2.f * d->cap : a.series ? d->cap : d->scale;
    a.shift_n = fast ? d->cap : 0.f;
    a.dscale = fast ? 4.f * d->scale : d->scale;
    a.D = d->D; a.B = d->B; a.H = d->H; a.Hk = d->Hkv; a.G = d->H / d->Hkv; a.Lq = d->Lq; a.Lk = d->Lk;
    a.nkt = (d->Lk + 127) / 128; a.nq64 = (d->Lq + 63) / 64;
    return a;
}

#define CHECK_LAUNCH()                                              \
    do {                                                            \
        hipError_t e_ = hipGetLastError();                          \
        if (e_ != hipSuccess) return pf_set_err(hipGetErrorString(e_)); \
    } while (0)

template <int D, int MODE, int KS>
int launch_fwd_rows(const RArgs& a, hipStream_t stream) {
    const size_t lds = 4 * FWD_KB<D, KS> * 2 * D + 96 + (KS == 2 ? 2 * 192 * 4 : 0) + (MODE & 2 ? table_floats(MAX_RADIUS) * 4 : 0);
    PF_SET_MAX_LDS_ONCE((range_fwd_kernel<D, MODE, KS>), (int)lds);
    range_fwd_kernel<D, MODE, KS><<<(unsigned)(a.nqt * a.H * a.B), 256, lds, stream>>>(a);
    CHECK_LAUNCH();
    return 0;
}

template <int D, int MODE>
int launch_fwd(const RArgs& a, bool few, hipStream_t stream) {
    if (!few) return small_fwd(a.D, a.Lq, a.H, a.B) ? launch_fwd_rows<D, MODE, 2>(a, stream) : launch_fwd_rows<D, MODE, 1>(a, stream);
    const size_t lds = 4 * 4 * 32 * 2 * D + 64;                      // the meeting area [4][32][D + 4] fp32 is smaller
    PF_SET_MAX_LDS_ONCE((range_split_kernel<D, MODE>), (int)lds);
    range_split_kernel<D, MODE><<<(unsigned)(a.nrb * a.Hk * a.B * a.nsplit), 256, lds, stream>>>(a);
    CHECK_LAUNCH();
    if (a.nsplit > 1) {
        const long long rows = (long long)a.B * a.Hk * a.Lq * a.G;
        range_join_kernel<D><<<(unsigned)((rows + 3) / 4), 256, 0, stream>>>(a);
        CHECK_LAUNCH();
    }
    return 0;
}

template <int D, int MODE, int KS>
int lds_dq(int R) { return 4 * DQ_KB<D, MODE, KS> * 2 * D + 96 + (MODE & 2 ? (table_floats(R) + 3 + 4 * (2 * R + 1) + 3 + 4 * SKEW) * 4 : 0); }
template <int D, int MODE, bool BOTH>
int lds_dkv(int R) {
    const int rt = D == 64 ? 64 : 32, rows = BOTH ? lds_dq<D, MODE, 2>(R) : 0;
    const int keys = 2 * (2 * rt * 2 * D + 2048) + (KV_V_LDS<D, MODE> ? 4 * 32 * 2 * D : 0) + (MODE & 2 ? table_floats(R) * 4 : 0);
    return keys > rows ? keys : rows;
}

template <int D, int MODE, int KS>
int launch_dq(const RArgs& a, unsigned row_wgs, hipStream_t stream) {
    if (row_wgs == 0) return 0;
    PF_SET_MAX_LDS_ONCE((range_dq_kernel<D, MODE, KS>), (lds_dq<D, MODE, KS>(MAX_RADIUS)));
    range_dq_kernel<D, MODE, KS><<<row_wgs, 256, (size_t)lds_dq<D, MODE, KS>(a.R), stream>>>(a);
    CHECK_LAUNCH();
    return 0;
}

template <int D, int MODE>
int launch_bwd(const RArgs& a, hipStream_t stream) {
    if (a.Lq > 0) {
        range_prep_kernel<D><<<dim3((a.Lq + 63) / 64, a.H, a.B), 256, 0, stream>>>(a);
        CHECK_LAUNCH();
    }
    const unsigned row_wgs = (unsigned)(a.nqt * a.H * a.B);
    const bool small = small_dq(a.D, a.Lq, a.H, a.B);
    // with D = 128 and a bias the row workgroups' LDS would leave one key workgroup per compute unit
    constexpr bool BOTH = D == 64 || !(MODE & 2);
    if (BOTH && small) {
        if (a.key_wgs + row_wgs > 0) {
            PF_SET_MAX_LDS_ONCE((range_dkv_kernel<D, MODE, BOTH>), (lds_dkv<D, MODE, BOTH>(MAX_RADIUS)));
            range_dkv_kernel<D, MODE, BOTH><<<a.key_pad + row_wgs, 256, (size_t)lds_dkv<D, MODE, BOTH>(a.R), stream>>>(a);
            CHECK_LAUNCH();
        }
    } else {
        if (a.key_wgs > 0) {
            PF_SET_MAX_LDS_ONCE((range_dkv_kernel<D, MODE, false>), (lds_dkv<D, MODE, false>(MAX_RADIUS)));
            range_dkv_kernel<D, MODE, false><<<(unsigned)a.key_wgs, 256, (size_t)lds_dkv<D, MODE, false>(a.R), stream>>>(a);
            CHECK_LAUNCH();
        }
        if (const int rc = BOTH || !small ? launch_dq<D, MODE, 1>(a, row_wgs, stream) : launch_dq<D, MODE, BOTH ? 1 : 2>(a, row_wgs, stream)) return rc;
    }
    if (a.kv_split > 1) {
        range_kvjoin_kernel<D><<<(unsigned)(((long long)a.B * a.Hk * a.Lk + 3) / 4), 256, 0, stream>>>(a);
        CHECK_LAUNCH();
    }
    return 0;
}

}  // namespace

extern "C" long long pf_attention_ranges_workspace_bytes(const pf_attn_ranges_desc* d) {
    return check_ranges(d, false) ? -1 : fwd_bytes(d);
}

extern "C" long long pf_attention_ranges_bwd_workspace_bytes(const pf_attn_ranges_desc* d) {
    if (check_ranges(d, true)) return -1;
    const BwdSizes s = bwd_sizes(d);
    return s.all();
}

extern "C" int pf_attention_ranges_which(const pf_attn_ranges_desc* d) {
    return check_ranges(d, false) ? -1 : (d->H == 0 || few_rows(d) ? 2 : 1);
}

extern "C" int pf_attention_ranges_rows(const pf_attn_ranges_desc* d, int gradient) {
    if (check_ranges(d, gradient != 0)) return -1;
    if (gradient) return small_dq(d->D, d->Lq, d->H, d->B) ? 64 : 128;
    if (d->H == 0 || few_rows(d)) return 32;
    const bool small = small_fwd(d->D, d->Lq, d->H, d->B);
    const int nqt = row_groups(d->Lq, small), resident = d->D == 64 ? (small ? FWD_WAVES<64, 2> : FWD_WAVES<64, 1>) : (small ? FWD_WAVES<128, 2> : FWD_WAVES<128, 1>);
    const long long nwg = (long long)nqt * d->H * d->B;
    return (small ? 64 : 128) + (d->a_lo && nqt <= SORTED_TILES && nwg <= 0x7fffffffLL && sorted_launch((int)nwg, resident) ? 1 : 0);
}

extern "C" int pf_attention_ranges_bf16(const pf_attn_ranges_desc* d, hipStream_t stream) {
    if (const char* e = check_ranges(d, false)) return pf_set_err(e);
    if (!d->B || !d->H || !d->Lq) return 0;
    const long long need = fwd_bytes(d);
    if (need && (!d->workspace || ((uintptr_t)d->workspace & 15) || d->workspace_bytes < need))
        return pf_set_err("pf_attention_ranges_bf16: workspace missing, unaligned or too small");
    RArgs a = range_args(d);
    const bool few = few_rows(d);
    const int nqt = row_groups(d->Lq, small_fwd(d->D, d->Lq, d->H, d->B));
    const long long grid = few ? (long long)row_blocks(d) * d->Hkv * d->B * splits(d) : (long long)nqt * d->H * d->B;
    if (grid > MOST_WGS) return pf_set_err("pf_attention_ranges_bf16: 2^24 workgroups or more");
    if (const char* e = check_overlap(d, false)) return pf_set_err(e);
    a.nqt = nqt;
    a.nrb = row_blocks(d);
    a.nsplit = few ? splits(d) : 1;
    a.parts = (float*)d->workspace;
    switch ((d->D == 64 ? 0 : 8) + mode(d)) {
        case 0: return launch_fwd<64, 0>(a, few, stream);
        case 1: return launch_fwd<64, 1>(a, few, stream);
        case 2: return launch_fwd<64, 2>(a, few, stream);
        case 3: return launch_fwd<64, 3>(a, few, stream);
        case 5: return launch_fwd<64, 5>(a, few, stream);
        case 7: return launch_fwd<64, 7>(a, few, stream);
        case 8: return launch_fwd<128, 0>(a, few, stream);
        case 9: return launch_fwd<128, 1>(a, few, stream);
        case 10: return launch_fwd<128, 2>(a, few, stream);
        case 11: return launch_fwd<128, 3>(a, few, stream);
        case 13: return launch_fwd<128, 5>(a, few, stream);
        default: return launch_fwd<128, 7>(a, few, stream);
    }
}

extern "C" int pf_attention_ranges_bwd(const pf_attn_ranges_desc* d, hipStream_t stream) {
    if (const char* e = check_ranges(d, true)) return pf_set_err(e);
    const BwdSizes s = bwd_sizes(d);
    const long long need = s.all();
    if (need && (!d->workspace || ((uintptr_t)d->workspace & 15) || d->workspace_bytes < need))
        return pf_set_err("pf_attention_ranges_bwd: workspace missing, unaligned or too small");
    if (d->B > 65535 || d->H > 65535) return pf_set_err("pf_attention_ranges_bwd: more than 65535 batch entries or heads");
    if (!d->H) return 0;
    const int nqt = row_groups(d->Lq, small_dq(d->D, d->Lq, d->H, d->B));
    const long long key_wgs = (long long)((d->Lk + 127) / 128) * kv_splits(d) * d->Hkv * d->B;
    if ((long long)nqt * d->H * d->B + key_wgs + 7 > MOST_WGS || (d->Lq + 63) / 64 > MOST_WGS ||
        (long long)(d->Lq + 63) / 64 * (d->H / d->Hkv) > 0x7fffffffLL)
        return pf_set_err("pf_attention_ranges_bwd: 2^24 workgroups or more");
    if (const char* e = check_overlap(d, true)) return pf_set_err(e);
    RArgs a = range_args(d);
    char* w = (char*)d->workspace;
    a.stat = (float*)w;
    a.vis = (int*)(w += s.stat);
    a.tiles = (int*)(w += s.vis);
    a.dbias_parts = (float*)(w += s.tiles);
    a.kv_parts = (float*)(w += s.parts);
    a.kv_split = kv_splits(d);
    a.key_wgs = (int)key_wgs;
    a.key_pad = (a.key_wgs + 7) / 8 * 8;
    a.nqt = nqt;
    a.dbias = d->dbias;
    int rc = 0;
    if (d->B) switch ((d->D == 64 ? 0 : 8) + mode(d)) {
        case 0: rc = launch_bwd<64, 0>(a, stream); break;
        case 1: rc = launch_bwd<64, 1>(a, stream); break;
        case 2: rc = launch_bwd<64, 2>(a, stream); break;
        case 3: rc = launch_bwd<64, 3>(a, stream); break;
        case 5: rc = launch_bwd<64, 5>(a, stream); break;
        case 7: rc = launch_bwd<64, 7>(a, stream); break;
        case 8: rc = launch_bwd<128, 0>(a, stream); break;
        case 9: rc = launch_bwd<128, 1>(a, stream); break;
        case 10: rc = launch_bwd<128, 2>(a, stream); break;
        case 11: rc = launch_bwd<128, 3>(a, stream); break;
        case 13: rc = launch_bwd<128, 5>(a, stream); break;
        default: rc = launch_bwd<128, 7>(a, stream); break;
    }
    if (rc == 0 && d->dbias) {
        range_dbias_kernel<<<dim3((2 * a.R + 1 + 63) / 64, a.H), 256, 0, stream>>>(a);
        CHECK_LAUNCH();
    }
    return rc;
}
