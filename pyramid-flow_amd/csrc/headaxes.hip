// RMSNorm of every query / key head and its rotation by several position axes, in one pass, and the gradient of both.
//
// For one head row x (D channels, D = 64 or 128), gains w, P rotated channel pairs and a scale s (queries only):
//     r = (mean x^2 + eps)^(-1/2),   n = x r w   (n = x without gains),   y = s R(theta) n,
//     theta_p = pos[axis(p)] freq(p),   R turns pair p = (2p, 2p+1), or (p, p + P) with `halves`; the rest passes through.
// Backward, with g = s R(-theta) dy:
//     dw = sum over rows of g x r,   dx = r (w g) - x r^3 / D sum_c(w g x)        (dx = g without gains).
// A position may be any float (fractions from interpolated grids, far positions of long streams): the angle is formed in 64
// bits, reduced to one turn there, and only then becomes a 32-bit fraction, so that 1e6 steps cost no digits.
//
// Bound: HBM.  Every row is read once and written once (backward: x and dy read, dx written); the angles of a token are
// computed once per wave and serve all of its heads, so neither an [L][D/2][2] table nor its upload exists.  One unit = one
// head row = D / 8 lanes of 16 bytes; a wave owns one token (or a slice of its heads when there are few tokens).
#include "common.h"
#include "pyflow_hip.h"
#include "rows_view.h"

int pf_set_err(const char* m);

namespace {

struct View { bf16_t* p; long long bs, ld, hs; };

struct HArgs {
    View q, k, qo, ko, dq, dk;          // forward: q, k -> qo, ko.  backward: (dq, dk, q, k) -> qo, ko
    const float* wq; const float* wk;
    const float* pos; long long pos_bs, pos_ld;
    const double* freq; const int* axis;
    int n_axes;
    int B, L, H, Hk, P, halves;
    float eps, q_scale;
    int chunks, per_chunk;              // wave-iterations of one token, split over `chunks` waves
    long long first_wave;               // forward: of this launch
    float* parts;                       // backward: [workgroup][2][D] partial gain gradients
};

// (cos, sin) of the pairs that this lane's 8 channels belong to: adjacent pairs -> 4, halves -> 8 (one per channel, the sine
// already carrying the sign of the channel's side).  Lane p computes pair p once (P <= 64), the others fetch it: the 64-bit
// product and the two series are half of the kernel's instructions when every lane does its own pairs (with the next row's load
// in flight and wave-uniform iterations 131 -> 98 us for 2 x 15488 tokens of 60 heads, 4.8 TB/s).
PF_DEVICE void lane_angles(const HArgs& p, int b, int tok, int sub, float* c, float* s) {
    const int lane = threadIdx.x & 63;
    float cs = 1.f, sn = 0.f;
    if (lane < p.P) {
        const float pos = p.pos[b * p.pos_bs + tok * p.pos_ld + min(max(p.axis[lane], 0), p.n_axes - 1)];
        const double turns = (double)pos * p.freq[lane] * 0.15915494309189533577;                  // / 2 pi
        sincospif(2.f * (float)(turns - rint(turns)), &sn, &cs);
    }
    if (p.halves) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int ch = sub * 8 + i, pr = ch < p.P ? ch : min(ch - p.P, 63);
            c[i] = __shfl(cs, pr);
            s[i] = __shfl(sn, pr);
            s[i] = ch < p.P ? -s[i] : s[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int pr = min(sub * 4 + i, 63);
            c[i] = __shfl(cs, pr);
            s[i] = __shfl(sn, pr);
        }
    }
}

// v <- R(+-theta) v on the lane's 8 channels (dir = -1: the inverse rotation).  halves: the partner channel of (lane, e) sits
// at the same e of the lane P / 8 further on (channels < P) or back
PF_DEVICE void rotate8(const HArgs& p, float* v, const float* c, const float* s, int sub, float dir) {
    if (p.halves) {
        const int shift = p.P >> 3;
        const int lane = threadIdx.x & 63;
        const int other = sub < shift ? lane + shift : (sub < 2 * shift ? lane - shift : lane);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float w = __shfl(v[e], other);
            if (sub < 2 * shift) v[e] = __builtin_fmaf(v[e], c[e], w * (dir * s[e]));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (sub * 4 + i >= p.P) continue;                   // passes through as it is, an infinity too
            const float x0 = v[2 * i], x1 = v[2 * i + 1], sn = dir * s[i];
            v[2 * i] = __builtin_fmaf(x0, c[i], -(x1 * sn));
            v[2 * i + 1] = __builtin_fmaf(x0, sn, x1 * c[i]);
        }
    }
}

template <int LPU>
PF_DEVICE float unit_sum(float x) {
#pragma unroll
    for (int o = 1; o < LPU; o <<= 1) x += __shfl_xor(x, o);
    return x;
}

// Wave-iterations of a token: the query heads in groups of UPW units, then the key heads (a wave-iteration is all queries or
// all keys, so gains and strides are wave-uniform).
struct Unit { bool isq, on; long long h; };
template <int UPW>
PF_DEVICE Unit unit_of(const HArgs& p, int it, int slot) {
    const int iq = (p.H + UPW - 1) / UPW;
    const bool isq = it < iq;
    const int h = (isq ? it : it - iq) * UPW + slot;
    return {isq, h < (isq ? p.H : p.Hk), h};
}
PF_DEVICE u32x4_t load_unit(const View& v, const Unit& u, int b, int tok, int sub) {
    u32x4_t r = {0u, 0u, 0u, 0u};
    if (u.on) r = *(const u32x4_t*)(v.p + b * v.bs + tok * v.ld + u.h * v.hs + sub * 8);
    return r;
}

template <int D>
__global__ __launch_bounds__(256) void heads_fwd_kernel(const HArgs p) {
    constexpr int LPU = D / 8, UPW = 64 / LPU;
    const int lane = threadIdx.x & 63, sub = lane % LPU;
    const long long wave = p.first_wave + (long long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long long tokb = wave / p.chunks;
    if (tokb >= (long long)p.B * p.L) return;
    const int chunk = (int)(wave - tokb * p.chunks);
    const int b = (int)(tokb / p.L), tok = (int)(tokb - (long long)b * p.L);
    const int its = (p.H + UPW - 1) / UPW + (p.Hk + UPW - 1) / UPW;
    int it = chunk * p.per_chunk;
    const int end = min(its, it + p.per_chunk);
    Unit u = unit_of<UPW>(p, it, lane / LPU);
    u32x4_t raw = load_unit(u.isq ? p.q : p.k, u, b, tok, sub);         // in flight while the angles are computed
    float c[8], s[8], wq[8], wk[8];
    lane_angles(p, b, tok, sub, c, s);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        wq[e] = (p.wq ? p.wq[sub * 8 + e] : 1.f) * p.q_scale;
        wk[e] = p.wk ? p.wk[sub * 8 + e] : 1.f;
    }
    while (it < end) {
        const Unit cur = u;
        float v[8];
        unpack8(raw, v);
        if (++it < end) {
            u = unit_of<UPW>(p, it, lane / LPU);
            raw = load_unit(u.isq ? p.q : p.k, u, b, tok, sub);
        }
        float r = 1.f;
        if (cur.isq ? p.wq != nullptr : p.wk != nullptr) {
            float ss = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) ss = __builtin_fmaf(v[e], v[e], ss);
            r = rsqrtf(__builtin_fmaf(unit_sum<LPU>(ss), 1.f / D, p.eps));
        }
        if (cur.isq) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] *= r * wq[e];
        } else if (p.wk) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] *= r * wk[e];
        }
        rotate8(p, v, c, s, sub, 1.f);
        const View& out = cur.isq ? p.qo : p.ko;
        if (cur.on) *(u32x4_t*)(out.p + b * out.bs + tok * out.ld + cur.h * out.hs + sub * 8) = pack8(v);
    }
}

// Gain gradients: every lane keeps the sums of its 8 channels over the tokens of its wave; units of a wave, waves of a
// workgroup and workgroups are then added in a fixed order (the same bits every time; no atomics).  Registers are cut for four waves
// per SIMD: 7808 tokens of 60 heads take 47 us with the sums' launch (180 MB: 3.8 TB/s), 56 us with three.
template <int D>
__global__ __launch_bounds__(256, 4) void heads_bwd_kernel(const HArgs p) {
    constexpr int LPU = D / 8, UPW = 64 / LPU;
    __shared__ float red[4][2][D];
    const int lane = threadIdx.x & 63, sub = lane % LPU, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    float wq[8], wk[8], aq[8], ak[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        wq[e] = p.wq ? p.wq[sub * 8 + e] : 1.f;
        wk[e] = p.wk ? p.wk[sub * 8 + e] : 1.f;
        aq[e] = ak[e] = 0.f;
    }
    const int its = (p.H + UPW - 1) / UPW + (p.Hk + UPW - 1) / UPW;
    const long long waves = (long long)p.B * p.L * p.chunks;
    for (long long wave = (long long)blockIdx.x * 4 + wid; wave < waves; wave += (long long)gridDim.x * 4) {
        const long long tokb = wave / p.chunks;
        const int chunk = (int)(wave - tokb * p.chunks);
        const int b = (int)(tokb / p.L), tok = (int)(tokb - (long long)b * p.L);
        int it = chunk * p.per_chunk;
        const int end = min(its, it + p.per_chunk);
        Unit u = unit_of<UPW>(p, it, lane / LPU);
        auto norm_of = [&](const Unit& n) { return n.isq ? p.wq != nullptr : p.wk != nullptr; };
        u32x4_t rg = load_unit(u.isq ? p.dq : p.dk, u, b, tok, sub), rx = {0u, 0u, 0u, 0u};
        if (norm_of(u)) rx = load_unit(u.isq ? p.q : p.k, u, b, tok, sub);
        float c[8], s[8];
        lane_angles(p, b, tok, sub, c, s);
        while (it < end) {
            const Unit cur = u;
            float g[8], x[8];
            unpack8(rg, g);
            unpack8(rx, x);
            if (++it < end) {
                u = unit_of<UPW>(p, it, lane / LPU);
                rg = load_unit(u.isq ? p.dq : p.dk, u, b, tok, sub);
                if (norm_of(u)) rx = load_unit(u.isq ? p.q : p.k, u, b, tok, sub);
            }
            if (cur.isq) {
#pragma unroll
                for (int e = 0; e < 8; ++e) g[e] *= p.q_scale;
            }
            rotate8(p, g, c, s, sub, -1.f);
            if (norm_of(cur)) {
                float ss = 0.f, st = 0.f, wg[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    wg[e] = (cur.isq ? wq[e] : wk[e]) * g[e];
                    ss = __builtin_fmaf(x[e], x[e], ss);
                    st = __builtin_fmaf(wg[e], x[e], st);
                }
                const float r = rsqrtf(__builtin_fmaf(unit_sum<LPU>(ss), 1.f / D, p.eps));
                const float k = unit_sum<LPU>(st) * (1.f / D) * r * r * r;
                if (cur.on) {                                          // a row of zeros and eps 0 would leave 0 x inf
                    if (cur.isq) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) aq[e] = __builtin_fmaf(g[e], x[e] * r, aq[e]);
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e) ak[e] = __builtin_fmaf(g[e], x[e] * r, ak[e]);
                    }
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) g[e] = __builtin_fmaf(r, wg[e], -(x[e] * k));
            }
            const View& out = cur.isq ? p.qo : p.ko;
            if (cur.on) *(u32x4_t*)(out.p + b * out.bs + tok * out.ld + cur.h * out.hs + sub * 8) = pack8(g);
        }
    }
    if (!p.parts) return;                                       // uniform over the launch
#pragma unroll
    for (int e = 0; e < 8; ++e) {
#pragma unroll
        for (int o = LPU; o < 64; o <<= 1) {
            aq[e] += __shfl_xor(aq[e], o);
            ak[e] += __shfl_xor(ak[e], o);
        }
        if (lane < LPU) {
            red[wid][0][sub * 8 + e] = aq[e];
            red[wid][1][sub * 8 + e] = ak[e];
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * D; i += 256) {
        const float* r = &red[0][0][0] + i;
        p.parts[(long long)blockIdx.x * 2 * D + i] = (r[0] + r[2 * D]) + (r[4 * D] + r[6 * D]);
    }
}

// dw[i] = sum over workgroups of parts[wg][i], i < 2 D (queries, then keys): 32 columns per workgroup, 32 row groups (with 8 of
// them the launch took 32 us of loads in a row, more than half of the gradient kernel itself)
__global__ __launch_bounds__(1024) void heads_dw_kernel(const float* parts, float* dwq, float* dwk, int nwg, int D) {
    __shared__ float red[32][33];
    const int x = threadIdx.x & 31, grp = threadIdx.x >> 5, col = blockIdx.x * 32 + x;
    float a = 0.f;
#pragma unroll 8
    for (int w = grp; w < nwg; w += 32) a += parts[(long long)w * 2 * D + col];
    red[grp][x] = a;
    __syncthreads();
    if (grp == 0) {
        float t = 0.f;
#pragma unroll
        for (int g = 0; g < 32; ++g) t += red[g][x];
        if (col < D) {
            if (dwq) dwq[col] = t;
        } else if (dwk) {
            dwk[col - D] = t;
        }
    }
}

constexpr int BWD_GRID = 1024;             // four workgroups per compute unit, all resident

int bwd_grid(long long waves) { return (int)((waves + 3) / 4 < BWD_GRID ? (waves + 3) / 4 : BWD_GRID); }

// wave-iterations of one token over `chunks` waves: one wave per token amortises the angles over all of its heads; with few
// tokens every iteration gets a wave of its own (the call is latency then, not bandwidth)
void split_heads(const pf_heads_desc* d, int* chunks, int* per_chunk) {
    const int upw = 64 / (d->D / 8), its = (d->H + upw - 1) / upw + (d->Hkv + upw - 1) / upw;
    *per_chunk = (long long)d->B * d->L * its <= 8192 ? 1 : its;
    *chunks = (its + *per_chunk - 1) / *per_chunk;
}

bool bad_view(const pf_rows_view& v) {
    return !v.p || ((uintptr_t)v.p & 15) || v.batch < 0 || v.row < 0 || v.head < 0 || ((v.batch | v.row | v.head) & 7);
}

View view(const pf_rows_view& v) { return {(bf16_t*)v.p, v.batch, v.row, v.head}; }

const char* check_heads(const pf_heads_desc* d, bool grad) {
    if (!d) return "pf_qk_norm_rope_axes: null descriptor";
    if (d->D != 64 && d->D != 128) return "pf_qk_norm_rope_axes: head_dim must be 64 or 128";
    if (d->B < 0 || d->L < 0 || d->H < 0 || d->Hkv < 0) return "pf_qk_norm_rope_axes: negative size";
    if (d->B == 0 || d->L == 0 || d->H + d->Hkv == 0) return nullptr;
    if ((long long)d->B * d->L > 0x7fffffffLL) return "pf_qk_norm_rope_axes: more than 2^31 - 1 tokens";
    if (d->H + d->Hkv > 65536) return "pf_qk_norm_rope_axes: too many heads";
    if (d->n_pairs < 0 || 2 * d->n_pairs > d->D) return "pf_qk_norm_rope_axes: more rotated channels than the head has";
    if (d->halves && d->n_pairs % 8) return "pf_qk_norm_rope_axes: half pairs need a multiple of 8 pairs";
    if (d->n_pairs && (!d->pos || !d->freq || !d->axis)) return "pf_qk_norm_rope_axes: null position / frequency / axis";
    if (d->n_pairs && d->n_axes < 1) return "pf_qk_norm_rope_axes: no position axis";
    if (d->pos_row < 0 || d->pos_batch < 0) return "pf_qk_norm_rope_axes: negative position stride";
    if ((d->H && (bad_view(d->Q) || bad_view(d->Qo))) || (d->Hkv && (bad_view(d->K) || bad_view(d->Ko))))
        return "pf_qk_norm_rope_axes: rows must be 16-byte aligned with strides that are multiples of 8 elements";
    if (grad && ((d->H && bad_view(d->dQ)) || (d->Hkv && bad_view(d->dK))))
        return "pf_qk_norm_rope_axes_bwd: gradient rows must be 16-byte aligned with strides that are multiples of 8 elements";
    return nullptr;
}

// an output may be the input (gradient: or the gradient) of its own heads, element for element, and shares nothing else
const char* check_overlap(const pf_heads_desc* d, bool grad) {
    const int B = d->B, L = d->L, H[2] = {d->H, d->Hkv}, D = d->D;
    const pf_rows_view* const out[2] = {&d->Qo, &d->Ko};
    const pf_rows_view* const in[2][2] = {{&d->Q, &d->dQ}, {&d->K, &d->dK}};
    for (int o = 0; o < 2; ++o) {
        if (rows_folded(*out[o], B, L, H[o], D)) return "pf_qk_norm_rope_axes: an output overlaps itself";
        for (int i = 0; i < 2; ++i)
            for (int n = 0; n < (grad ? 2 : 1); ++n)
                if (!(i == o && rows_same(*out[o], *in[i][n], B, L, H[i])) && rows_share(*out[o], B, L, H[o], *in[i][n], B, L, H[i], D))
                    return "pf_qk_norm_rope_axes: an output overlaps an input and is not it";
    }
    return rows_share(d->Qo, B, L, H[0], d->Ko, B, L, H[1], D) ? "pf_qk_norm_rope_axes: the outputs overlap" : nullptr;
}

HArgs heads_args(const pf_heads_desc* d) {
    HArgs a{};
    a.q = view(d->Q); a.k = view(d->K); a.qo = view(d->Qo); a.ko = view(d->Ko); a.dq = view(d->dQ); a.dk = view(d->dK);
    a.wq = d->wq; a.wk = d->wk;
    a.pos = d->pos; a.pos_bs = d->pos_batch; a.pos_ld = d->pos_row;
    a.freq = d->freq; a.axis = d->axis; a.n_axes = d->n_axes;
    a.B = d->B; a.L = d->L; a.H = d->H; a.Hk = d->Hkv; a.P = d->n_pairs; a.halves = d->halves;
    a.eps = d->eps; a.q_scale = d->q_scale;
    split_heads(d, &a.chunks, &a.per_chunk);
    return a;
}

}  // namespace

#define CHECK_LAUNCH()                                              \
    do {                                                            \
        hipError_t e_ = hipGetLastError();                          \
        if (e_ != hipSuccess) return pf_set_err(hipGetErrorString(e_)); \
    } while (0)

extern "C" int pf_qk_norm_rope_axes(const pf_heads_desc* d, hipStream_t stream) {
    if (const char* e = check_heads(d, false)) return pf_set_err(e);
    if (d->B == 0 || d->L == 0 || d->H + d->Hkv == 0) return 0;
    if (const char* e = check_overlap(d, false)) return pf_set_err(e);
    HArgs a = heads_args(d);
    constexpr long long MOST = 1 << 23;                         // workgroups of a launch: 2^32 threads wrap around without an error
    for (long long left = ((long long)d->B * d->L * a.chunks + 3) / 4; left > 0; left -= MOST, a.first_wave += 4 * MOST) {
        const unsigned grid = (unsigned)(left < MOST ? left : MOST);
        if (d->D == 64) heads_fwd_kernel<64><<<grid, 256, 0, stream>>>(a);
        else heads_fwd_kernel<128><<<grid, 256, 0, stream>>>(a);
        CHECK_LAUNCH();
    }
    return 0;
}

extern "C" long long pf_qk_norm_rope_axes_bwd_workspace_bytes(const pf_heads_desc* d) {
    if (check_heads(d, true)) return -1;
    if (d->B == 0 || d->L == 0 || d->H + d->Hkv == 0) return 0;
    int chunks, per;
    split_heads(d, &chunks, &per);
    return (long long)bwd_grid((long long)d->B * d->L * chunks) * 2 * d->D * 4;
}

extern "C" int pf_qk_norm_rope_axes_bwd(const pf_heads_desc* d, float* dwq, float* dwk, void* workspace, long long workspace_bytes,
                                        hipStream_t stream) {
    if (const char* e = check_heads(d, true)) return pf_set_err(e);
    if ((dwq && !d->wq) || (dwk && !d->wk)) return pf_set_err("pf_qk_norm_rope_axes_bwd: a gain gradient without its gains");
    const bool gains = dwq || dwk, empty = d->B == 0 || d->L == 0 || d->H + d->Hkv == 0;
    if (gains && !empty && (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < pf_qk_norm_rope_axes_bwd_workspace_bytes(d)))
        return pf_set_err("pf_qk_norm_rope_axes_bwd: workspace missing, unaligned or too small");
    if (const char* e = check_overlap(d, true)) return pf_set_err(e);
    HArgs a = heads_args(d);
    int grid = 0;
    if (!empty) {
        grid = bwd_grid((long long)d->B * d->L * a.chunks);
        a.parts = gains ? (float*)workspace : nullptr;
        if (d->D == 64) heads_bwd_kernel<64><<<grid, 256, 0, stream>>>(a);
        else heads_bwd_kernel<128><<<grid, 256, 0, stream>>>(a);
        CHECK_LAUNCH();
    }
    if (gains) {                                                // no tokens: the sums are zero
        heads_dw_kernel<<<2 * d->D / 32, 1024, 0, stream>>>((const float*)workspace, dwq, dwk, grid, d->D);
        CHECK_LAUNCH();
    }
    return 0;
}
