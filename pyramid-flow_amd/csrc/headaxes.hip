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
    float* parts;                       // backward: [workgroup][2][D] partial gain gradients
};

// (cos, sin) of the pairs that this lane's 8 channels belong to: adjacent pairs -> 4, halves -> 8 (one per channel, the sine
// already carrying the sign of the channel's side); pairs behind P are the identity
template <int D>
PF_DEVICE void lane_angles(const HArgs& p, int b, int tok, int sub, float* c, float* s) {
    const float* pos = p.pos + b * p.pos_bs + tok * p.pos_ld;
    const int n = p.halves ? 8 : 4;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        c[i] = 1.f;
        s[i] = 0.f;
        if (i >= n) continue;
        int pr = sub * n + i;
        float sign = 1.f;
        if (p.halves) {
            if (pr >= 2 * p.P) continue;
            sign = pr < p.P ? -1.f : 1.f;
            pr = pr < p.P ? pr : pr - p.P;
        } else if (pr >= p.P) {
            continue;
        }
        const double turns = (double)pos[min(max(p.axis[pr], 0), p.n_axes - 1)] * p.freq[pr] * 0.15915494309189533577;      // / 2 pi
        const float f = (float)(turns - rint(turns));
        float sn, cs;
        sincospif(2.f * f, &sn, &cs);
        c[i] = cs;
        s[i] = sign * sn;
    }
}

// v <- R(+-theta) v on the lane's 8 channels (dir = -1: the inverse rotation).  halves: the partner channel of (lane, e) sits
// at the same e of the lane P / 8 further on (channels < P) or back
template <int D>
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

template <int D>
__global__ __launch_bounds__(256) void heads_fwd_kernel(const HArgs p) {
    constexpr int LPU = D / 8, UPW = 64 / LPU;
    const int lane = threadIdx.x & 63, sub = lane % LPU;
    const long long wave = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const long long tokb = wave / p.chunks;
    if (tokb >= (long long)p.B * p.L) return;
    const int chunk = (int)(wave - tokb * p.chunks);
    const int b = (int)(tokb / p.L), tok = (int)(tokb - (long long)b * p.L);
    float c[8], s[8], wq[8], wk[8];
    lane_angles<D>(p, b, tok, sub, c, s);
    if (p.wq) {
#pragma unroll
        for (int e = 0; e < 8; ++e) wq[e] = p.wq[sub * 8 + e];
    }
    if (p.wk) {
#pragma unroll
        for (int e = 0; e < 8; ++e) wk[e] = p.wk[sub * 8 + e];
    }
    const int total = p.H + p.Hk;
    const int u0 = chunk * p.per_chunk * UPW, u1 = min(total, u0 + p.per_chunk * UPW);
    for (int u = u0; u < u1; u += UPW) {
        const int h = u + lane / LPU;
        const bool on = h < u1, isq = h < p.H;
        const View& in = isq ? p.q : p.k;
        const View& out = isq ? p.qo : p.ko;
        const int hh = isq ? h : h - p.H;
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (on) unpack8(*(const u32x4_t*)(in.p + b * in.bs + tok * in.ld + hh * in.hs + sub * 8), v);
        const bool norm = isq ? p.wq != nullptr : p.wk != nullptr;
        if (p.wq || p.wk) {                                     // uniform: the reduction runs on all lanes
            float ss = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) ss = __builtin_fmaf(v[e], v[e], ss);
            const float r = rsqrtf(__builtin_fmaf(unit_sum<LPU>(ss), 1.f / D, p.eps));
            if (norm) {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = v[e] * r * (isq ? wq[e] : wk[e]);
            }
        }
        rotate8<D>(p, v, c, s, sub, 1.f);
        if (on) {
            const float f = isq ? p.q_scale : 1.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] *= f;
            *(u32x4_t*)(out.p + b * out.bs + tok * out.ld + hh * out.hs + sub * 8) = pack8(v);
        }
    }
}

// Gain gradients: every lane keeps the sums of its 8 channels over the tokens of its wave; units of a wave, waves of a
// workgroup and workgroups are then added in a fixed order (the same bits every time; no atomics).
template <int D>
__global__ __launch_bounds__(256) void heads_bwd_kernel(const HArgs p) {
    constexpr int LPU = D / 8, UPW = 64 / LPU;
    __shared__ float red[4][2][D];
    const int lane = threadIdx.x & 63, sub = lane % LPU, wid = threadIdx.x >> 6;
    float wq[8], wk[8], aq[8], ak[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        wq[e] = p.wq ? p.wq[sub * 8 + e] : 1.f;
        wk[e] = p.wk ? p.wk[sub * 8 + e] : 1.f;
        aq[e] = ak[e] = 0.f;
    }
    const int total = p.H + p.Hk;
    const long long waves = (long long)p.B * p.L * p.chunks;
    for (long long wave = (long long)blockIdx.x * 4 + wid; wave < waves; wave += (long long)gridDim.x * 4) {
        const long long tokb = wave / p.chunks;
        const int chunk = (int)(wave - tokb * p.chunks);
        const int b = (int)(tokb / p.L), tok = (int)(tokb - (long long)b * p.L);
        float c[8], s[8];
        lane_angles<D>(p, b, tok, sub, c, s);
        const int u0 = chunk * p.per_chunk * UPW, u1 = min(total, u0 + p.per_chunk * UPW);
        for (int u = u0; u < u1; u += UPW) {
            const int h = u + lane / LPU;
            const bool on = h < u1, isq = h < p.H;
            const View& in = isq ? p.q : p.k;
            const View& dy = isq ? p.dq : p.dk;
            const View& out = isq ? p.qo : p.ko;
            const int hh = isq ? h : h - p.H;
            const bool norm = isq ? p.wq != nullptr : p.wk != nullptr;
            float g[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            if (on) {
                unpack8(*(const u32x4_t*)(dy.p + b * dy.bs + tok * dy.ld + hh * dy.hs + sub * 8), g);
                if (norm) unpack8(*(const u32x4_t*)(in.p + b * in.bs + tok * in.ld + hh * in.hs + sub * 8), x);
                const float f = isq ? p.q_scale : 1.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) g[e] *= f;
            }
            rotate8<D>(p, g, c, s, sub, -1.f);
            if (p.wq || p.wk) {
                float ss = 0.f, st = 0.f, w[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    w[e] = isq ? wq[e] : wk[e];
                    ss = __builtin_fmaf(x[e], x[e], ss);
                    st = __builtin_fmaf(w[e] * g[e], x[e], st);
                }
                const float r = rsqrtf(__builtin_fmaf(unit_sum<LPU>(ss), 1.f / D, p.eps));
                const float k = unit_sum<LPU>(st) * (1.f / D) * r * r * r;
                if (on && norm) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float gx = g[e] * x[e] * r;
                        aq[e] += isq ? gx : 0.f;
                        ak[e] += isq ? 0.f : gx;
                        g[e] = __builtin_fmaf(r, w[e] * g[e], -(x[e] * k));
                    }
                }
            }
            if (on) *(u32x4_t*)(out.p + b * out.bs + tok * out.ld + hh * out.hs + sub * 8) = pack8(g);
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

// dw[i] = sum over workgroups of parts[wg][i], i < 2 D (queries, then keys): 32 columns per workgroup, 8 row groups
__global__ __launch_bounds__(256) void heads_dw_kernel(const float* parts, float* dwq, float* dwk, int nwg, int D) {
    __shared__ float red[8][32];
    const int col = blockIdx.x * 32 + (threadIdx.x & 31), grp = threadIdx.x >> 5;
    float a = 0.f;
    for (int w = grp; w < nwg; w += 8) a += parts[(long long)w * 2 * D + col];
    red[grp][threadIdx.x & 31] = a;
    __syncthreads();
    if (grp == 0) {
        float t = 0.f;
#pragma unroll
        for (int g = 0; g < 8; ++g) t += red[g][threadIdx.x];
        if (col < D) {
            if (dwq) dwq[col] = t;
        } else if (dwk) {
            dwk[col - D] = t;
        }
    }
}

constexpr int BWD_GRID = 1024;

int bwd_grid(long long waves) { return (int)((waves + 3) / 4 < BWD_GRID ? (waves + 3) / 4 : BWD_GRID); }

// wave-iterations of one token over `chunks` waves: one wave per token amortises the angles over all of its heads; with few
// tokens every iteration gets a wave of its own (the call is latency then, not bandwidth)
void split_heads(const pf_heads_desc* d, int* chunks, int* per_chunk) {
    const int upw = 64 / (d->D / 8), its = (d->H + d->Hkv + upw - 1) / upw;
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
    const HArgs a = heads_args(d);
    const unsigned grid = (unsigned)(((long long)d->B * d->L * a.chunks + 3) / 4);
    if (d->D == 64) heads_fwd_kernel<64><<<grid, 256, 0, stream>>>(a);
    else heads_fwd_kernel<128><<<grid, 256, 0, stream>>>(a);
    CHECK_LAUNCH();
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
        heads_dw_kernel<<<2 * d->D / 32, 256, 0, stream>>>((const float*)workspace, dwq, dwk, grid, d->D);
        CHECK_LAUNCH();
    }
    return 0;
}
