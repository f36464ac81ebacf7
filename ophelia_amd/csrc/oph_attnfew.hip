// Cross attention for up to 4 rows of a key head (a decoder step): the forward of oph_seq_attn_forward without matrix instructions.
//
// Eight lanes share a key, a wave takes 8 keys at a time and a workgroup of 8 waves 64: every lane holds D/8 columns of its key's and
// value's row, so that both are read once, 128 bytes together, and a score costs D/8 multiplications and three lane exchanges.  Every
// group of eight lanes runs a softmax of its own over the keys it sees; the groups, waves and splits are joined at the end.  With so
// few rows a matrix instruction would work on 28 to 31 rows of padding, for fp32 at an eighth of the 16-bit rate.
#include "oph_attn.h"

#include <math.h>

namespace ophseq {

template <int CTRL> __device__ __forceinline__ float lanes(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
// sum over the 8 lanes of a group, in all of them: neighbours, pairs of two, then the mirrored other half
__device__ __forceinline__ float sum8(float x) {
    x += lanes<0xB1>(x);
    x += lanes<0x4E>(x);
    return x + lanes<0x141>(x);
}

template <class T, int DP, int ROWS>
__global__ __launch_bounds__(512) void attn_few(const AttnP p) {
    constexpr int PER = El<T>::PER16, E = DP / 8, NP = E / PER, NW = 8;      // columns and 16-byte pieces of a lane
    constexpr int U = NP * ROWS >= 16 ? 1 : NP * ROWS >= 8 ? 2 : 4;           // keys of a group at a time
    typedef T vec __attribute__((ext_vector_type(PER)));
    __shared__ float acc_of[NW][ROWS][DP];
    __shared__ float ml[NW][ROWS][2];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, group = lane >> 3, li = lane & 7;
    const int M = p.Tq * p.G;
    const int lin = on_xcd(p, blockIdx.x, p.B * p.Hk * p.nsplit), split = lin % p.nsplit;
    const Where w = where(p, lin / p.nsplit, 1);
    const float c = p.scale * LOG2E;
    const Span span = split_span(w.klen, 8, p.nsplit, split, w.qlen > 0);
    const int kbeg = span.beg, kend = span.end;

    float q[ROWS][E], acc[ROWS][E], m[ROWS], l[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        const T* row = row_ptr<T>(p, p.q, w, r, p.qs[0], p.qs[1], p.qs[2]);
        const bool ok = r < M && row_time(p, r) < w.qlen;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int d = (i * 8 + li) * PER;
            const vec x = __builtin_bit_cast(vec, load16(row + (d < p.D ? d : 0)));
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                q[r][i * PER + j] = ok && d < p.D ? (float)x[j] * c : 0.f;
                acc[r][i * PER + j] = 0.f;
            }
        }
        m[r] = -INFINITY;
        l[r] = 0.f;
    }

    const T* k = (const T*)p.k + w.b * p.ks[0] + w.hk * p.ks[2];
    const T* v = (const T*)p.v + w.b * p.vs[0] + w.hk * p.vs[2];
    for (int key0 = kbeg + wave * 8 + group; key0 - group < kend; key0 += U * NW * 8) {
        u32x4 kr[U][NP], vr[U][NP];
        bool ok[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int key = key0 + u * NW * 8;
            const int64_t at = min(key, kend - 1);
            ok[u] = key < kend;
            if (p.mask && ok[u]) ok[u] = p.mask[w.b * p.ms[0] + at * p.ms[1]] != 0;
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                const int d = (i * 8 + li) * PER;
                kr[u][i] = load16(k + at * p.ks[1] + (d < p.D ? d : 0));
                vr[u][i] = load16(v + at * p.vs[1] + (d < p.D ? d : 0));
            }
        }
        float s[ROWS][U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int r = 0; r < ROWS; ++r) s[r][u] = 0.f;
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                const vec x = __builtin_bit_cast(vec, (i * 8 + li) * PER < p.D ? kr[u][i] : u32x4{0, 0, 0, 0});
#pragma unroll
                for (int j = 0; j < PER; ++j)
#pragma unroll
                    for (int r = 0; r < ROWS; ++r) s[r][u] = fmaf(q[r][i * PER + j], (float)x[j], s[r][u]);
            }
        }
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            float top = m[r];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                s[r][u] = sum8(s[r][u]);
                s[r][u] = ok[u] ? s[r][u] : -INFINITY;
                top = fmaxf(top, s[r][u]);
            }
            const float base = top == -INFINITY ? 0.f : top, shrink = exp2_(m[r] - base);
            l[r] *= shrink;
            if (__any(shrink != 1.f))
#pragma unroll
                for (int e = 0; e < E; ++e) acc[r][e] *= shrink;
            m[r] = top;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                s[r][u] = exp2_(s[r][u] - base);
                l[r] += s[r][u];
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                const vec x = __builtin_bit_cast(vec, ok[u] ? vr[u][i] : u32x4{0, 0, 0, 0});
#pragma unroll
                for (int j = 0; j < PER; ++j)
#pragma unroll
                    for (int r = 0; r < ROWS; ++r) acc[r][i * PER + j] = fmaf(s[r][u], (float)x[j], acc[r][i * PER + j]);
            }
    }

    // the 8 groups of the wave: the common maximum, then sums in which every exchange halves what a lane holds
    const int b5 = lane >> 5 & 1, b4 = lane >> 4 & 1, b3 = lane >> 3 & 1;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        float top = m[r];
#pragma unroll
        for (int i = 8; i < 64; i <<= 1) top = fmaxf(top, __shfl_xor(top, i));
        const float weight = exp2_(m[r] - (top == -INFINITY ? 0.f : top));
        float sum = l[r] * weight;
#pragma unroll
        for (int i = 8; i < 64; i <<= 1) sum += __shfl_xor(sum, i);
        if (lane == 0) { ml[wave][r][0] = top; ml[wave][r][1] = sum; }
        float h1[E / 2], h2[E / 4], h3[E / 8];
#pragma unroll
        for (int e = 0; e < E / 2; ++e) {
            const float lo = acc[r][e] * weight, hi = acc[r][e + E / 2] * weight;
            h1[e] = (b5 ? hi : lo) + __shfl_xor(b5 ? lo : hi, 32);
        }
#pragma unroll
        for (int e = 0; e < E / 4; ++e) h2[e] = (b4 ? h1[e + E / 4] : h1[e]) + __shfl_xor(b4 ? h1[e] : h1[e + E / 4], 16);
#pragma unroll
        for (int e = 0; e < E / 8; ++e) {
            h3[e] = (b3 ? h2[e + E / 8] : h2[e]) + __shfl_xor(b3 ? h2[e] : h2[e + E / 8], 8);
            const int at = b5 * (E / 2) + b4 * (E / 4) + b3 * (E / 8) + e;    // which of the group's E columns
            acc_of[wave][r][(at / PER * 8 + li) * PER + at % PER] = h3[e];
        }
    }
    __syncthreads();
    // the 8 waves, in their order
    for (int i = tid; i < ROWS * DP; i += 512) {
        const int r = i / DP, d = i % DP;
        if (r >= M || d >= p.D) continue;
        float top = -INFINITY;
#pragma unroll
        for (int x = 0; x < NW; ++x) top = fmaxf(top, ml[x][r][0]);
        float sum = 0.f, o = 0.f;
#pragma unroll
        for (int x = 0; x < NW; ++x) {
            const float weight = exp2_(ml[x][r][0] - (top == -INFINITY ? 0.f : top));
            sum += ml[x][r][1] * weight;
            o += acc_of[x][r][d] * weight;
        }
        const int t = row_time(p, r), h = w.hk * p.G + r - t * p.G;
        if (p.nsplit == 1) {
            const bool live = t < w.qlen && sum != 0.f;
            ((T*)p.o0)[(((int64_t)w.b * p.Tq + t) * (p.Hk * p.G) + h) * p.D + d] = (T)(live ? o / sum : 0.f);
            if (d == 0) p.lse[((int64_t)w.b * (p.Hk * p.G) + h) * p.Tq + t] = live ? (top + log2f(sum)) * LN2 : -INFINITY;
        } else {
            const int64_t unit = (int64_t)(w.b * p.Hk + w.hk) * p.nsplit + split;
            p.part[(unit * unit_rows<T>() + r) * DP + d] = o;
            if (d == 0) { p.aux[(unit * unit_rows<T>() + r) * 2] = top; p.aux[(unit * unit_rows<T>() + r) * 2 + 1] = sum; }
        }
    }
}

template <class T, int DP> static int few_rows(const AttnP& p, dim3 grid, void* stream) {
    const int M = p.Tq * p.G;
    if (M == 1) return launch<AttnP>(attn_few<T, DP, 1>, grid, 512, p, 0, stream);
    if (M == 2) return launch<AttnP>(attn_few<T, DP, 2>, grid, 512, p, 0, stream);
    if constexpr (DP == 128) return launch<AttnP>(attn_few<T, DP, 4>, grid, 512, p, 0, stream);
    return fail(-4 /* OPH_ERR_UNSUPPORTED */, "attention: %d rows", M);      // not planned
}
template <class T> static int few_type(const AttnP& p, dim3 grid, void* stream) {
    if (p.D <= 64) return few_rows<T, 64>(p, grid, stream);
    if (p.D <= 128) return few_rows<T, 128>(p, grid, stream);
    return few_rows<T, 256>(p, grid, stream);
}
int attn_few_forward(const AttnP& p, int dtype, int64_t groups, void* stream) {
    const dim3 grid((unsigned)groups);
    if (dtype == OPH_SEQ_F32) return few_type<float>(p, grid, stream);
    if (dtype == OPH_SEQ_BF16) return few_type<bf16_t>(p, grid, stream);
    return few_type<f16_t>(p, grid, stream);
}

}  // namespace ophseq
