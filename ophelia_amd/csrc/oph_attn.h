// What the forward and the gradient kernels of cross attention share.
//
// Rows.  The G = Hq/Hk query heads that read one key head are folded into the row axis: row r of (sequence b, key head hk) is query
// t = r / G of head hk*G + r % G.  Keys and values are then read once for the whole group, a single token of a grouped model fills G
// rows of a tile, and the sum over the group in dk, dv is part of the contraction.
//
// Layout of a 32x32 product: lane l holds column l % 32 and the 16 rows 8g + 4(l/32) + i (g, i = 0..3) in register 4g + i.  Scores are
// formed with the axis that the next product contracts as ROWS; registers 8s..8s+7 of a lane then are, without any exchange
// between lanes, its 8 elements of the operand of the next product's step s, if the other operand takes its elements in the same
// order: element j of lane half e is row 16s + 8(j/4) + 4e + j%4.  trans_frag() reads them so from a row-major tile in LDS.
#pragma once
#include "oph_seq.h"
#include "oph_split.h"

#pragma GCC visibility push(hidden)
namespace ophseq {

struct AttnP {                       // at most 256 bytes: a larger block of arguments costs microseconds per launch
    const void *q, *k, *v, *out, *dout;
    void *o0, *o1;                   // forward: out | gradient: dq, or dk and dv
    float *lse, *aux, *part;         // aux: forward's maxima and sums of the splits | gradient's delta
    const int *q_lens, *k_lens;
    const uint8_t* mask;
    int64_t qs[3], ks[3], vs[3], ds[3], ms[2];
    int B, Tq, Tk, Hk, G, D;
    unsigned magic;                  // r / G = umulhi(r, magic) for G > 1
    float scale;
    int nsplit, chunk;
};
static_assert(sizeof(AttnP) <= 256, "AttnP");

struct Where { int b, hk, tile, qlen, klen; };

__device__ __forceinline__ int clampi(int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; }

// Workgroups go round robin over the 8 XCDs.  The list of (sequence, key head, tile, split) is dealt out in runs of `chunk`: long runs keep the
// tiles that read the same keys on one L2, short ones spread sequences of different lengths over the machine (run_of()).
__device__ __forceinline__ int on_xcd(const AttnP& p, int id, int n) {
    if (p.chunk <= 1) return id;
    const int round = 8 * p.chunk, x = id & 7, s = id >> 3, c = s / p.chunk;
    return id < n / round * round ? (c * 8 + x) * p.chunk + s - c * p.chunk : id;
}

__device__ __forceinline__ Where where(const AttnP& p, int lin, int tiles) {
    Where w;
    const int bh = lin / tiles;
    w.tile = lin - bh * tiles;
    w.b = bh / p.Hk;
    w.hk = bh - w.b * p.Hk;
    w.qlen = p.q_lens ? clampi(p.q_lens[w.b], 0, p.Tq) : p.Tq;
    w.klen = p.k_lens ? clampi(p.k_lens[w.b], 0, p.Tk) : p.Tk;
    return w;
}

__device__ __forceinline__ int row_time(const AttnP& p, int r) { return p.G == 1 ? r : (int)__umulhi((unsigned)r, p.magic); }

// pointer to the D elements of row r of q (or of anything with q's strides); r is clamped into the existing rows
template <class T>
__device__ __forceinline__ const T* row_ptr(const AttnP& p, const void* base, const Where& w, int r, int64_t sb, int64_t st, int64_t sh) {
    r = clampi(r, 0, p.Tq * p.G - 1);
    const int t = row_time(p, r), g = r - t * p.G;
    return (const T*)base + w.b * sb + t * st + (int64_t)(w.hk * p.G + g) * sh;
}

// Which of the keys key0 + lane may be attended, in two steps: the mask's byte is loaded with (before) the keys it belongs to, and only
// asked for when they are used.  Nothing is read where no key before kend is left.  bit i of key_bits(): key key0 + i (i < 64).
__device__ __forceinline__ uint8_t key_byte(const AttnP& p, const Where& w, int key0, int kend, int lane) {
    const int at = flag_index(key0, lane, kend);
    return p.mask && at >= 0 ? p.mask[w.b * p.ms[0] + at * p.ms[1]] : 1;
}
__device__ __forceinline__ uint64_t key_bits(uint8_t byte, int key0, int kend, int lane) { return __ballot(byte != 0 && key0 + lane < kend); }

// the operand pieces of one row: 8 elements of every 16, by lane half; zeros where !ok and beyond D
template <class T, int DP>
__device__ __forceinline__ void row_frags(frag_t<T> (&f)[DP / 16], const T* row, int D, bool ok, int half) {
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
        const int d = s * 16 + half * 8;
        const bool in = ok && d < D;
        const T* at = row + (d < D ? d : 0);
        u32x4 lo = load16(at), hi = u32x4{0, 0, 0, 0};
        if (sizeof(T) == 4) hi = load16(at + 4);
        lo = in ? lo : u32x4{0, 0, 0, 0};
        hi = in ? hi : u32x4{0, 0, 0, 0};
        f[s] = bits_to_frag<T>(lo, hi);
    }
}

// A tile of rows in LDS, row-major.  The padding spreads the rows' pieces over the banks, for reads along a row (16 bytes of 32 rows)
// and across (4 rows x 32 bytes, or 2 x 128): of 16, 32, 48 and 64 bytes 48 leaves the fewest conflicts (a third of 16's and 64's; 4 x 16 heads
// of 4096 x 4096 x 128 bf16: 610, 577, 571 and 605 us).
template <class T, int DP> struct Tile {
    static constexpr int STRIDE = DP * (int)sizeof(T) + 48;
    static constexpr int bytes(int rows) { return rows * STRIDE; }
};

// element s of the row operand of rows row0..row0+31
template <class T, int DP> __device__ __forceinline__ frag_t<T> row_frag(const char* tile, int row0, int s, int lane) {
    const char* at = tile + (row0 + (lane & 31)) * Tile<T, DP>::STRIDE + (s * 16 + (lane >> 5) * 8) * (int)sizeof(T);
    const u32x4 lo = *(const u32x4*)at;
    u32x4 hi = {0, 0, 0, 0};
    if (sizeof(T) == 4) hi = *(const u32x4*)(at + 16);
    return bits_to_frag<T>(lo, hi);
}

// operand with the tile's columns d0..d0+31 as its rows (or columns) and the tile's rows row0..row0+15 as the contracted axis, in the
// order above.  16 bits: a group of 16 lanes hands in 4 rows of 16 columns and gets them back column by column.
template <class T, int DP> __device__ __forceinline__ frag_t<T> trans_frag(const char* tile, int row0, int d0, int lane) {
    constexpr int ST = Tile<T, DP>::STRIDE;
    if constexpr (sizeof(T) == 4) {
        frag_t<T> f;
        const char* at = tile + (row0 + 4 * (lane >> 5)) * ST + (d0 + (lane & 31)) * 4;
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = *(const float*)(at + (8 * (j / 4) + j % 4) * ST);
        return f;
    } else {
        const char* at = tile + (row0 + 4 * (lane >> 5) + ((lane & 15) >> 2)) * ST + (d0 + 16 * ((lane >> 4) & 1) + 4 * (lane & 3)) * 2;
        typedef __attribute__((address_space(3))) s16x4 lds4;
        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)at);
        const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(at + 8 * ST));
        return __builtin_bit_cast(frag_t<T>, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    }
}

// Registers 8s..8s+7 of a product as the operand of the next: fp32 as they are, 16 bits rounded to nearest even.  This is where probabilities and
// score gradients lose bits: the matrix instruction takes 16-bit operands, and a second product with what was cut off would cost as much as
// the first.  Each is off by at most half a step (2^-9 or 2^-12 of it), sums and statistics stay
// float32: 4 x 16 heads of 4096 x 4096 x 128 bf16 come out 2.3e-3 from 64 bits, unrounded probabilities 1.7e-3 (the result's own rounding).
template <class T> __device__ __forceinline__ frag_t<T> next_frag(const f32x16& x, int s) {
    f32x8 v;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = x[8 * s + j];
    return __builtin_convertvector(v, frag_t<T>);
}

// Rows on their way from memory to a tile: load() issues the loads, store() writes what is valid and zeros elsewhere.
template <class T, int DP, int ROWS, int THREADS> struct Stage {
    static constexpr int PER = El<T>::PER16, CPR = DP / PER, N = ROWS * CPR / THREADS, STEP = THREADS / CPR;
    static_assert(ROWS * CPR % THREADS == 0 && THREADS % CPR == 0, "Stage");
    u32x4 x[N];
    template <class F> __device__ __forceinline__ void load(F row, int D, int tid) {
        const int d = tid % CPR * PER;
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = load16(row(i * STEP + tid / CPR) + (d < D ? d : 0));
    }
    // consecutive rows that are all there: `at` is this thread's place in the first of them (own()), no multiplications on the way
    static __device__ __forceinline__ const T* own(const T* first, int64_t stride, int D, int tid) {
        const int d = tid % CPR * PER;
        return first + tid / CPR * stride + (d < D ? d : 0);
    }
    __device__ __forceinline__ void load_run(const T* at, int64_t stride) {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = load16(at + i * (STEP * stride));
    }
    __device__ __forceinline__ void store(char* tile, uint64_t bits, int D, int tid) const {
        constexpr uint64_t FULL = ROWS == 64 ? ~0ull : (1ull << (ROWS & 63)) - 1;
        char* at = tile + tid / CPR * Tile<T, DP>::STRIDE + tid % CPR * 16;
        if (bits == FULL && D == DP) {
#pragma unroll
            for (int i = 0; i < N; ++i) *(u32x4*)(at + i * (STEP * Tile<T, DP>::STRIDE)) = x[i];
            return;
        }
        const bool in = tid % CPR * PER < D;
#pragma unroll
        for (int i = 0; i < N; ++i)
            *(u32x4*)(at + i * (STEP * Tile<T, DP>::STRIDE)) = in && ((bits >> (i * STEP + tid / CPR)) & 1) ? x[i] : u32x4{0, 0, 0, 0};
    }
};

// rows of a unit of attn_split, attn_few and attn16_forward, whose splits attn_join joins
template <class T> constexpr int unit_rows() { return sizeof(T) == 4 ? 16 : 32; }

// writes of this wave to LDS are visible to its own later reads by other lanes
__device__ __forceinline__ void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// ---- host side -----------------------------------------------------------------------------------------------------------------
int run_of(const oph_seq_attn* a, int64_t groups, bool few);
int attn16_launch(const AttnP& p, int64_t groups, int what, void* stream);      // oph_attn32.hip: 0 forward, 1 dq, 2 dk and dv
int attn_few_forward(const AttnP& p, int dtype, int64_t groups, void* stream);     // oph_attnfew.hip: M <= 4
int attn_check(const oph_seq_attn* a, bool gradient);
AttnP attn_params(const oph_seq_attn* a);
int64_t attn_forward_workspace(const oph_seq_attn* a);
int64_t attn_gradient_workspace(const oph_seq_attn* a);

}  // namespace ophseq
#pragma GCC visibility pop
