// Embedding lookup with scaling, and its gradient by sorted tokens: oph_seq_embed_lookup, oph_seq_embed_gradient.
//
// Gradient.  embed_order lists the positions of every table row in ascending order, row after row (a stable sort by row, in one
// launch): each workgroup owns one bucket of rows (row mod buckets), reads all ids from the L2, keeps those of its bucket in LDS (or, where
// one wave meets more than KEEP, reads them again) and learns from the same reading how many tokens lie in the buckets before its own.
// embed_sum walks the sorted tokens in pieces, one run of equal rows after the other; a run inside a piece goes straight to the
// gradient, what crosses a border is left in `part` and summed by embed_join, every fourth piece by one wave, then the four.  No floating-point
// atomics: n, units and type alone decide the order of a sum.
#include "oph_seq.h"
#include "../../include/ophelia_hip.h"

#include <algorithm>
#include <type_traits>

namespace ophseq {

constexpr int FEW_ROWS = 512, FEW_TOKENS = 4096;            // most of embed_rows
constexpr int ZEROS = 8;                                    // rows that a group of embed_sum looks through
constexpr int WAVES = 16, LOCAL = 1024, KEEP = 256;         // embed_order: waves, most rows of a bucket, tokens that a wave keeps

struct EmbedP {
    const void *ids, *src;          // src: table or dout
    void* out;                      // rows or gradient
    int* head;                      // [0]: number of sorted tokens, from [4] on: their positions, their rows, then every row's number of tokens
    float* part;                    // [piece][begun before | goes on][U4]
    int64_t n, stride;
    int vocab, units, u4, zero_pad, lpr, buckets, shift, chunk, sums;      // chunk: tokens of a piece | sums: workgroups of embed_sum that sum
    float scale;
};

// the row that token i names; -1: none
template <class I> __device__ __forceinline__ int row_of(const EmbedP& p, int64_t i) {
    const int64_t id = ((const I*)p.ids)[i];
    return id < 0 || id >= p.vocab || (id == 0 && p.zero_pad) ? -1 : (int)id;
}

// PER16 consecutive elements of a row as floats; `left` elements remain in the row
template <class T> __device__ __forceinline__ void load_piece(float (&x)[El<T>::PER16], const T* at, int left) {
    constexpr int PER = El<T>::PER16;
    typedef T vec __attribute__((ext_vector_type(PER)));
    if (left >= PER) {
        const vec v = __builtin_bit_cast(vec, load16(at));
#pragma unroll
        for (int j = 0; j < PER; ++j) x[j] = (float)v[j];
    } else {
#pragma unroll
        for (int j = 0; j < PER; ++j) x[j] = j < left ? (float)at[j] : 0.f;
    }
}
template <class T> __device__ __forceinline__ void store_piece(T* at, const float (&x)[El<T>::PER16], int left) {
    constexpr int PER = El<T>::PER16;
    typedef T vec __attribute__((ext_vector_type(PER)));
    if (left >= PER) {
        vec v;
#pragma unroll
        for (int j = 0; j < PER; ++j) v[j] = (T)x[j];
        store16(at, __builtin_bit_cast(u32x4, v));
    } else {
#pragma unroll
        for (int j = 0; j < PER; ++j)
            if (j < left) at[j] = (T)x[j];
    }
}

// lpr lanes (a power of two) copy a row, 16 bytes at a time
template <class T, class I> __global__ __launch_bounds__(256) void embed_lookup(const EmbedP p) {
    constexpr int PER = El<T>::PER16;
    const int lane = threadIdx.x & (p.lpr - 1);
    const int64_t step = (int64_t)gridDim.x * (256 / p.lpr);
    for (int64_t i = (int64_t)blockIdx.x * (256 / p.lpr) + threadIdx.x / p.lpr; i < p.n; i += step) {
        const int row = row_of<I>(p, i);
        const T* from = (const T*)p.src + (row < 0 ? 0 : row) * p.stride;
        T* to = (T*)p.out + i * p.units;
        for (int c = lane * PER; c < p.units; c += p.lpr * PER) {
            float x[PER];
            if (row >= 0) load_piece<T>(x, from + c, p.units - c);
#pragma unroll
            for (int j = 0; j < PER; ++j) x[j] = row >= 0 ? x[j] * p.scale : 0.f;
            store_piece<T>(to + c, x, p.units - c);
        }
    }
}

// bucket b = blockIdx.x holds rows b, b + buckets, ...; the row's number inside it is row >> shift
template <class I> __global__ __launch_bounds__(64 * WAVES) void embed_order(const EmbedP p) {
    __shared__ int count[WAVES][LOCAL];
    __shared__ int2 kept[WAVES][KEEP];
    __shared__ int wsum[WAVES], wless[WAVES];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, bucket = blockIdx.x;
    const int local = (p.vocab - bucket + p.buckets - 1) >> p.shift;            // rows of this bucket, at most LOCAL
    for (int w = 0; w < WAVES; ++w)
        if (tid < local) count[w][tid] = 0;
    __syncthreads();
    const int64_t per = (p.n + 64 * WAVES - 1) / (64 * WAVES) * 64;
    const int64_t beg = wave * per, end = std::min(p.n, beg + per);
    int less = 0, found = 0;
    const unsigned lowest = p.zero_pad ? 1 : 0, rows = (unsigned)p.vocab - lowest;
    auto look = [&](int64_t i0, auto ahead) {                                      // at the 64 * ahead tokens from i0 on
        constexpr int AHEAD = decltype(ahead)::value;
        I id[AHEAD];
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) id[a] = ((const I*)p.ids)[std::min(i0 + 64 * a + lane, p.n - 1)];
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {                                        // the counting is on lane masks, a few instructions per 64 tokens
            const unsigned row = (unsigned)id[a];
            uint64_t there = __ballot(row - lowest < rows) & (sizeof(I) == 8 ? __ballot((uint64_t)id[a] >> 32 == 0) : ~0ull);
            const int64_t left = end - (i0 + 64 * a);
            if (left < 64) there &= left > 0 ? (1ull << left) - 1 : 0;
            const unsigned b = row & (p.buckets - 1);
            less += __popcll(__ballot(b < (unsigned)bucket) & there);
            const uint64_t all = __ballot(b == (unsigned)bucket) & there;
            if (all) {
                const int to = found + __popcll(all & ((1ull << lane) - 1));
                if ((all >> lane) & 1) {
                    if (to < KEEP) kept[wave][to] = make_int2((int)(i0 + 64 * a + lane), (int)row);
                    atomicAdd(&count[wave][row >> p.shift], 1);
                }
                found += __popcll(all);
            }
        }
    };
    int64_t i0 = beg;
    for (; i0 + 64 * 16 <= end; i0 += 64 * 16) look(i0, std::integral_constant<int, 16>());
    for (; i0 < end; i0 += 64 * 4) look(i0, std::integral_constant<int, 4>());
    if (lane == 0) wless[wave] = less;
    __syncthreads();
    // exclusive sums over (row, wave): thread = row
    int own = 0;
    if (tid < local)
        for (int w = 0; w < WAVES; ++w) own += count[w][tid];
    int run = own;
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) {
        const int x = __shfl_up(run, i);
        if (lane >= i) run += x;
    }
    if (lane == 63) wsum[wave] = run;
    __syncthreads();
    int base = 0;
    for (int w = 0; w < WAVES; ++w) base += wless[w] + (w < wave ? wsum[w] : 0);
    int at = base + run - own;
    if (tid < local)
        for (int w = 0; w < WAVES; ++w) {
            const int c = count[w][tid];
            count[w][tid] = at;
            at += c;
        }
    if (bucket == p.buckets - 1 && tid == 64 * WAVES - 1) p.head[0] = at;       // the last thread's end is the end of all
    __syncthreads();
    int *pos = p.head + 4, *key = pos + p.n;
    if (tid < local) key[p.n + ((int64_t)tid << p.shift) + bucket] = own;
    auto place = [&](int at, int row, bool mine) {                               // of a wave's tokens in order, 64 at a time
        uint64_t todo = __ballot(mine);
        while (todo) {
            const int leader = __ffsll((unsigned long long)todo) - 1;
            const int r = __builtin_amdgcn_readlane(row, leader);
            const uint64_t same = __ballot(mine && row == r);
            const int first = count[wave][r >> p.shift];
            if (mine && row == r) {
                const int to = first + __popcll(same & ((1ull << lane) - 1));
                pos[to] = at;
                key[to] = r;
            }
            if (lane == leader) count[wave][r >> p.shift] = first + __popcll(same);
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            todo &= ~same;
        }
    };
    if (found <= KEEP) {
        for (int e = lane; e - lane < found; e += 64) {
            const int2 x = kept[wave][min(e, KEEP - 1)];
            place(x.x, x.y, e < found);
        }
    } else {
        for (int64_t i = beg + lane; i - lane < end; i += 64) {
            const int row = i < end ? row_of<I>(p, i) : -1;
            place((int)i, row, row >= 0 && (row & (p.buckets - 1)) == bucket);
        }
    }
}

// lpr lanes per (piece, lpr * PER16 channels).  The workgroups from `sums` on write the rows that no token names: stores that run beside
// the others' loads.
template <class T> __global__ __launch_bounds__(256) void embed_sum(const EmbedP p) {
    constexpr int PER = El<T>::PER16, AHEAD = 2;
    const int lane = threadIdx.x & (p.lpr - 1), count = p.head[0];
    const int64_t piece = (int64_t)blockIdx.x * (256 / p.lpr) + threadIdx.x / p.lpr;
    const int c = (blockIdx.y * p.lpr + lane) * PER, left = p.units - c;
    if (left <= 0) return;
    const int *pos = p.head + 4, *key = pos + p.n;
    if ((int)blockIdx.x >= p.sums) {
        const float zero[PER] = {};
        const int64_t row0 = (piece - (int64_t)p.sums * (256 / p.lpr)) * ZEROS;
#pragma unroll
        for (int r = 0; r < ZEROS; ++r)
            if (row0 + r < p.vocab && key[p.n + row0 + r] == 0) store_piece<T>((T*)p.out + (row0 + r) * p.units + c, zero, left);
        return;
    }
    if (piece * p.chunk >= count) return;
    const int beg = (int)piece * p.chunk, end = min(count, beg + p.chunk);
    const T* src = (const T*)p.src + c;
    int cur = key[beg];
    bool begun = beg > 0 && key[beg - 1] == cur;
    const int after = end < count ? key[end] : -1;
    float acc[PER] = {};
    auto flush = [&](bool goes_on) {
        if (begun || goes_on) {
            float* to = p.part + (piece * 2 + (begun ? 0 : 1)) * p.u4 + c;
#pragma unroll
            for (int j = 0; j < PER; j += 4)
                if (j < left) *(f32x4*)(to + j) = f32x4{acc[j], acc[j + 1], acc[j + 2], acc[j + 3]};   // u4 is left rounded up to 4
        } else {
            float x[PER];
#pragma unroll
            for (int j = 0; j < PER; ++j) x[j] = acc[j] * p.scale;
            store_piece<T>((T*)p.out + (int64_t)cur * p.units + c, x, left);
        }
    };
    int row[AHEAD], at[AHEAD];                                                  // of the next tokens, a round ahead of their rows' loads
    auto look = [&](int i) {
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
            const int k = min(i + a, end - 1);
            row[a] = key[k];
            at[a] = pos[k];
        }
    };
    look(beg);
    for (int i = beg; i < end; i += AHEAD) {
        float x[AHEAD][PER];
        int now[AHEAD];
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
            now[a] = row[a];
            load_piece<T>(x[a], src + (int64_t)at[a] * p.stride, left);
        }
        look(i + AHEAD);
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
            if (i + a >= end) break;
            if (now[a] != cur) {
                flush(false);
                cur = now[a];
                begun = false;
#pragma unroll
                for (int j = 0; j < PER; ++j) acc[j] = 0.f;
            }
#pragma unroll
            for (int j = 0; j < PER; ++j) acc[j] += x[a][j];
        }
    }
    flush(cur == after);
}

// a workgroup per (piece in which a run begins that goes on in the next, 256 channels): its parts, every fourth by one wave, then the four
// sums
template <class T> __global__ __launch_bounds__(256) void embed_join(const EmbedP p) {
    __shared__ f32x4 sums[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, count = p.head[0];
    const int64_t piece = blockIdx.x, beg = piece * p.chunk, end = beg + p.chunk;
    if (end >= count) return;                                                   // the last piece's runs end in it
    const int *key = p.head + 4 + p.n, row = key[end - 1];
    if (key[end] != row || (beg > 0 && key[beg - 1] == row)) return;             // ends here, or began before: row fills the piece then
    int64_t parts = 0;                                                          // pieces that the run goes on through
    for (;;) {
        const int64_t at = (piece + 1 + parts + lane) * p.chunk;
        const uint64_t on = __ballot(at < count && key[min(at, (int64_t)count - 1)] == row);
        parts += on == ~0ull ? 64 : __ffsll((unsigned long long)~on) - 1;
        if (on != ~0ull) break;
    }
    const int c = (blockIdx.y * 64 + lane) * 4;
    const float* at = p.part + c;
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    if (c < p.u4) {
        if (wave == 0) s = *(const f32x4*)(at + (piece * 2 + 1) * p.u4);
#pragma unroll 8
        for (int64_t q = wave; q < parts; q += 4) s += *(const f32x4*)(at + (piece + 1 + q) * 2 * p.u4);
    }
    sums[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && c < p.units) {
        s = sums[0][lane];
#pragma unroll
        for (int w = 1; w < 4; ++w) s += sums[w][lane];
        T* to = (T*)p.out + (int64_t)row * p.units + c;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (c + j < p.units) to[j] = (T)(s[j] * p.scale);
    }
}

// A small table and few tokens, in one launch: a workgroup per (row, lpr * PER16 channels) lists the row's tokens in LDS, its groups of lpr
// lanes take them in turn, and the groups' sums are added in their order.
template <class T, class I> __global__ __launch_bounds__(256) void embed_rows(const EmbedP p) {
    constexpr int PER = El<T>::PER16, AHEAD = 8, MOST = FEW_TOKENS / 4;
    __shared__ int list[4][MOST];
    __shared__ int counts[4];
    __shared__ __attribute__((aligned(16))) float sums[256 * PER];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row = blockIdx.x;
    const int n = (int)p.n, per = (n + 255) / 256 * 64, beg = wave * per, end = min(n, beg + per);
    int found = 0;
    for (int i0 = beg; i0 < end; i0 += 64 * AHEAD) {
        I id[AHEAD];
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) id[a] = ((const I*)p.ids)[min(i0 + 64 * a + lane, n - 1)];
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
            const int i = i0 + 64 * a + lane;
            const bool mine = id[a] == (I)row && i < end;
            const uint64_t all = __ballot(mine);
            if (mine) list[wave][found + __popcll(all & ((1ull << lane) - 1))] = i;
            found += __popcll(all);
        }
    }
    if (lane == 0) counts[wave] = row == 0 && p.zero_pad ? 0 : found;
    __syncthreads();
    const int c1 = counts[0], c2 = c1 + counts[1], c3 = c2 + counts[2], count = c3 + counts[3];
    const int li = tid & (p.lpr - 1), group = tid / p.lpr, groups = 256 / p.lpr, c = (blockIdx.y * p.lpr + li) * PER, left = p.units - c;
    float acc[PER] = {};
    if (left > 0)
        for (int e = group; e < count; e += groups * AHEAD) {
            float x[AHEAD][PER];
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
                const int k = min(e + a * groups, count - 1), w = (k >= c1) + (k >= c2) + (k >= c3);
                const int i = list[w][k - (w == 0 ? 0 : w == 1 ? c1 : w == 2 ? c2 : c3)];
                load_piece<T>(x[a], (const T*)p.src + (int64_t)i * p.stride + c, left);
            }
#pragma unroll
            for (int a = 0; a < AHEAD; ++a)
#pragma unroll
                for (int j = 0; j < PER; ++j) acc[j] += e + a * groups < count ? x[a][j] : 0.f;
        }
#pragma unroll
    for (int j = 0; j < PER; ++j) sums[tid * PER + j] = acc[j];
    __syncthreads();
    if (group || left <= 0) return;
    for (int g = 1; g < groups; ++g)
#pragma unroll
        for (int j = 0; j < PER; ++j) acc[j] += sums[(g * p.lpr + li) * PER + j];
#pragma unroll
    for (int j = 0; j < PER; ++j) acc[j] *= p.scale;
    store_piece<T>((T*)p.out + (int64_t)row * p.units + c, acc, left);
}

// ---- host side ---------------------------------------------------------------------------------------------------------------------------
static int check(const void* ids, int id_bytes, int64_t n, int64_t stride, int vocab, int units, float scale, int dtype, const char* what) {
    if (!type_bytes(dtype)) return fail(OPH_ERR_INVALID, "%s: dtype %d is not one of OPH_SEQ_*", what, dtype);
    if (id_bytes != 4 && id_bytes != 8) return fail(OPH_ERR_INVALID, "%s: ids of %d bytes (4 or 8)", what, id_bytes);
    if (n < 0 || n > 1 << 27) return fail(OPH_ERR_INVALID, "%s: %lld ids", what, (long long)n);
    if (vocab < 1 || vocab > 1 << 28 || units < 1 || units > 1 << 24) return fail(OPH_ERR_INVALID, "%s: table of %d rows of %d", what, vocab, units);
    if (stride < 0) return fail(OPH_ERR_INVALID, "%s: negative stride", what);
    if (n && !ids) return fail(OPH_ERR_INVALID, "%s: ids must not be NULL", what);
    if (!(scale - scale == 0.f)) return fail(OPH_ERR_INVALID, "%s: scale %g is not finite", what, (double)scale);
    return OPH_OK;
}
static int lanes_for(int units, int dtype) {
    const int pieces = (int)cdiv(units, 16 / type_bytes(dtype));
    int l = 1;
    while (l < pieces && l < 64) l *= 2;
    return l;
}
static int bucket_count(int vocab) {
    int b = 1;
    while ((b < 256 && b < vocab) || (int64_t)b * LOCAL < vocab) b *= 2;
    return b;
}
// Tokens of a piece.  Many short pieces with two rows in flight each beat long ones with more: with inputs that are in no cache, 32768 tokens x
// 1024 bf16 of 32000 rows take 45 us (pieces of 8: 49, of 32: 58; four rows ahead 50, eight 56); few tokens fill the machine with shorter ones.
static bool few(int64_t n, int vocab);
static int chunk_for(int64_t n) { return n <= 8192 ? 8 : 16; }
static int64_t part_offset(int64_t n, int vocab) { return cdiv((4 + 2 * n + vocab) * 4, 16) * 16; }

template <class T, class I> static int lookup(const EmbedP& p, void* stream) {
    return launch<EmbedP>(embed_lookup<T, I>, dim3((unsigned)std::min<int64_t>(cdiv(p.n, 256 / p.lpr), 1 << 20)), 256, p, 0, stream);
}
// embed_rows instead of three launches: 2400 tokens of 57 rows of 128 fp32 take 5.5 us instead of 14.  One workgroup then sums all tokens of a
// row, so that runs have to be short on average.
static bool few(int64_t n, int vocab) { return n <= FEW_TOKENS && vocab <= FEW_ROWS && n <= 64 * (int64_t)vocab; }
template <class T, class I> static int gradient(EmbedP p, void* stream) {
    if (few(p.n, p.vocab))
        return launch<EmbedP>(embed_rows<T, I>, dim3(p.vocab, (unsigned)cdiv(p.units, p.lpr * El<T>::PER16)), 256, p, 0, stream);
    if (int rc = launch<EmbedP>(embed_order<I>, dim3(p.buckets), 64 * WAVES, p, 0, stream)) return rc;
    const int64_t pieces = cdiv(p.n, p.chunk), groups = 256 / p.lpr;
    p.sums = (int)cdiv(pieces, groups);
    const dim3 grid((unsigned)(p.sums + cdiv(cdiv(p.vocab, ZEROS), groups)), (unsigned)cdiv(p.units, p.lpr * El<T>::PER16));
    if (int rc = launch<EmbedP>(embed_sum<T>, grid, 256, p, 0, stream)) return rc;
    if (pieces <= 1) return OPH_OK;
    return launch<EmbedP>(embed_join<T>, dim3((unsigned)pieces, (unsigned)cdiv(p.units, 256)), 256, p, 0, stream);
}
template <class T> static int lookup_i(const EmbedP& p, int id_bytes, void* s) { return id_bytes == 4 ? lookup<T, int32_t>(p, s) : lookup<T, int64_t>(p, s); }
template <class T> static int gradient_i(const EmbedP& p, int id_bytes, void* s) { return id_bytes == 4 ? gradient<T, int32_t>(p, s) : gradient<T, int64_t>(p, s); }

}  // namespace ophseq

using namespace ophseq;
extern "C" {

int oph_seq_embed_lookup(const void* ids, int id_bytes, int64_t n, const void* table, int64_t table_stride, int vocab, int units, float scale,
                         int zero_pad, int dtype, void* out, int device, void* stream) {
    if (int rc = check(ids, id_bytes, n, table_stride, vocab, units, scale, dtype, "embedding lookup")) return rc;
    if (!n) return OPH_OK;
    if (!table || !out) return fail(OPH_ERR_INVALID, "embedding lookup: table and out must not be NULL");
    OnDevice on(device);
    if (on.status) return on.status;
    EmbedP p = {};
    p.ids = ids; p.src = table; p.out = out; p.n = n; p.stride = table_stride; p.vocab = vocab; p.units = units; p.zero_pad = zero_pad != 0;
    p.lpr = lanes_for(units, dtype);
    p.scale = scale;
    if (dtype == OPH_SEQ_F32) return lookup_i<float>(p, id_bytes, stream);
    if (dtype == OPH_SEQ_BF16) return lookup_i<bf16_t>(p, id_bytes, stream);
    return lookup_i<f16_t>(p, id_bytes, stream);
}

int64_t oph_seq_embed_workspace(int64_t n, int vocab, int units) {
    if (int rc = check(&n, 4, n, 0, vocab, units, 1.f, OPH_SEQ_F32, "embedding gradient")) return rc;
    if (few(n, vocab)) return 0;
    return part_offset(n, vocab) + cdiv(n, chunk_for(n)) * 2 * cdiv(units, 4) * 16;
}

int oph_seq_embed_gradient(const void* ids, int id_bytes, int64_t n, const void* dout, int64_t dout_stride, int vocab, int units, float scale,
                           int zero_pad, int dtype, void* grad, void* workspace, size_t workspace_bytes, int device, void* stream) {
    if (int rc = check(ids, id_bytes, n, dout_stride, vocab, units, scale, dtype, "embedding gradient")) return rc;
    if (!grad || (n && !dout)) return fail(OPH_ERR_INVALID, "embedding gradient: dout and grad must not be NULL");
    const int64_t need = oph_seq_embed_workspace(n, vocab, units);
    if (need && (!workspace || (int64_t)workspace_bytes < need || ((uintptr_t)workspace & 15)))
        return fail(OPH_ERR_INVALID, "embedding gradient: the workspace must hold %lld bytes, 16-byte aligned", (long long)need);
    OnDevice on(device);
    if (on.status) return on.status;
    EmbedP p = {};
    p.ids = ids; p.src = dout; p.out = grad; p.n = n; p.stride = dout_stride; p.vocab = vocab; p.units = units; p.zero_pad = zero_pad != 0;
    p.u4 = (int)cdiv(units, 4) * 4;
    p.lpr = lanes_for(units, dtype);
    p.scale = scale;
    p.buckets = bucket_count(vocab);
    while ((1 << p.shift) < p.buckets) ++p.shift;
    p.head = (int*)workspace;
    p.chunk = chunk_for(n);
    p.part = (float*)((char*)workspace + part_offset(n, vocab));      // not followed where the workspace is empty
    if (dtype == OPH_SEQ_F32) return gradient_i<float>(p, id_bytes, stream);
    if (dtype == OPH_SEQ_BF16) return gradient_i<bf16_t>(p, id_bytes, stream);
    return gradient_i<f16_t>(p, id_bytes, stream);
}

}  // extern "C"
