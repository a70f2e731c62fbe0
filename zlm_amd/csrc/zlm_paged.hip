// zlm_paged.hip -- CDNA4 (gfx950) kernels over a paged KV cache: q/k head norm,
// RoPE and the append of a batch's K and V (f16 or 4-bit q4_0 blocks), the rows
// read back, and the attention of the batch over its sequences' pages.  Built as a
// device-only code object (hipcc --genco) and loaded by the host library.
//
// A page holds `page` positions of every kv head, K and V in a pool each.  The
// two layouts are the MFMA operand orders of the attention below, so that its
// lanes load whole operands from memory without a transpose.  Per head of a page:
//   K  f16  [page][hd]
//      q4_0 [page][hd/32][16 nibble bytes in GGUF order], then f16 [page][hd/32]
//   V, by groups of 8 positions
//      f16  [page/8][hd][8]
//      q4_0 one word of 8 nibbles per (group, dim), position j's at bits
//           4*(j/2) + 16*(j%2): [page/8][hd], then f16 scales [page/8][hd/32][8]
// A q4_0 value is d * (nibble - 8).  d has at most 8 significant bits, so that
// d * (nibble - 8) is exact in f16, and is at most 2720 in size, so that 24 d is
// finite in f16: the decode below is one exact fma.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "paged_args.h"

namespace {

using zlm::Paged;
using AppendArgs = zlm::PagedAppend;
using ReadArgs = zlm::PagedRead;
using AttnArgs = zlm::PagedAttend;

constexpr uint32_t kWave = 64;
constexpr uint32_t kMaxSeqs = zlm::kPagedMaxSeqs;

typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));

template <int HD, bool Q4>
struct Row {
    static constexpr uint32_t kBytes = Q4 ? HD / 2 + HD / 16 : HD * 2;
};

// The sequence of row t (n_seqs when it lies behind the last one): the number of
// sequences that end at or before t, counted by the whole wave (all of q_start is
// loaded at once, one memory latency).
__device__ __forceinline__ uint32_t seq_of(const Paged& p, int32_t t, uint32_t lane) {
    uint32_t s = 0;
    for (uint32_t b = 0; b < p.n_seqs; b += kWave) {
        const bool done = b + lane < p.n_seqs && p.q_start[b + lane + 1] <= t;
        s += __builtin_popcountll(__ballot(done));
    }
    return __builtin_amdgcn_readfirstlane(s);
}

// Row t's sequence and position; false for a row that belongs to none.  What the
// batch's arrays hold never leads outside the buffers: rows end at n_tokens.
struct RowAt {
    uint32_t s;
    int32_t row0, row1;  // the sequence's rows
    int32_t pos, first;  // t's position, that of row0
};

__device__ __forceinline__ bool row_at(const Paged& p, uint32_t t, uint32_t lane, RowAt& r) {
    r.s = seq_of(p, static_cast<int32_t>(t), lane);
    if (r.s >= p.n_seqs) return false;
    r.row0 = p.q_start[r.s];
    const int32_t row1 = p.q_start[r.s + 1];
    r.row1 = min(row1, static_cast<int32_t>(p.n_tokens));
    if (static_cast<int32_t>(t) < r.row0 || static_cast<int32_t>(t) >= r.row1 || r.row0 < 0) return false;
    const uint32_t past = static_cast<uint32_t>(p.kv_len[r.s]) - static_cast<uint32_t>(row1);
    r.pos = static_cast<int32_t>(past + t);
    r.first = static_cast<int32_t>(past + static_cast<uint32_t>(r.row0));
    return true;
}

// The page of position `pos` of sequence s, or -1.
__device__ __forceinline__ int32_t page_of(const Paged& p, uint32_t s, int32_t pos) {
    if (pos < 0 || (static_cast<uint32_t>(pos) >> p.page_shift) >= p.table_stride) return -1;
    const int32_t id = p.table[static_cast<size_t>(s) * p.table_stride + (static_cast<uint32_t>(pos) >> p.page_shift)];
    return static_cast<uint32_t>(id) < p.n_pages ? id : -1;
}

template <int HD, bool Q4>
__device__ __forceinline__ size_t head_base(const Paged& p, uint32_t page, uint32_t h) {
    const uint32_t head_bytes = Row<HD, Q4>::kBytes << p.page_shift;
    return (static_cast<size_t>(page) * p.n_kv + h) * head_bytes;
}

// The value of another lane of the row of 16, by a DPP control.
template <int kCtrl, class T>
__device__ __forceinline__ T dpp(T v) {
    if constexpr (sizeof(T) == 4) {
        return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), kCtrl, 0xf, 0xf, true));
    } else {
        const uint64_t u = __builtin_bit_cast(uint64_t, v);
        const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(u), kCtrl, 0xf, 0xf, true);
        const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(u >> 32), kCtrl, 0xf, 0xf, true);
        return __builtin_bit_cast(T, static_cast<uint64_t>(hi) << 32 | lo);
    }
}
constexpr int kXor1 = 0xb1, kXor2 = 0x4e, kHalfMirror = 0x141, kMirror = 0x140;

// The value of the neighbouring row of 16 (rows 0 and 1, 2 and 3).
__device__ __forceinline__ uint32_t next_row(uint32_t v) {
    const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    const uint32_t x = a[0], y = a[1];
    return threadIdx.x & 16 ? x : y;
}

// The value of lane + or - 32.
__device__ __forceinline__ double other_half(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = static_cast<uint32_t>(u), hi = static_cast<uint32_t>(u >> 32);
    const auto a = __builtin_amdgcn_permlane32_swap(lo, lo, false, false);
    const auto b = __builtin_amdgcn_permlane32_swap(hi, hi, false, false);
    const uint32_t a0 = a[0], a1 = a[1], b0 = b[0], b1 = b[1];
    const bool upper = (threadIdx.x & 32) != 0;
    return __builtin_bit_cast(double, static_cast<uint64_t>(upper ? b0 : b1) << 32 | (upper ? a0 : a1));
}

// Two sums a step closer: x's in the lanes whose bit is clear, y's in the others.
template <bool kHalves>  // the bit: 32, or 16
__device__ __forceinline__ double fold(double x, double y) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x), v = __builtin_bit_cast(uint64_t, y);
    const auto swap = [](uint64_t p, uint64_t q) {
        const uint32_t a = static_cast<uint32_t>(p), b = static_cast<uint32_t>(q);
        return kHalves ? __builtin_amdgcn_permlane32_swap(a, b, false, false)
                       : __builtin_amdgcn_permlane16_swap(a, b, false, false);
    };
    const auto lo = swap(u, v), hi = swap(u >> 32, v >> 32);
    const uint32_t l0 = lo[0], l1 = lo[1], h0 = hi[0], h1 = hi[1];
    return __builtin_bit_cast(double, static_cast<uint64_t>(h0) << 32 | l0) +
           __builtin_bit_cast(double, static_cast<uint64_t>(h1) << 32 | l1);
}

// Four sums over the wave at the price of one and a half: 0, 2, 1 and 3 in its rows.
__device__ __forceinline__ double wave_sums(const double v[4]) {
    double x = fold<false>(fold<true>(v[0], v[1]), fold<true>(v[2], v[3]));
    x += dpp<kXor1>(x);
    x += dpp<kXor2>(x);
    x += dpp<kHalfMirror>(x);
    return x + dpp<kMirror>(x);
}
__device__ __forceinline__ double of_row(double v, int row) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(u), 16 * row);
    const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(u >> 32), 16 * row);
    return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}

// The q4_0 block of 32 values, one a lane of each half wave: d from the first of
// the largest, and this lane's nibble.  T: what the values are exact in.
template <class T>
__device__ __forceinline__ uint32_t quantise(T x, uint32_t lane, _Float16* d_out) {
    const float xf = static_cast<float>(x), a = __builtin_fabsf(xf);
    float mx = a;
    mx = __builtin_fmaxf(mx, dpp<kXor1>(mx));
    mx = __builtin_fmaxf(mx, dpp<kXor2>(mx));
    mx = __builtin_fmaxf(mx, dpp<kHalfMirror>(mx));
    mx = __builtin_fmaxf(mx, dpp<kMirror>(mx));
    mx = __builtin_fmaxf(mx, __builtin_bit_cast(float, next_row(__builtin_bit_cast(uint32_t, mx))));
    const auto half = [&](uint64_t b) { return static_cast<uint32_t>(lane & 32 ? b >> 32 : b); };
    uint64_t largest = __ballot(a == mx);
    if constexpr (sizeof(T) > sizeof(float)) {
        // several that are one number in 32 bits (a tie, rare past blocks of zeros): the largest in 64
        const uint64_t low = largest & 0xffffffffull, high = largest >> 32;
        if ((low & (low - 1)) | (high & (high - 1))) {
            const T b = a == mx ? __builtin_fabs(x) : T(0);
            T top = b;
            top = __builtin_fmax(top, dpp<kXor1>(top));
            top = __builtin_fmax(top, dpp<kXor2>(top));
            top = __builtin_fmax(top, dpp<kHalfMirror>(top));
            top = __builtin_fmax(top, dpp<kMirror>(top));
            const uint64_t u = __builtin_bit_cast(uint64_t, top);
            top = __builtin_fmax(top, __builtin_bit_cast(T, static_cast<uint64_t>(next_row(static_cast<uint32_t>(u >> 32))) << 32 |
                                                                next_row(static_cast<uint32_t>(u))));
            largest &= __ballot(b == top);
        }
    }
    const uint32_t at = half(largest), negative = half(__ballot(xf < 0.0f));
    const bool nan = half(__ballot(xf != xf)) != 0;
    const bool minus = (negative & at & (0u - at)) != 0;  // the first's sign
    // -m/8 to 8 significant bits (bf16), then to f16 (further only below its normal range)
    const uint32_t u = __builtin_bit_cast(uint32_t, mx * 0.125f);
    const float r = __builtin_bit_cast(float, (u + 0x7fffu + ((u >> 16) & 1u)) & 0xffff0000u);
    const _Float16 size = static_cast<_Float16>(__builtin_fminf(r, 2720.0f));
    const float df = static_cast<float>(size);
    // floor(x/d + 8.5): nearly so by a reciprocal, then what it leaves tells, exactly
    const T xs = minus ? x : -x, dd = static_cast<T>(df);
    float c = __builtin_floorf(__builtin_fmaf(static_cast<float>(xs), __builtin_amdgcn_rcpf(df), 8.5f));
    c = __builtin_fminf(__builtin_fmaxf(c, -1.0f), 17.0f);
    const bool over = __builtin_fma(static_cast<T>(8.5f - c), dd, xs) < T(0);
    const bool under = __builtin_fma(static_cast<T>(7.5f - c), dd, xs) >= T(0);
    c += under ? 1.0f : over ? -1.0f : 0.0f;
    c = size != 0 ? __builtin_fminf(__builtin_fmaxf(c, 0.0f), 15.0f) : 8.0f;
    // a block with a NaN reads back as NaN
    *d_out = nan ? __builtin_bit_cast(_Float16, static_cast<uint16_t>(0x7e00)) : minus ? size : -size;
    return static_cast<uint32_t>(c);
}

// A workgroup: one row; its waves (and those of the row's other workgroups) deal the
// heads, four at a time, so that the sums of their norms take one pass over the lanes (or
// one, where there are waves for all).
// A lane holds dims lane + 64 j; the rotation's pair (i, i + hd/2) is in one
// lane for hd 128 and 256 and in lanes i and i + 32 for hd 64.  Angles, norm,
// rotation and the 4-bit decisions are formed in 64 bits: a rounding of the angle at
// position 1e5 in 32 bits is 4e-3.  The angles' functions are most of the
// arithmetic; the workgroup forms them once for all of its heads.
// 64 dims of V's 8-position groups are written by one wave, all of the group's rows in
// this call together: no two waves write one word.  The rows' workgroups take the heads
// in turn (left to the group's first row they were all on one XCD, every eighth
// workgroup's: prompts of 7270 rows together took 160 us, and 75 so).
template <int HD, bool Q4>
__device__ __forceinline__ void append(const AppendArgs& a) {
    const Paged& p = a.p;
    constexpr int N = HD / 64;  // dims a lane
    constexpr uint32_t kH = 4;  // heads a step, at most
    __shared__ double turns[2][HD / 2];
    const uint32_t tid = threadIdx.x, lane = tid & (kWave - 1);
    const uint32_t t = blockIdx.x;
    const uint32_t waves = gridDim.y * 4, wave = __builtin_amdgcn_readfirstlane(blockIdx.y * 4 + tid / kWave);
    const uint32_t heads = a.n_heads + p.n_kv;
    const float* row = a.qkv + t * a.stride + lane;
    uint32_t h = a.per * wave;
    // the next heads' values, on their way while these are worked on; past the last head its own
    float next[kH][N], wq[N], wk[N];
    const auto load = [&](uint32_t h0) {
#pragma unroll
        for (uint32_t i = 0; i < kH; i++)
#pragma unroll
            for (int j = 0; j < N; j++) next[i][j] = row[static_cast<size_t>(min(h0 + i, heads - 1)) * HD + 64 * j];
    };
    if (h < heads) load(h);
    const bool norm = a.q_norm != nullptr;
#pragma unroll
    for (int j = 0; j < N; j++) {
        wq[j] = norm ? a.q_norm[lane + 64 * j] : 1.0f;
        wk[j] = norm ? a.k_norm[lane + 64 * j] : 1.0f;
    }
    RowAt at;
    if (!row_at(p, t, lane, at)) return;  // a row behind the last sequence: left as it was
    const uint32_t s = at.s;
    const int32_t pos = at.pos;
    const uint32_t page = 1u << p.page_shift;
    const int32_t id = __builtin_amdgcn_readfirstlane(page_of(p, s, pos));
    if (tid < HD / 2) {
        const double turn = static_cast<double>(pos) * exp(a.log_base * (static_cast<double>(tid) * (-2.0 / HD)));
        sincos(turn, &turns[1][tid], &turns[0][tid]);
    }
    __syncthreads();
    double cs[N], sn[N];
#pragma unroll
    for (int j = 0; j < N; j++) {
        cs[j] = turns[0][(lane + 64 * j) % (HD / 2)];
        sn[j] = turns[1][(lane + 64 * j) % (HD / 2)];
    }
    for (; h < heads; h += a.per * waves) {
        double x[kH][N], inv = 1.0;
#pragma unroll
        for (uint32_t i = 0; i < kH; i++)
#pragma unroll
            for (int j = 0; j < N; j++) x[i][j] = next[i][j];
        load(h + a.per * waves);
        if (norm) {
            double ss[kH];
#pragma unroll
            for (uint32_t i = 0; i < kH; i++) {
                ss[i] = 0.0;
#pragma unroll
                for (int j = 0; j < N; j++) ss[i] = __builtin_fma(x[i][j], x[i][j], ss[i]);
            }
            inv = 1.0 / sqrt(wave_sums(ss) * (1.0 / HD) + static_cast<double>(a.eps));
        }
#pragma unroll
        for (uint32_t i = 0; i < kH; i++) {
            if (h + i >= heads || i >= a.per) break;
            const bool is_q = h + i < a.n_heads;
            if (norm) {
                const double f = of_row(inv, i >> 1 | (i & 1) << 1);
#pragma unroll
                for (int j = 0; j < N; j++) x[i][j] = x[i][j] * f * static_cast<double>(is_q ? wq[j] : wk[j]);
            }
            double y[N];
#pragma unroll
            for (int j = 0; j < N; j++) {
                double other;
                bool upper;
                if constexpr (HD == 64) {
                    other = other_half(x[i][0]);
                    upper = lane >= 32;
                } else {
                    other = x[i][(j + N / 2) % N];
                    upper = j >= N / 2;
                }
                y[j] = x[i][j] * cs[j] + (upper ? other : -other) * sn[j];
            }
            if (is_q) {
                float* dst = a.q_out + (static_cast<size_t>(t) * a.n_heads + h + i) * HD;
#pragma unroll
                for (int j = 0; j < N; j++) dst[lane + 64 * j] = pos < 0 ? 0.0f : static_cast<float>(y[j]);
                continue;
            }
            if (id < 0) continue;
            uint8_t* base = p.k + head_base<HD, Q4>(p, id, h + i - a.n_heads);
            const uint32_t off = static_cast<uint32_t>(pos) & (page - 1);
            if constexpr (!Q4) {
                _Float16* dst = reinterpret_cast<_Float16*>(base) + off * HD;
#pragma unroll
                for (int j = 0; j < N; j++) dst[lane + 64 * j] = static_cast<_Float16>(y[j]);  // one rounding
            } else {
#pragma unroll
                for (int j = 0; j < N; j++) {
                    _Float16 d;
                    const uint32_t n = quantise(y[j], lane, &d);
                    const uint32_t hi = next_row(n);
                    const uint32_t blk = 2 * j + lane / 32, e = lane & 31;
                    if (e < 16) base[off * (HD / 2) + blk * 16 + e] = static_cast<uint8_t>(n | (hi << 4));
                    if (e == 0) reinterpret_cast<_Float16*>(base + page * (HD / 2))[off * (HD / 32) + blk] = d;
                }
            }
        }
    }
    // V's 8-position groups: their rows of this call share their heads
    if (pos < 0 || id < 0) return;  // position 0 starts a group too
    const int32_t start = max(pos & ~7, at.first);
    const uint32_t j0 = static_cast<uint32_t>(start) & 7, mine = static_cast<uint32_t>(pos - start), t0 = t - mine;
    const uint32_t n_rows = min(8u - j0, static_cast<uint32_t>(at.row1) - t0);
    const uint32_t grp = (static_cast<uint32_t>(pos) & (page - 1)) >> 3;
    // 64 dims a wave; the last waves first: they had the fewest heads
    const uint32_t heads_of = mine < p.n_kv ? (p.n_kv - mine + n_rows - 1) / n_rows : 0;
    for (uint32_t i = waves - 1 - wave; i < heads_of * N; i += waves) {
        const uint32_t g = mine + n_rows * (i / N), dim = lane + 64 * (i % N);
        uint8_t* base = p.v + head_base<HD, Q4>(p, id, g);
        const float* src = a.qkv + t0 * a.stride + static_cast<size_t>(heads + g) * HD + dim;
        float x[8];
#pragma unroll
        for (uint32_t r = 0; r < 8; r++) x[r] = src[min(r, n_rows - 1) * a.stride];
        if constexpr (!Q4) {
            _Float16* dst = reinterpret_cast<_Float16*>(base) + (grp * HD + dim) * 8;
            if (n_rows == 8) {
                v8h o;
#pragma unroll
                for (int r = 0; r < 8; r++) o[r] = static_cast<_Float16>(x[r]);
                *reinterpret_cast<v8h*>(dst) = o;
            } else {
#pragma unroll
                for (uint32_t r = 0; r < 8; r++)
                    if (r < n_rows) dst[j0 + r] = static_cast<_Float16>(x[r]);
            }
        } else {
            uint32_t* word = reinterpret_cast<uint32_t*>(base) + grp * HD + dim;
            _Float16* sc = reinterpret_cast<_Float16*>(base + page * (HD / 2)) + (grp * (HD / 32) + dim / 32) * 8;
            uint32_t bits = 0, mask = 0;
#pragma unroll
            for (uint32_t r = 0; r < 8; r++) {
                if (r < n_rows) {  // wave-uniform
                    _Float16 d;
                    const uint32_t n = quantise(x[r], lane, &d);
                    const uint32_t to = j0 + r, sh = 4 * (to >> 1) + 16 * (to & 1);
                    bits |= n << sh;
                    mask |= 15u << sh;
                    if ((lane & 31) == 0) sc[to] = d;
                }
            }
            *word = n_rows == 8 ? bits : ((*word & ~mask) | bits);
        }
    }
}

// The batch's rows of the cache as f32, [n_tokens][n_kv][hd]; NaN where a
// position has no page, rows of negative positions 0.
template <int HD, bool Q4>
__device__ __forceinline__ void read_rows(const ReadArgs& a) {
    const Paged& p = a.p;
    const uint32_t lane = threadIdx.x & (kWave - 1), t = blockIdx.x;
    RowAt at;
    if (!row_at(p, t, lane, at)) return;
    const int32_t pos = at.pos, id = page_of(p, at.s, pos);
    const uint32_t page = 1u << p.page_shift, off = static_cast<uint32_t>(pos) & (page - 1);
    const uint32_t grp = off >> 3, in = off & 7;
    const uint32_t waves = gridDim.y * 4;
    constexpr int kH = 2, N = HD / 64;  // heads at a time: their loads are in flight together
    for (uint32_t h0 = blockIdx.y * 4 + threadIdx.x / kWave; h0 < p.n_kv; h0 += kH * waves) {
        float k[kH][N], v[kH][N];
#pragma unroll
        for (int i = 0; i < kH; i++) {
            const uint32_t h = min(h0 + i * waves, p.n_kv - 1);
#pragma unroll
            for (int j = 0; j < N; j++) {
                const uint32_t dim = lane + 64 * j;
                k[i][j] = v[i][j] = pos < 0 ? 0.0f : __builtin_nanf("");
                if (id < 0) continue;
                const uint8_t* kb = p.k + head_base<HD, Q4>(p, id, h);
                const uint8_t* vb = p.v + head_base<HD, Q4>(p, id, h);
                if constexpr (!Q4) {
                    k[i][j] = static_cast<float>(reinterpret_cast<const _Float16*>(kb)[off * HD + dim]);
                    v[i][j] = static_cast<float>(reinterpret_cast<const _Float16*>(vb)[(grp * HD + dim) * 8 + in]);
                } else {
                    const uint32_t b = kb[off * (HD / 2) + dim / 32 * 16 + (dim & 15)];
                    const float dk = reinterpret_cast<const _Float16*>(kb + page * (HD / 2))[off * (HD / 32) + dim / 32];
                    k[i][j] = (static_cast<float>((b >> (dim & 16 ? 4 : 0)) & 15) - 8.0f) * dk;
                    const uint32_t w = reinterpret_cast<const uint32_t*>(vb)[grp * HD + dim];
                    const float dv =
                        reinterpret_cast<const _Float16*>(vb + page * (HD / 2))[(grp * (HD / 32) + dim / 32) * 8 + in];
                    v[i][j] = (static_cast<float>((w >> (4 * (in >> 1) + 16 * (in & 1))) & 15) - 8.0f) * dv;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kH; i++) {
            const uint32_t h = h0 + i * waves;
            if (h >= p.n_kv) break;
            const size_t o = (static_cast<size_t>(t) * p.n_kv + h) * HD + lane;
#pragma unroll
            for (int j = 0; j < N; j++) {
                a.k_out[o + 64 * j] = k[i][j];
                a.v_out[o + 64 * j] = v[i][j];
            }
        }
    }
}

// ---- attention ---------------------------------------------------------------
//
// out[t, head] = sum_j softmax_j(scale q . k_j) v_j over the positions
// [max(0, pos - window + 1), pos] of the row's sequence.
//
// Both products run on v_mfma_f32_16x16x32_f16 with the queries in the N
// dimension: S^T = K Q^T, O^T = V^T P^T.  A lane then holds, of query row n =
// lane % 16, the scores of 8 consecutive positions 8q .. 8q+7 (q = lane / 16) --
// the K rows of the two 16-row tiles of a 32-position block are dealt so -- which
// is just the B operand of the second product: the probabilities go from the first
// product to the second without leaving the lane, and a row's maximum, sum and
// rescale are one register for all of the lane's output.
//
// K and V are exact in f16 (4-bit values by the choice of their scales).  q and
// the probabilities enter as a sum of two f16 each, about 22 bits, so the result
// has the accuracy of f32 products at half of f16's matrix rate.  q is scaled by a
// power of two of its row's own, so neither part leaves f16's range.
constexpr uint32_t kUnit = 128;  // positions of a unit of work: 32 for each of a workgroup's 4 waves
// What an item costs besides its units, in units: its q and first K and V come one
// after another, and its sums are joined. Measured at 64 sequences of 820
// to 8192 positions and 8 heads: 90.3 us with none, 86.6 with two or four, 88.6 with eight.
constexpr uint32_t kItem = 2;

// Over the four lanes of a query row (lane % 16): a swap gives a lane both its own
// and the other's value, in some order.
template <class F>
__device__ __forceinline__ float over_q(float x, const F& f) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const uint32_t a0 = a[0], a1 = a[1];
    const uint32_t v = __builtin_bit_cast(uint32_t, f(__builtin_bit_cast(float, a0), __builtin_bit_cast(float, a1)));
    const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    const uint32_t b0 = b[0], b1 = b[1];
    return f(__builtin_bit_cast(float, b0), __builtin_bit_cast(float, b1));
}
__device__ __forceinline__ float max_over_q(float x) {
    return over_q(x, [](float y, float z) { return __builtin_fmaxf(y, z); });
}
__device__ __forceinline__ float sum_over_q(float x) {
    return over_q(x, [](float y, float z) { return y + z; });
}

// Eight 4-bit values of a word as f16, in the order nibble 0, 4, 1, 5, 2, 6, 3, 7.
// A nibble in mantissa bits 9..6 of 16.0 is 16 + n; (16 + n) d - 24 d is exact.
__device__ __forceinline__ v8h decode8(uint32_t w, v2h d0, v2h d1, v2h d2, v2h d3) {
    // one scalar and one vector register: v_and_or_b32 takes no two literals
    uint32_t mask = 0x03c003c0u, sixteen = 0x4c004c00u;
    asm("" : "+s"(mask));
    asm("" : "+v"(sixteen));
    const auto at = [&](uint32_t x) { return __builtin_bit_cast(v2h, (x & mask) | sixteen); };
    const v2h x0 = at(w << 6), x1 = at(w << 2), x2 = at(w >> 2), x3 = at(w >> 6);
    const v2h c = {static_cast<_Float16>(-24.0f), static_cast<_Float16>(-24.0f)};
    const v2h y0 = __builtin_elementwise_fma(x0, d0, c * d0), y1 = __builtin_elementwise_fma(x1, d1, c * d1);
    const v2h y2 = __builtin_elementwise_fma(x2, d2, c * d2), y3 = __builtin_elementwise_fma(x3, d3, c * d3);
    return v8h{y0.x, y0.y, y1.x, y1.y, y2.x, y2.y, y3.x, y3.y};
}

// The operands of 32 positions as loaded.
template <int HD, bool Q4>
struct KRaw {
    uint32_t w[2][HD / 32][Q4 ? 1 : 4];
    uint32_t d[2][HD / 128 ? HD / 128 : 1];  // a register each: two in one would be waited for where they meet
};
template <int HD, bool Q4>
struct VRaw {
    uint32_t w[HD / 16][Q4 ? 1 : 4];
    v4u d[Q4 ? HD / 64 : 1];
};

// The pages of a 32-position block: one, or two of 16 positions.  -1: none.
struct Pages {
    int32_t a, b;
    __device__ __forceinline__ int32_t of(bool second) const {
        const int32_t x = a, y = b;
        return second ? y : x;
    }
};

// One for all of the wave, by scalar loads: a vector load here would be waited for with
// all the K and V loads that went out before it.  What the table holds, not looked at
// yet: that waits for it.
__device__ __forceinline__ int32_t entry_at(const Paged& p, uint32_t s, uint32_t pos) {
    const uint32_t i = __builtin_amdgcn_readfirstlane(min(pos >> p.page_shift, p.table_stride - 1));
    typedef const __attribute__((address_space(4))) int32_t* Table;
    return ((Table)(uintptr_t)p.table)[static_cast<size_t>(__builtin_amdgcn_readfirstlane(s)) * p.table_stride + i];
}

__device__ __forceinline__ Pages entries_at(const Paged& p, uint32_t s, uint32_t kb) {
    return {entry_at(p, s, kb), entry_at(p, s, kb + 16)};
}

__device__ __forceinline__ Pages pages_of(const Paged& p, const Pages& e, uint32_t kb) {
    return {static_cast<uint32_t>(e.a) < p.n_pages && kb >> p.page_shift < p.table_stride ? e.a : -1,
            static_cast<uint32_t>(e.b) < p.n_pages && (kb + 16) >> p.page_shift < p.table_stride ? e.b : -1};
}

// K position of matrix row m (0..15) of tile t in a 32-position block.
__device__ __forceinline__ uint32_t k_row(uint32_t m, int t) { return 8 * (m >> 2) + (m & 3) + 4 * t; }

// A lane's addresses in a 32-position block: its K row of tile 0 and its 8 positions
// of V, and their scales.  Tile 1's K row is the fourth on from tile 0's, in the same
// page, so all of a block's loads are these and constants.
struct Spots {
    const uint8_t *k, *ks, *v, *vs;
};

template <int HD, bool Q4>
__device__ __forceinline__ Spots spots_of(const Paged& p, const Pages& g, uint32_t h, uint32_t kb, uint32_t lane) {
    const uint32_t m = lane & 15, q = lane >> 4, page = 1u << p.page_shift;
    const size_t a = head_base<HD, Q4>(p, max(g.a, 0), h), b = head_base<HD, Q4>(p, max(g.b, 0), h);
    const size_t kh = m >= 8 ? b : a, vh = q >= 2 ? b : a;
    const uint32_t row = (kb + k_row(m, 0)) & (page - 1), grp = ((kb + 8 * q) & (page - 1)) >> 3;
    Spots s;
    if constexpr (!Q4) {
        s.k = p.k + (kh + row * (HD * 2) + 16 * q);
        s.v = p.v + (vh + (grp * HD + m) * 16);
        s.ks = s.vs = nullptr;
    } else {
        s.k = p.k + (kh + row * (HD / 2) + (HD == 64 ? 8 : 16) * q);
        s.ks = p.k + (kh + page * (HD / 2) + row * (HD / 16) + (HD == 64 ? 2 * (q >> 1) : 2 * q));
        s.v = p.v + (vh + (grp * HD + 4 * m) * 4);
        s.vs = p.v + (vh + page * (HD / 2) + (grp * (HD / 32) + (m >> 3)) * 16);
    }
    return s;
}

template <int HD, bool Q4>
__device__ __forceinline__ void load_k(const Spots& s, KRaw<HD, Q4>& r) {
#pragma unroll
    for (int t = 0; t < 2; t++) {
        if constexpr (!Q4) {
#pragma unroll
            for (int i = 0; i < HD / 32; i++)
                *reinterpret_cast<v4u*>(r.w[t][i]) = *reinterpret_cast<const v4u*>(s.k + t * (8 * HD) + 64 * i);
        } else if constexpr (HD == 64) {  // half of block q / 2
            const v2u x = *reinterpret_cast<const v2u*>(s.k + t * (2 * HD));
            r.w[t][0][0] = x.x;
            r.w[t][1][0] = x.y;
            r.d[t][0] = *reinterpret_cast<const uint16_t*>(s.ks + t * (HD / 4));
        } else {
#pragma unroll
            for (int b = 0; b < HD / 128; b++) {  // block q + 4 b
                const v4u x = *reinterpret_cast<const v4u*>(s.k + t * (2 * HD) + 64 * b);
                r.w[t][4 * b][0] = x.x;
                r.w[t][4 * b + 1][0] = x.y;
                r.w[t][4 * b + 2][0] = x.z;
                r.w[t][4 * b + 3][0] = x.w;
                r.d[t][b] = *reinterpret_cast<const uint16_t*>(s.ks + t * (HD / 4) + 8 * b);
            }
        }
    }
}

template <int HD, bool Q4>
__device__ __forceinline__ v8h k_operand(const KRaw<HD, Q4>& r, int t, int i) {
    if constexpr (!Q4) {
        return __builtin_bit_cast(v8h, *reinterpret_cast<const v4u*>(r.w[t][i]));
    } else {
        const _Float16 d = __builtin_bit_cast(_Float16, static_cast<uint16_t>(r.d[t][HD == 64 ? 0 : i / 4]));
        const v2h dd = {d, d};
        return decode8(r.w[t][i][0], dd, dd, dd, dd);
    }
}

// The dim of slot j (0..7) of k-step i for lane quarter q: the order in which
// load_k's operands hold the head's dims.
template <int HD, bool Q4>
__device__ __forceinline__ constexpr uint32_t k_dim(uint32_t q, int i, int j) {
    if (!Q4) return 32 * i + 8 * q + j;
    // word w of block b: nibbles 0, 4, 1, 5, 2, 6, 3, 7; nibble n of a GGUF block word is
    // element 4 w + n / 2 + 16 (n % 2)
    const uint32_t b = HD == 64 ? q >> 1 : q + 4 * (i / 4), w = HD == 64 ? 2 * (q & 1) + i : i % 4;
    const uint32_t n = (j >> 1) + 4 * (j & 1);
    return 32 * b + 4 * w + n / 2 + 16 * (n & 1);
}

template <int HD, bool Q4>
__device__ __forceinline__ void load_v(const Spots& s, VRaw<HD, Q4>& r) {
    if constexpr (!Q4) {
#pragma unroll
        for (int c = 0; c < HD / 16; c++) *reinterpret_cast<v4u*>(r.w[c]) = *reinterpret_cast<const v4u*>(s.v + 256 * c);
    } else {
#pragma unroll
        for (int b = 0; b < HD / 64; b++) {  // dims 64 b + 4 m + {0, 1, 2, 3}
            const v4u x = *reinterpret_cast<const v4u*>(s.v + 256 * b);
            r.w[4 * b][0] = x.x;
            r.w[4 * b + 1][0] = x.y;
            r.w[4 * b + 2][0] = x.z;
            r.w[4 * b + 3][0] = x.w;
            r.d[b] = *reinterpret_cast<const v4u*>(s.vs + 32 * b);
        }
    }
}

// The dim of matrix row m of V's tile c.
template <int HD, bool Q4>
__device__ __forceinline__ constexpr uint32_t v_dim(int c, uint32_t m) {
    return Q4 ? 64 * (c / 4) + 4 * m + c % 4 : 16 * c + m;
}

template <int HD, bool Q4>
__device__ __forceinline__ v8h v_operand(const VRaw<HD, Q4>& r, int c) {
    if constexpr (!Q4) {
        return __builtin_bit_cast(v8h, *reinterpret_cast<const v4u*>(r.w[c]));
    } else {
        // (a bit cast of a vector's element takes the first one's bits: each goes through a scalar)
        const uint32_t d0 = r.d[c / 4].x, d1 = r.d[c / 4].y, d2 = r.d[c / 4].z, d3 = r.d[c / 4].w;
        return decode8(r.w[c][0], __builtin_bit_cast(v2h, d0), __builtin_bit_cast(v2h, d1),
                       __builtin_bit_cast(v2h, d2), __builtin_bit_cast(v2h, d3));
    }
}

// V's operands with the positions outside [lo, hi) zero: what lies there may be
// anything, and 0 times a NaN is a NaN.
template <int HD, bool Q4>
__device__ __forceinline__ void clear_v(VRaw<HD, Q4>& r, int32_t at, int32_t lo, int32_t hi) {
    uint32_t keep[4];  // by pair of positions
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int32_t a = at + 2 * i;
        keep[i] = (a >= lo && a < hi ? 0xffffu : 0u) | (a + 1 >= lo && a + 1 < hi ? 0xffff0000u : 0u);
    }
    const v4u k = {keep[0], keep[1], keep[2], keep[3]};
    if constexpr (Q4) {  // a scale of 0 makes the value 0
#pragma unroll
        for (int b = 0; b < HD / 64; b++) r.d[b] &= k;
    } else {
#pragma unroll
        for (int c = 0; c < HD / 16; c++) *reinterpret_cast<v4u*>(r.w[c]) &= k;
    }
}

// A wave's 16 query rows: the operand parts of q and the factor that takes a
// product of theirs to the softmax's exponent of two.
template <int HD>
struct QTile {
    v8h hi[HD / 32], lo[HD / 32];
    float factor;
};

template <int HD, bool Q4>
__device__ __forceinline__ void load_q(QTile<HD>& qt, const float* row, uint32_t q, float scale) {
    // the lane's dims, in runs of four
    float x[HD / 32][8];
    float mx = 0.0f;
#pragma unroll
    for (int i = 0; i < HD / 32; i++) {
        v4f run[2];
        if constexpr (Q4) {
            // two runs of a word: elements 4 w .. 4 w + 3 and 16 on, in the order of k_dim
            const uint32_t d = k_dim<HD, Q4>(q, i, 0);
            run[0] = *reinterpret_cast<const v4f*>(row + d);
            run[1] = *reinterpret_cast<const v4f*>(row + d + 16);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int nib = (j >> 1) + 4 * (j & 1);
                x[i][j] = run[nib & 1][nib / 2];
            }
        } else {
            run[0] = *reinterpret_cast<const v4f*>(row + 32 * i + 8 * q);
            run[1] = *reinterpret_cast<const v4f*>(row + 32 * i + 8 * q + 4);
#pragma unroll
            for (int j = 0; j < 8; j++) x[i][j] = run[j / 4][j % 4];
        }
#pragma unroll
        for (int j = 0; j < 8; j++) mx = __builtin_fmaxf(mx, __builtin_fabsf(x[i][j]));
    }
    mx = max_over_q(mx);
    // the row's largest to [2^13, 2^14); a row of zeros, infinities or NaN stays as it is
    int e = 0;
    if (mx > 0.0f && mx < INFINITY) e = 14 - __builtin_amdgcn_frexp_expf(mx);
    // the factor is positive: a negative scale's sign goes to q
    // (and it is not 0, which a masked -inf must not meet)
    qt.factor = __builtin_fmaxf(ldexpf(__builtin_fabsf(scale), -e), 0x1p-126f);
    const float sign = scale < 0.0f ? -1.0f : 1.0f;
#pragma unroll
    for (int i = 0; i < HD / 32; i++)
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float y = ldexpf(x[i][j] * sign, e);
            const _Float16 a = static_cast<_Float16>(y);
            qt.hi[i][j] = a;
            qt.lo[i][j] = static_cast<_Float16>(y - static_cast<float>(a));
        }
}

// The running softmax of a wave's 16 rows over blocks of 32 positions.
// Probabilities are 2^(s - m + kLift) with m the maximum when it last moved: it
// moves only when a score exceeds it by kSlack, so that the output is rescaled
// rarely; kLift + kSlack keep the largest below f16's 65504 and put the smallest
// that the pair of f16 resolves 2^-30 below a weight of 1.
constexpr float kLift = 6.0f, kSlack = 8.0f;

template <int HD>
struct Soft {
    float m, l;  // l: this lane's share of the row's sum
    v4f o[HD / 16];
};

template <int HD>
__device__ __forceinline__ void soft_clear(Soft<HD>& st) {
    st.m = -INFINITY;
    st.l = 0.0f;
#pragma unroll
    for (int c = 0; c < HD / 16; c++) st.o[c] = v4f{0, 0, 0, 0};
}

template <int HD, bool Q4>
__device__ __forceinline__ void scores(const KRaw<HD, Q4>& k, const QTile<HD>& qt, v4f s[2]) {
    s[0] = s[1] = v4f{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < HD / 32; i++) {
        const v8h a = k_operand<HD, Q4>(k, 0, i), b = k_operand<HD, Q4>(k, 1, i);
        s[0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qt.hi[i], s[0], 0, 0, 0);
        s[1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(b, qt.hi[i], s[1], 0, 0, 0);
        s[0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qt.lo[i], s[0], 0, 0, 0);
        s[1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(b, qt.lo[i], s[1], 0, 0, 0);
    }
}

// s: products of kT 16-position tiles, -inf where masked; times the row's factor they
// are exponents of two.  Moves the maximum if it has to; returns what the exponents add.
template <int HD, int kT>
__device__ __forceinline__ float soft_base(Soft<HD>& st, const v4f (&s)[kT], float factor) {
    float mx = s[0][0];
#pragma unroll
    for (int i = 1; i < 4 * kT; i++) mx = __builtin_fmaxf(mx, s[i / 4][i % 4]);
    mx *= factor;  // of 0 or more, so the largest stays it
    if (__any(mx > st.m + kSlack)) {
        mx = __builtin_fmaxf(max_over_q(mx), st.m);
        const float f = st.m == mx ? 1.0f : __builtin_amdgcn_exp2f(st.m - mx);  // -inf stays with -inf
        st.m = mx;
        st.l *= f;
#pragma unroll
        for (int c = 0; c < HD / 16; c++) st.o[c] *= f;
    }
    return kLift - (st.m == -INFINITY ? 0.0f : st.m);
}

// -1 that is no constant: with one what a first part leaves would become a conversion
// and a difference.
__device__ __forceinline__ float minus_one() {
    float x = -1.0f;
    asm("" : "+v"(x));
    return x;
}

// The two parts of P of two products, to elements i and i + 1; returns their sum.
__device__ __forceinline__ float soft_pair(float s0, float s1, float factor, float base, float minus, v8h& hi, v8h& lo, int i) {
    const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s0, factor, base));
    const float f = __builtin_amdgcn_exp2f(__builtin_fmaf(s1, factor, base));
    // the first part towards zero, two values an instruction; what it leaves is exact
    // and goes to the second part: 21 bits and more together
    const v2h x = __builtin_bit_cast(v2h, __builtin_amdgcn_cvt_pkrtz(e, f));
    const v2h y = __builtin_bit_cast(v2h, __builtin_amdgcn_cvt_pkrtz(__builtin_fmaf(static_cast<float>(x.x), minus, e),
                                                                      __builtin_fmaf(static_cast<float>(x.y), minus, f)));
    hi[i] = x.x;
    hi[i + 1] = x.y;
    lo[i] = y.x;
    lo[i + 1] = y.y;
    return e + f;
}

// A tile's second product waits for its first; the next tile's operand is decoded between.
template <int HD, bool Q4>
__device__ __forceinline__ void values(Soft<HD>& st, const VRaw<HD, Q4>& v, const v8h& hi, const v8h& lo) {
    v8h before = v_operand<HD, Q4>(v, 0);
    st.o[0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(before, hi, st.o[0], 0, 0, 0);
#pragma unroll
    for (int c = 1; c < HD / 16; c++) {
        const v8h a = v_operand<HD, Q4>(v, c);
        st.o[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, hi, st.o[c], 0, 0, 0);
        st.o[c - 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(before, lo, st.o[c - 1], 0, 0, 0);
        before = a;
    }
    st.o[HD / 16 - 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(before, lo, st.o[HD / 16 - 1], 0, 0, 0);
}

// Sequence s in units of work: its rows in tiles of 16 (rows x heads of a kv
// head's group), per tile and kv head the positions [lo, end) in units.
struct SeqWork {
    int32_t row0, len, end, first;  // rows, positions with them, position of the first row
    int32_t lo;                     // first position any row sees, down to a multiple of 32
    uint32_t tiles, units;          // per tile and head
};

// Positions that a sequence can have: what its pages hold, and no more than leaves the
// ends of the blocks and units around the last one below 2^31.  A row past them sees
// positions that are nowhere: it becomes NaN.
__device__ __forceinline__ uint64_t capacity(const Paged& p) {
    return min(static_cast<uint64_t>(p.table_stride) << p.page_shift, static_cast<uint64_t>((1u << 31) - 2 * kUnit));
}

__device__ __forceinline__ SeqWork seq_work(const AttnArgs& a, int32_t row0, int32_t row1, int32_t kv) {
    SeqWork w;
    const int32_t n = static_cast<int32_t>(a.p.n_tokens);
    w.row0 = min(max(row0, 0), n);
    w.len = max(min(row1, n) - w.row0, 0);
    w.first = static_cast<int32_t>(static_cast<uint32_t>(kv) - static_cast<uint32_t>(w.len));
    w.end = static_cast<int32_t>(min(static_cast<uint64_t>(max(kv, 0)), capacity(a.p)));
    const int32_t lo = a.window && w.first >= static_cast<int32_t>(a.window) ? w.first - static_cast<int32_t>(a.window) + 1 : 0;
    w.lo = min(lo, w.end) & ~31;
    w.tiles = (static_cast<uint32_t>(w.len) * a.group + 15) / 16;
    w.units = max((static_cast<uint32_t>(w.end - w.lo) + kUnit - 1) / kUnit, 1u);
    return w;
}

__device__ __forceinline__ SeqWork seq_work(const AttnArgs& a, uint32_t s) {
    return seq_work(a, a.p.q_start[s], a.p.q_start[s + 1], a.p.kv_len[s]);
}

// The batch's lengths, and prefix sums of its sequences' units (all tiles and heads).
struct Units {
    uint32_t prefix[kMaxSeqs + 1];
    int32_t row0[kMaxSeqs], row1[kMaxSeqs], kv[kMaxSeqs];
    uint32_t sums[4];
};

// Fills them; returns the total.  A batch whose sequences' rows are in order has fewer
// than kUnitsMost (the host's check); sums end there, and one that reaches it is left
// out whole: its row starts are out of order.
constexpr uint32_t kUnitsMost = 0x7fffffffu;

__device__ __forceinline__ uint32_t scan_units(const AttnArgs& a, Units& un) {
    const uint32_t tid = threadIdx.x, lane = tid & (kWave - 1), wid = tid / kWave;
    uint32_t base = 0;
    for (uint32_t b = 0; b < a.p.n_seqs; b += 256) {
        uint32_t x = 0;
        if (b + tid < a.p.n_seqs) {
            const int32_t row0 = a.p.q_start[b + tid], row1 = a.p.q_start[b + tid + 1], kv = a.p.kv_len[b + tid];
            un.row0[b + tid] = row0;
            un.row1[b + tid] = row1;
            un.kv[b + tid] = kv;
            const SeqWork w = seq_work(a, row0, row1, kv);
            if (static_cast<uint32_t>(w.len) * a.group <= a.few_rows)
                x = static_cast<uint32_t>(min(static_cast<uint64_t>(w.tiles) * a.p.n_kv * (w.units + kItem), static_cast<uint64_t>(kUnitsMost)));
        }
        uint32_t run = x;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t y = __shfl_up(run, o);
            if (static_cast<int>(lane) >= o) run = min(run + y, kUnitsMost);
        }
        if (lane == 63) un.sums[wid] = run;
        __syncthreads();
        uint32_t before = base, all = 0;
        for (uint32_t i = 0; i < 4; i++) {
            if (i < wid) before = min(before + un.sums[i], kUnitsMost);
            all = min(all + un.sums[i], kUnitsMost);
        }
        if (b + tid < a.p.n_seqs) un.prefix[b + tid] = before + run - x;
        base = min(base + all, kUnitsMost);
        __syncthreads();
    }
    if (tid == 0) un.prefix[a.p.n_seqs] = base;
    __syncthreads();
    return base == kUnitsMost ? 0 : base;
}

// Where unit u lies.
struct Place {
    uint32_t s, tile, h, unit;  // within the item (s, tile, h): its cost, then its units
};

__device__ __forceinline__ Place place_of(const AttnArgs& a, const Units& un, uint32_t u, SeqWork& w) {
    uint32_t lo = 0, hi = a.p.n_seqs;  // un.prefix[lo] <= u < un.prefix[hi]
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (un.prefix[mid] <= u) lo = mid;
        else hi = mid;
    }
    Place at;
    at.s = __builtin_amdgcn_readfirstlane(lo);
    w = seq_work(a, un.row0[at.s], un.row1[at.s], un.kv[at.s]);
    const uint32_t r = u - un.prefix[at.s], item = r / (w.units + kItem);
    at.unit = __builtin_amdgcn_readfirstlane(r % (w.units + kItem));
    at.tile = __builtin_amdgcn_readfirstlane(item / a.p.n_kv);
    at.h = __builtin_amdgcn_readfirstlane(item % a.p.n_kv);
    return at;
}

// Units of each workgroup: all alike.
__device__ __forceinline__ uint32_t share_of(uint32_t total, uint32_t grid) { return (total + grid - 1) / grid; }

// A partial result: 16 rows of hd sums, then the rows' maxima and sums.
template <int HD>
__device__ __forceinline__ float* part_slot(const AttnArgs& a, uint32_t slot) {
    return a.part + static_cast<size_t>(slot) * (16 * (HD + 2));
}

// A partial result is read by a workgroup on another part of the chip while its
// kernel runs: stores and loads of agent scope go past the caches that they do not
// share.
__device__ __forceinline__ void put_part(float* p, float v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float get_part(const float* p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The shares b0 .. b1 of an item added in order, and its rows written: kE values a
// thread, kP shares at a time, all of their loads in flight at once.
struct Join {
    float m[16][16], l[16][16];  // of the shares at hand, then their factors in m
    float top[16], sum[16], old[16];
};

template <int HD, int kE, int kP>
__device__ __forceinline__ void join_parts(const AttnArgs& a, const SeqWork& w, const Place& at, uint32_t b0, uint32_t b1,
                                           uint32_t tile_rows, Join& jn) {
    const uint32_t tid = threadIdx.x, n = tile_rows * HD;
    const auto part = [&](uint32_t b) { return part_slot<HD>(a, 2 * b + (b == b0 ? 1 : 0)); };
    float o[kE];
#pragma unroll
    for (int k = 0; k < kE; k++) o[k] = 0.0f;
    if (tid < 16) {
        jn.top[tid] = -INFINITY;
        jn.sum[tid] = 0.0f;
    }
    for (uint32_t b = b0; b <= b1; b += kP) {
        float v[kE][kP];
#pragma unroll
        for (int j = 0; j < kP; j++) {
            const float* p = part(min(b + j, b1));
#pragma unroll
            for (int k = 0; k < kE; k++) v[k][j] = get_part(p + min(tid + 256 * k, n - 1));
        }
        __syncthreads();
        for (uint32_t i = tid; i < 16 * kP; i += 256) {
            const uint32_t j = i / 16, row = i % 16;
            const bool has = b + j <= b1 && row < tile_rows;
            const float* p = part(min(b + j, b1)) + 16 * HD + min(row, tile_rows - 1);
            const float m = get_part(p), l = get_part(p + 16);
            jn.m[j][row] = has ? m : -INFINITY;
            jn.l[j][row] = has ? l : 0.0f;
        }
        __syncthreads();
        if (tid < 16) {
            const float was = jn.top[tid];
            float top = was;
#pragma unroll
            for (int j = 0; j < kP; j++) top = __builtin_fmaxf(top, jn.m[j][tid]);
            const float old = was == top ? 1.0f : __builtin_amdgcn_exp2f(was - top);
            float sum = jn.sum[tid] * old;
#pragma unroll
            for (int j = 0; j < kP; j++) {
                // without a maximum: nothing seen, or a sum of NaN
                const float m = jn.m[j][tid], l = jn.l[j][tid];
                const float g = m == -INFINITY ? (l == 0.0f ? 0.0f : 1.0f) : __builtin_amdgcn_exp2f(m - top);
                sum += l * g;
                jn.m[j][tid] = g;
            }
            jn.top[tid] = top;
            jn.sum[tid] = sum;
            jn.old[tid] = old;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kE; k++) {
            const uint32_t row = min((tid + 256 * k) / HD, 15u);
            o[k] *= jn.old[row];
#pragma unroll
            for (int j = 0; j < kP; j++)
                if (b + j <= b1) o[k] += v[k][j] * jn.m[j][row];
        }
    }
#pragma unroll
    for (int k = 0; k < kE; k++) {
        const uint32_t e = tid + 256 * k, row = e / HD, rr = 16 * at.tile + row;
        if (e >= n) continue;
        const float sum = jn.sum[row];
        const uint32_t tk = rr / a.group, hd = at.h * a.group + rr % a.group;
        a.out[(static_cast<size_t>(w.row0 + tk) * a.n_heads + hd) * HD + e % HD] = sum != 0.0f ? o[k] / sum : o[k];
    }
}

// Attention by few rows: the units of all sequences are laid end to end and cut
// into equal shares, one a workgroup, whatever the lengths are.  Within an item (a
// tile of 16 rows and its kv head) the four waves take every fourth 32 positions, and
// their sums are joined through LDS.  An item that shares cut is joined by the last
// of its workgroups to be done: each puts its sums into memory, waits until they are
// there and counts itself; the counter of an item is that of its first share, and is
// 0 again when the item is done.  The join adds the shares in their order, so results
// do not depend on which workgroup does it.
template <int HD, bool Q4>
__device__ __forceinline__ void attend_few(const AttnArgs& a) {
    __shared__ Units un;
    __shared__ float sm_m[4][16], sm_l[4][16];
    __shared__ __attribute__((aligned(16))) float sm_o[4][16][HD + 4];
    __shared__ Join jn;
    __shared__ uint32_t done;
    const uint32_t tid = threadIdx.x, lane = tid & (kWave - 1), wid = __builtin_amdgcn_readfirstlane(tid / kWave);
    const uint32_t n = lane & 15, q = lane >> 4;
    const uint32_t total = scan_units(a, un);
    const uint32_t share = share_of(total, gridDim.x);  // blockIdx.x of them: less than total + gridDim.x^2
    const int32_t win = static_cast<int32_t>(a.window);
    uint32_t u = blockIdx.x * share;
    const uint32_t u_end = min(u + share, total);
    while (u < u_end) {
        SeqWork w;
        Place at = place_of(a, un, u, w);
        const uint32_t item = u - at.unit, end = min(item + kItem + w.units, u_end);
        const uint32_t first = item + kItem;  // the item's first unit
        at.unit = max(u, first) - first;
        u = end;
        if (end <= first) break;  // the share ends in the item's cost: the next one has its units
        const uint32_t units = end - first - at.unit;
        const uint32_t rows = static_cast<uint32_t>(w.len) * a.group;
        const uint32_t r = 16 * at.tile + n;
        const bool live = r < rows;  // the others are computed and dropped
        const uint32_t tok = live ? r / a.group : 0, head = at.h * a.group + (live ? r % a.group : 0);
        const int32_t pos = w.first + static_cast<int32_t>(tok);
        const int32_t hi = pos + 1, lo = win && hi > win ? hi - win : 0;
        // what any row of the tile sees and what all of them see; rows are in order of position
        const uint32_t tok_b = (min(16 * at.tile + 16, rows) - 1) / a.group;
        const int32_t hi_a = w.first + static_cast<int32_t>(16 * at.tile / a.group) + 1;
        const int32_t hi_b = w.first + static_cast<int32_t>(tok_b) + 1;
        const int32_t tile_hi = min(hi_b, w.end);
        const int32_t tile_lo = win && hi_a > win ? hi_a - win : 0, all_lo = win && hi_b > win ? hi_b - win : 0;
        // this wave's blocks: every 128 positions from kb0, those that any row sees
        const int32_t kb0 = w.lo + static_cast<int32_t>(at.unit * kUnit + 32 * wid);
        const int32_t skip = max(tile_lo - 31 - kb0, 0);
        const uint32_t i0 = (static_cast<uint32_t>(skip) + kUnit - 1) / kUnit;
        const uint32_t i1 = tile_hi > kb0 ? min(units, (static_cast<uint32_t>(tile_hi - kb0) + kUnit - 1) / kUnit) : 0;
        // The next block's K is on its way from the moment that this one's scores are
        // done, its V from when this one's is used: no register waits for its turn.  (A
        // second set of them, loaded a block ahead, measured 93 us where this takes 90, at
        // 64 sequences of 820 to 8192 positions and 8 heads; f16, 6 of up to 32001: 119 and
        // 107.)  Past the last block that one is loaded again: loads under a condition
        // would be waited for where it ends.
        KRaw<HD, Q4> kr;
        VRaw<HD, Q4> vr;
        Pages pg = {-1, -1}, ahead = {-1, -1};
        QTile<HD> qt;
        Soft<HD> st;
        const auto kb_of = [&](uint32_t i) { return static_cast<uint32_t>(kb0) + kUnit * min(i, i1 - 1); };
        if (i0 < i1) ahead = entries_at(a.p, at.s, kb_of(i0));
        load_q<HD, Q4>(qt, a.q + (static_cast<size_t>(w.row0 + tok) * a.n_heads + head) * HD, q, a.scale);
        soft_clear<HD>(st);
        if (pos >= 0 && static_cast<uint64_t>(pos) >= capacity(a.p)) st.l = __builtin_nanf("");
        if (i0 < i1) {
            pg = pages_of(a.p, ahead, kb_of(i0));
            const Spots spots = spots_of<HD, Q4>(a.p, pg, at.h, kb_of(i0), lane);
            load_k<HD, Q4>(spots, kr);
            load_v<HD, Q4>(spots, vr);
            ahead = entries_at(a.p, at.s, kb_of(i0 + 1));
        }
        for (uint32_t i = i0; i < i1; i++) {
            const int32_t kb = static_cast<int32_t>(kb_of(i));
            v4f s[2];
            scores<HD, Q4>(kr, qt, s);
            const Pages next = pages_of(a.p, ahead, kb_of(i + 1));
            const Spots spots = spots_of<HD, Q4>(a.p, next, at.h, kb_of(i + 1), lane);
            load_k<HD, Q4>(spots, kr);
            ahead = entries_at(a.p, at.s, kb_of(i + 2));
            if (kb < all_lo || kb + 32 > min(hi_a, w.end) || pg.a < 0 || pg.b < 0) {
                const int32_t p0 = kb + static_cast<int32_t>(8 * q);
                const bool no_page = pg.of(q >= 2) < 0;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int32_t x = p0 + e;
                    float v = s[e / 4][e % 4];
                    if (no_page) v = __builtin_nanf("");
                    s[e / 4][e % 4] = x < lo || x >= hi ? -INFINITY : v;
                }
                clear_v<HD, Q4>(vr, p0, tile_lo, no_page ? tile_lo : tile_hi);
            }
            v8h ph, pl;
            const float base = soft_base<HD, 2>(st, s, qt.factor), minus = minus_one();
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; e += 2) sum += soft_pair(s[e / 4][e % 4], s[e / 4][e % 4 + 1], qt.factor, base, minus, ph, pl, e);
            st.l += sum;
            values<HD, Q4>(st, vr, ph, pl);
            load_v<HD, Q4>(spots, vr);
            pg = next;
        }
        // join the waves
        const float l = sum_over_q(st.l);
        if (q == 0) {
            sm_m[wid][n] = st.m;
            sm_l[wid][n] = l;
        }
#pragma unroll
        for (int c = 0; c < HD / 16; c++)
#pragma unroll
            for (int i = 0; i < 4; i++) sm_o[wid][n][v_dim<HD, Q4>(c, 4 * q + i)] = st.o[c][i];
        __syncthreads();
        const bool whole = units == w.units;
        float* slot = part_slot<HD>(a, 2 * blockIdx.x + (at.unit == 0 ? 1 : 0));
        const uint32_t tile_rows = min(rows - 16 * at.tile, 16u);
        for (uint32_t e = tid; e < tile_rows * HD / 4; e += 256) {
            const uint32_t row = e / (HD / 4), d = 4 * (e % (HD / 4)), rr = 16 * at.tile + row;
            float m = sm_m[0][row];
            for (int i = 1; i < 4; i++) m = __builtin_fmaxf(m, sm_m[i][row]);
            float sum = 0.0f;
            v4f o = {0, 0, 0, 0};
            for (int i = 0; i < 4; i++) {
                const float f = sm_m[i][row] == -INFINITY ? (sm_l[i][row] == 0.0f ? 0.0f : 1.0f)
                                                          : __builtin_amdgcn_exp2f(sm_m[i][row] - m);
                sum += sm_l[i][row] * f;
                o += *reinterpret_cast<const v4f*>(&sm_o[i][row][d]) * f;
            }
            if (whole) {
                if (sum != 0.0f) o /= sum;  // a row that sees nothing: 0
                const uint32_t tk = rr / a.group, hd = at.h * a.group + rr % a.group;
                *reinterpret_cast<v4f*>(a.out + (static_cast<size_t>(w.row0 + tk) * a.n_heads + hd) * HD + d) = o;
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++) put_part(slot + row * HD + d + i, o[i]);
                if (d == 0) {
                    put_part(slot + 16 * HD + row, m);
                    put_part(slot + 16 * HD + 16 + row, sum);
                }
            }
        }
        if (!whole) {
            const uint32_t b0 = first / share, b1 = (first + w.units - 1) / share;
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's part is in memory
            __syncthreads();                                   // and every wave's
            if (tid == 0)
                done = __hip_atomic_fetch_add(a.counts + b0, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == b1 - b0;
            __syncthreads();
            if (done) {
                if (tile_rows * HD <= 512) join_parts<HD, 2, 16>(a, w, at, b0, b1, tile_rows, jn);
                else join_parts<HD, HD / 16, 4>(a, w, at, b0, b1, tile_rows, jn);
                if (tid == 0) __hip_atomic_store(a.counts + b0, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
        }
        __syncthreads();
    }
}

// ---- many rows ----
//
// A workgroup owns 16 kRt rows a wave of one kv head (the rows of consecutive
// tokens, each with its group of q heads) and walks the positions they see, 32 kBlocks
// at a time: the waves load and decode a share each of the K and V operands into LDS,
// in the lanes' order, while all multiply from the other buffer.  A workgroup of eight
// waves decodes half as often as one of four.  With heads of 256 a tile has 64 rows;
// kHalved: two waves share 16 of them, each with one block of a stage, and join their
// sums at the end.
//
// What bounds it is matrix and vector issue in turn, 59% and 32% of the CUs' cycles: the
// two parts of q and of P make four products of what f16 alone would take two of, and those
// run at 1.21 PFLOP/s where a library product of two 16384 x 16384 matrices reaches 1.32
// here (2048 rows of 32 q and 8 kv heads of 128 over 8000 positions, q4_0: 387 us).
template <int HD, bool kHalved = false>
struct Many {
    static constexpr int kRt = HD == 256 ? 1 : 2;      // tiles of 16 rows a wave
    static constexpr int kBlocks = HD == 256 && !kHalved ? 1 : 2;  // 32-position blocks a stage
    static constexpr uint32_t kWaves = HD == 128 || kHalved ? 8 : 4;
    static constexpr uint32_t kRowWaves = kHalved ? kWaves / 2 : kWaves;
    static constexpr int kMine = kHalved ? kBlocks / 2 : kBlocks;  // blocks of a stage a wave multiplies
    static constexpr bool kBoth = HD == 256;                       // a wave loads of K and of V
    static constexpr uint32_t kRows = 16 * kRt * kRowWaves;
    static constexpr uint32_t kStage = 32 * kBlocks;
};

template <int HD, int kBlocks>
struct Operands {  // one stage
    v8h k[kBlocks][2][HD / 32][kWave];
    v8h v[kBlocks][HD / 16][kWave];
};

// A wave's share of a stage as loaded: K's or V's four operands of a block, or both
// (hd 128: the first four waves load K's, the others V's; hd 64: the even, the odd ones).
template <int HD, bool Q4>
struct Share {
    static constexpr int kOne = Q4 ? 1 : 4, kV = Many<HD>::kBoth ? kOne : 0;  // V's first
    v4u w[kV + kOne];
    v4u vd;
    uint32_t kd;
    Pages g;
    uint32_t kb;
};

template <int HD>
struct Job {  // which: block, K tile, 4-operand run of K and of V
    uint32_t blk, t, kb, vb;
    bool k, v;
};

template <int HD>
__device__ __forceinline__ Job<HD> job_of(uint32_t w) {
    if constexpr (HD == 256) return {w >> 2, w & 1, w >> 1 & 1, w & 3, true, true};  // (four waves: block 0)
    if constexpr (HD == 128) return {w >> 1 & 1, w & 1, 0, w & 1, w < 4, w >= 4};
    return {w >> 1, 0, 0, 0, (w & 1) == 0, (w & 1) != 0};
}

template <int HD, bool Q4>
__device__ __forceinline__ void share_load(const Paged& p, const Job<HD>& job, uint32_t h, uint32_t lane,
                                           Share<HD, Q4>& r) {
    const uint32_t m = lane & 15, q = lane >> 4, page = 1u << p.page_shift;
    const size_t b0 = head_base<HD, Q4>(p, max(r.g.a, 0), h), b1 = head_base<HD, Q4>(p, max(r.g.b, 0), h);
    const uint8_t* kbase = p.k + (m >= 8 ? b1 : b0);
    const uint8_t* vbase = p.v + (q >= 2 ? b1 : b0);
    const uint32_t grp = ((r.kb + 8 * q) & (page - 1)) >> 3;
    if (job.k) {
        const uint32_t off = (r.kb + k_row(m, job.t)) & (page - 1);
        if constexpr (HD == 64) {
            const uint32_t off1 = (r.kb + k_row(m, 1)) & (page - 1);
            if constexpr (Q4) {
                const v2u x = *reinterpret_cast<const v2u*>(kbase + off * 32 + 8 * q);
                const v2u y = *reinterpret_cast<const v2u*>(kbase + off1 * 32 + 8 * q);
                r.w[0] = v4u{x.x, x.y, y.x, y.y};
                const uint16_t* sc = reinterpret_cast<const uint16_t*>(kbase + page * 32) + (q >> 1);
                r.kd = sc[off * 2] | static_cast<uint32_t>(sc[off1 * 2]) << 16;
            } else {
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    r.w[i] = *reinterpret_cast<const v4u*>(kbase + off * 128 + 64 * i + 16 * q);
                    r.w[2 + i] = *reinterpret_cast<const v4u*>(kbase + off1 * 128 + 64 * i + 16 * q);
                }
            }
        } else if constexpr (Q4) {
            r.w[0] = *reinterpret_cast<const v4u*>(kbase + off * (HD / 2) + 16 * q + 64 * job.kb);
            r.kd = reinterpret_cast<const uint16_t*>(kbase + page * (HD / 2))[off * (HD / 32) + q + 4 * job.kb];
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
                r.w[i] = *reinterpret_cast<const v4u*>(kbase + off * (HD * 2) + 64 * (4 * job.kb + i) + 16 * q);
        }
    }
    if (job.v) {
        if constexpr (Q4) {
            r.w[r.kV] = *reinterpret_cast<const v4u*>(vbase + (grp * HD + 64 * job.vb + 4 * m) * 4);
            r.vd = reinterpret_cast<const v4u*>(vbase + page * (HD / 2))[grp * (HD / 32) + 2 * job.vb + (m >> 3)];
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
                r.w[r.kV + i] =
                    *reinterpret_cast<const v4u*>(vbase + (grp * HD + 16 * (4 * job.vb + i) + m) * 16);
        }
    }
}

// The share decoded into the stage's operands.  `edge`: positions outside [lo, hi)
// or without a page may be among them: their V becomes 0, a K without a page NaN.
template <int HD, bool Q4, int kBlocks>
__device__ __forceinline__ void share_store(const Job<HD>& job, Share<HD, Q4>& r, Operands<HD, kBlocks>& to, uint32_t lane,
                                            int32_t lo, int32_t hi) {
    const uint32_t m = lane & 15, q = lane >> 4;
    const bool edge = static_cast<int32_t>(r.kb) < lo || static_cast<int32_t>(r.kb) + 32 > hi || r.g.a < 0 || r.g.b < 0;
    v4u keep = {~0u, ~0u, ~0u, ~0u};
    bool no_k = false;
    if (edge) {
        no_k = r.g.of(m >= 8) < 0;
        const int32_t at = static_cast<int32_t>(r.kb + 8 * q), end = r.g.of(q >= 2) < 0 ? lo : hi;
        uint32_t x[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int32_t a = at + 2 * i;
            x[i] = (a >= lo && a < end ? 0xffffu : 0u) | (a + 1 >= lo && a + 1 < end ? 0xffff0000u : 0u);
        }
        keep = v4u{x[0], x[1], x[2], x[3]};
    }
    if (job.k) {
        v8h o[4];
        if constexpr (Q4) {
            const uint32_t x[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w};
            const uint32_t d0 = (r.kd & 0xffffu) * 0x10001u, d1 = HD == 64 ? (r.kd >> 16) * 0x10001u : d0;
            const v2h s0 = __builtin_bit_cast(v2h, d0), s1 = __builtin_bit_cast(v2h, d1);
#pragma unroll
            for (int i = 0; i < 4; i++) o[i] = i < 2 ? decode8(x[i], s0, s0, s0, s0) : decode8(x[i], s1, s1, s1, s1);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) o[i] = __builtin_bit_cast(v8h, r.w[i]);
        }
        const _Float16 nan = __builtin_bit_cast(_Float16, static_cast<uint16_t>(0x7e00));
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (edge && no_k) o[i] = v8h{nan, nan, nan, nan, nan, nan, nan, nan};
            if constexpr (HD == 64) to.k[job.blk][i / 2][i % 2][lane] = o[i];
            else to.k[job.blk][job.t][4 * job.kb + i][lane] = o[i];
        }
    }
    if (job.v) {
        if constexpr (Q4) {
            const v4u d = r.vd & keep;
            const uint32_t d0 = d.x, d1 = d.y, d2 = d.z, d3 = d.w;
            const v4u y = r.w[r.kV];
            const uint32_t x[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int i = 0; i < 4; i++)
                to.v[job.blk][4 * job.vb + i][lane] =
                    decode8(x[i], __builtin_bit_cast(v2h, d0), __builtin_bit_cast(v2h, d1), __builtin_bit_cast(v2h, d2),
                            __builtin_bit_cast(v2h, d3));
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const v4u x = r.w[r.kV + i] & keep;
                to.v[job.blk][4 * job.vb + i][lane] = __builtin_bit_cast(v8h, x);
            }
        }
    }
}

// A workgroup's item: tile `tile` of the rows of sequence s.
struct Item {
    uint32_t s, tile, h, split;
    bool any;
};

// Tiles of the sequences with more than few_rows rows, in order; the grid has one
// workgroup for each (a bound of their number), kv head and split.
template <int HD>
__device__ __forceinline__ Item item_of(const AttnArgs& a, uint32_t block, uint32_t* prefix, uint32_t* sums, SeqWork& w) {
    constexpr uint32_t kRows = Many<HD>::kRows;
    Item it;
    it.h = block % a.p.n_kv;
    it.split = block / a.p.n_kv % a.splits;
    const uint32_t tile = block / a.p.n_kv / a.splits;
    const uint32_t tid = threadIdx.x, lane = tid & (kWave - 1), wid = tid / kWave;
    uint32_t base = 0;
    it.any = false;
    for (uint32_t b = 0; b < a.p.n_seqs; b += blockDim.x) {
        uint32_t x = 0;
        if (b + tid < a.p.n_seqs) {
            const uint32_t rows = static_cast<uint32_t>(seq_work(a, b + tid).len) * a.group;
            x = rows > a.few_rows ? (rows + kRows - 1) / kRows : 0;
        }
        uint32_t run = x;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t y = __shfl_up(run, o);
            if (static_cast<int>(lane) >= o) run += y;
        }
        if (lane == 63) sums[wid] = run;
        __syncthreads();
        uint32_t before = base;
        for (uint32_t i = 0; i < blockDim.x / kWave; i++) {
            if (i < wid) before += sums[i];
            base += sums[i];
        }
        const uint32_t end = before + run;
        if (tile >= end - x && tile < end) {  // one thread at most
            prefix[0] = b + tid;
            prefix[1] = end - 1 - tile;  // the last tile first: it sees the most
        }
        if (tile < base) {
            it.any = true;
            break;
        }
        __syncthreads();
    }
    __syncthreads();
    if (!it.any) return it;
    it.s = __builtin_amdgcn_readfirstlane(prefix[0]);
    it.tile = __builtin_amdgcn_readfirstlane(prefix[1]);
    w = seq_work(a, it.s);
    return it;
}

// The positions that an item's rows see, and its split's part of them.
struct Span {
    int32_t lo, hi;      // of the item
    int32_t from, to;    // of the split
    uint32_t parts;      // splits that have any
};

template <int HD>
__device__ __forceinline__ Span span_of(const AttnArgs& a, const Item& it, const SeqWork& w) {
    constexpr uint32_t kRows = Many<HD>::kRows;
    const uint32_t rows = static_cast<uint32_t>(w.len) * a.group;
    const uint32_t first_tok = kRows * it.tile / a.group, last_tok = (min(kRows * (it.tile + 1), rows) - 1) / a.group;
    Span s;
    s.hi = max(min(w.first + static_cast<int32_t>(last_tok) + 1, w.end), 0);
    const int32_t first_hi = w.first + static_cast<int32_t>(first_tok) + 1;
    s.lo = a.window && first_hi > static_cast<int32_t>(a.window) ? first_hi - static_cast<int32_t>(a.window) : 0;
    const int32_t start = min(s.lo, s.hi) & ~31;
    // splits of at least 256 positions, in whole stages of any form
    const uint32_t n = static_cast<uint32_t>(s.hi - start), step = 64;
    const uint32_t each = max((n + a.splits - 1) / a.splits, 256u);
    const uint32_t part = (each + step - 1) / step * step;
    s.parts = max((n + part - 1) / part, 1u);
    s.from = static_cast<int32_t>(min(static_cast<uint64_t>(start) + static_cast<uint64_t>(part) * it.split, static_cast<uint64_t>(s.hi)));
    s.to = static_cast<int32_t>(min(static_cast<uint64_t>(s.from) + part, static_cast<uint64_t>(s.hi)));
    return s;
}

template <int HD>
__device__ __forceinline__ float* many_slot(const AttnArgs& a, uint32_t block) {
    return a.part + static_cast<size_t>(block) * (Many<HD>::kRows * (HD + 2));
}

// What the scheduler may move past a step of the products: all but them and their operands.
constexpr int kMoves = 0x2 | 0x4 | 0x10;  // VALU, SALU, VMEM

template <int HD, bool Q4, bool kHalved>
__device__ __forceinline__ void attend_many(const AttnArgs& a) {
    using M = Many<HD, kHalved>;
    using Stage = Operands<HD, M::kBlocks>;
    __shared__ __attribute__((aligned(16))) Stage ops[2];
    __shared__ uint32_t prefix[2], sums[8];
    const uint32_t tid = threadIdx.x, lane = tid & (kWave - 1), wid = __builtin_amdgcn_readfirstlane(tid / kWave);
    const uint32_t n = lane & 15, q = lane >> 4;
    SeqWork w;
    const Item it = item_of<HD>(a, blockIdx.x, prefix, sums, w);
    if (!it.any) return;
    const Span sp = span_of<HD>(a, it, w);
    if (it.split >= sp.parts) return;
    const uint32_t rows = static_cast<uint32_t>(w.len) * a.group;
    const uint32_t row0 = M::kRows * it.tile + 16 * M::kRt * (wid % M::kRowWaves), half = kHalved ? wid / M::kRowWaves : 0;
    QTile<HD> qt[M::kRt];
    Soft<HD> st[M::kRt];
    int32_t hi[M::kRt], lo[M::kRt];
#pragma unroll
    for (int i = 0; i < M::kRt; i++) {
        const uint32_t r = row0 + 16 * i + n;
        const bool live = r < rows;
        const uint32_t tok = live ? r / a.group : 0, head = it.h * a.group + (live ? r % a.group : 0);
        const int32_t pos = w.first + static_cast<int32_t>(tok);
        hi[i] = live ? pos + 1 : 0;
        lo[i] = a.window && hi[i] > static_cast<int32_t>(a.window) ? hi[i] - static_cast<int32_t>(a.window) : 0;
        load_q<HD, Q4>(qt[i], a.q + (static_cast<size_t>(w.row0 + tok) * a.n_heads + head) * HD, q, a.scale);
        soft_clear<HD>(st[i]);
        if (!live) st[i].m = 0.0f;
        if (live && pos >= 0 && static_cast<uint64_t>(pos) >= capacity(a.p)) st[i].l = __builtin_nanf("");
    }
    // the wave's rows are in order of position: what any of them and what all of them see
    const bool wave_live = row0 < rows;
    const uint32_t tok_a = min(row0, rows - 1) / a.group, tok_b = (min(row0 + 16 * M::kRt, rows) - 1) / a.group;
    const int32_t win = static_cast<int32_t>(a.window);
    const int32_t hi_a = w.first + static_cast<int32_t>(tok_a) + 1, hi_b = w.first + static_cast<int32_t>(tok_b) + 1;
    const int32_t any_lo = win && hi_a > win ? hi_a - win : 0, all_lo = win && hi_b > win ? hi_b - win : 0;
    const bool full_tile = row0 + 16 * M::kRt <= rows;

    const Job<HD> job = job_of<HD>(wid);
    Share<HD, Q4> sh;
    Pages ahead = {-1, -1};  // of the stage after the one that is loaded next
    const auto start_load = [&](uint32_t at) {
        sh.kb = at + 32 * job.blk;
        sh.g = pages_of(a.p, ahead, sh.kb);
        share_load<HD, Q4>(a.p, job, it.h, lane, sh);
        ahead = entries_at(a.p, it.s, sh.kb + M::kStage);
    };
    uint32_t at = static_cast<uint32_t>(sp.from), buf = 0;
    const uint32_t to = static_cast<uint32_t>(sp.to);
    if (at < to) {
        ahead = entries_at(a.p, it.s, at + 32 * job.blk);
        start_load(at);
        share_store<HD, Q4, M::kBlocks>(job, sh, ops[0], lane, sp.lo, sp.hi);
    }
    __syncthreads();
    for (; at < to; at += M::kStage) {
        const bool more = at + M::kStage < to;
        if (more) start_load(at + M::kStage);
        const Stage& op = ops[buf];
        constexpr int32_t kSpan = 32 * M::kMine;
        const int32_t kb = static_cast<int32_t>(at) + kSpan * static_cast<int32_t>(half);
        if (wave_live && kb < hi_b && kb + kSpan > any_lo) {
            // The operands of the stage in the order of their use, K's tiles, then V's: each
            // comes from LDS kAhead steps before its products.
            constexpr int kTiles = 2 * M::kMine, kK = kTiles * (HD / 32), kV = HD / 16, kAll = kK + M::kMine * kV;
            constexpr int kAhead = 3;
            v8h x[kAhead];
            const auto operand = [&](int j) {
                return j < kK ? op.k[M::kMine * half + j / (HD / 16)][j & 1][j / 2 % (HD / 32)][lane]
                              : op.v[M::kMine * half + (j - kK) / kV][(j - kK) % kV][lane];
            };
#pragma unroll
            for (int j = 0; j < kAhead; j++) x[j] = operand(j);
            __builtin_amdgcn_sched_barrier(kMoves);
            v4f s[M::kRt][kTiles];
#pragma unroll
            for (int r = 0; r < M::kRt; r++)
#pragma unroll
                for (int i = 0; i < kTiles; i++) s[r][i] = v4f{0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < kK; j++) {
                const int tile = 2 * (j / (HD / 16)) + (j & 1), i = j / 2 % (HD / 32);
                const v8h y = x[j % kAhead];
#pragma unroll
                for (int r = 0; r < M::kRt; r++) s[r][tile] = __builtin_amdgcn_mfma_f32_16x16x32_f16(y, qt[r].hi[i], s[r][tile], 0, 0, 0);
#pragma unroll
                for (int r = 0; r < M::kRt; r++) s[r][tile] = __builtin_amdgcn_mfma_f32_16x16x32_f16(y, qt[r].lo[i], s[r][tile], 0, 0, 0);
                x[j % kAhead] = operand(j + kAhead);
                __builtin_amdgcn_sched_barrier(kMoves);
            }
            float base[M::kRt];
            const bool masked = kb < all_lo || kb + kSpan > hi_a || !full_tile;
#pragma unroll
            for (int r = 0; r < M::kRt; r++) {
                if (masked) {
#pragma unroll
                    for (int j = 0; j < 4 * kTiles; j++) {
                        const int32_t p = kb + 32 * (j / 8) + static_cast<int32_t>(8 * q) + j % 8;
                        s[r][j / 4][j % 4] = p < lo[r] || p >= hi[r] ? -INFINITY : s[r][j / 4][j % 4];
                    }
                }
                base[r] = soft_base<HD, kTiles>(st[r], s[r], qt[r].factor);
            }
            // Block by block: the next one's probabilities between the products of this one's.
            v8h ph[2][M::kRt], pl[2][M::kRt];
            const float minus = minus_one();
            const auto pair = [&](int blk, int i) {  // of 4 kRt of a block
                const int r = i / 4, e = 2 * (i % 4);
                const v4f& v = s[r][2 * blk + e / 4];
                st[r].l += soft_pair(v[e % 4], v[e % 4 + 1], qt[r].factor, base[r], minus, ph[blk & 1][r], pl[blk & 1][r], e);
            };
#pragma unroll
            for (int i = 0; i < 4 * M::kRt; i++) pair(0, i);
#pragma unroll
            for (int j = kK; j < kAll; j++) {
                const int blk = (j - kK) / kV, c = (j - kK) % kV;
                const v8h y = x[j % kAhead];
#pragma unroll
                for (int r = 0; r < M::kRt; r++) st[r].o[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(y, ph[blk & 1][r], st[r].o[c], 0, 0, 0);
#pragma unroll
                for (int r = 0; r < M::kRt; r++) st[r].o[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(y, pl[blk & 1][r], st[r].o[c], 0, 0, 0);
                if (j + kAhead < kAll) x[j % kAhead] = operand(j + kAhead);
                if (blk + 1 < M::kMine) {
#pragma unroll
                    for (int i = c * 4 * M::kRt / kV; i < (c + 1) * 4 * M::kRt / kV; i++) pair(blk + 1, i);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if (more) share_store<HD, Q4, M::kBlocks>(job, sh, ops[buf ^ 1], lane, sp.lo, sp.hi);
        __syncthreads();
        buf ^= 1;
    }
    if constexpr (kHalved) {
        // the other half's sums through LDS, lane by lane
        static_assert(M::kRt == 1 && sizeof(ops) >= M::kRowWaves * kWave * (4 * HD / 16 + 2) * sizeof(float), "room for them");
        v4f* const o = reinterpret_cast<v4f*>(ops) + (wid % M::kRowWaves) * (HD / 16) * kWave + lane;
        float* const ml = reinterpret_cast<float*>(reinterpret_cast<v4f*>(ops) + M::kRowWaves * (HD / 16) * kWave) +
                          (wid % M::kRowWaves) * 2 * kWave + lane;
        if (half) {
#pragma unroll
            for (int c = 0; c < HD / 16; c++) o[c * kWave] = st[0].o[c];
            ml[0] = st[0].m;
            ml[kWave] = st[0].l;
        }
        __syncthreads();
        if (half) return;
        const float m1 = ml[0], l1 = ml[kWave], m = __builtin_fmaxf(st[0].m, m1);
        // without a maximum: nothing seen, or a sum of NaN
        const auto factor = [&](float mi, float li) {
            return mi == -INFINITY ? (li == 0.0f ? 0.0f : 1.0f) : __builtin_amdgcn_exp2f(mi - m);
        };
        const float f0 = factor(st[0].m, st[0].l), f1 = factor(m1, l1);
        st[0].m = m;
        st[0].l = st[0].l * f0 + l1 * f1;
#pragma unroll
        for (int c = 0; c < HD / 16; c++) st[0].o[c] = st[0].o[c] * f0 + o[c * kWave] * f1;
    }
    float* slot = many_slot<HD>(a, blockIdx.x);
#pragma unroll
    for (int i = 0; i < M::kRt; i++) {
        const uint32_t r = row0 + 16 * i + n;
        const float l = sum_over_q(st[i].l);
        if (r >= rows) continue;
        const uint32_t tok = r / a.group, head = it.h * a.group + r % a.group, in_tile = r - M::kRows * it.tile;
        const bool whole = sp.parts == 1;
        float* dst = whole ? a.out + (static_cast<size_t>(w.row0 + tok) * a.n_heads + head) * HD : slot + in_tile * HD;
        const float f = whole && l != 0.0f ? 1.0f / l : 1.0f;
#pragma unroll
        for (int c = 0; c < HD / 16; c++) {
            if constexpr (Q4) {
                // tiles 4 k .. 4 k + 3 hold runs of dims: 64 k + 16 q + 4 i + {0 .. 3}
                if (c % 4 == 0) {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const v4f o = {st[i].o[c][e], st[i].o[c + 1][e], st[i].o[c + 2][e], st[i].o[c + 3][e]};
                        *reinterpret_cast<v4f*>(dst + 16 * c + 16 * q + 4 * e) = o * f;
                    }
                }
            } else {
                *reinterpret_cast<v4f*>(dst + 16 * c + 4 * q) = st[i].o[c] * f;
            }
        }
        if (!whole && q == 0) {
            slot[M::kRows * HD + in_tile] = st[i].m;
            slot[M::kRows * HD + M::kRows + in_tile] = l;
        }
    }
}

// The join of an item's splits: a workgroup an item and 16 of its rows.
template <int HD, bool Q4>
__device__ __forceinline__ void merge_many(const AttnArgs& a) {
    using M = Many<HD>;
    __shared__ uint32_t prefix[2], sums[8];
    const uint32_t block = blockIdx.x / a.p.n_kv * a.p.n_kv * a.splits + blockIdx.x % a.p.n_kv;  // its first split's
    SeqWork w;
    const Item it = item_of<HD>(a, block, prefix, sums, w);
    if (!it.any) return;
    const Span sp = span_of<HD>(a, it, w);
    const uint32_t rows = static_cast<uint32_t>(w.len) * a.group;
    if (sp.parts == 1 || M::kRows * it.tile + 16 * blockIdx.y >= rows) return;
    // four splits of all of a thread's values in flight at once: the call is their latency
    constexpr int kE = HD / 64, kP = 4;
    const uint32_t d = 4 * (threadIdx.x % (HD / 4)), row0 = 16 * blockIdx.y + threadIdx.x / (HD / 4);
    constexpr uint32_t kStep = 256 / (HD / 4);  // rows
    float top[kE], sum[kE];
    v4f o[kE];
#pragma unroll
    for (int k = 0; k < kE; k++) {
        top[k] = -INFINITY;
        sum[k] = 0.0f;
        o[k] = v4f{0, 0, 0, 0};
    }
    for (uint32_t i = 0; i < sp.parts; i += kP) {
        float m[kE][kP], l[kE][kP];
        v4f v[kE][kP];
#pragma unroll
        for (int j = 0; j < kP; j++) {
            const float* slot = many_slot<HD>(a, block + min(i + j, sp.parts - 1) * a.p.n_kv);
#pragma unroll
            for (int k = 0; k < kE; k++) {
                const uint32_t row = min(row0 + kStep * k, rows - 1 - M::kRows * it.tile);  // rows past the last were not written
                m[k][j] = slot[M::kRows * HD + row];
                l[k][j] = slot[M::kRows * HD + M::kRows + row];
                v[k][j] = *reinterpret_cast<const v4f*>(slot + row * HD + d);
            }
        }
#pragma unroll
        for (int k = 0; k < kE; k++) {
            const float was = top[k];
#pragma unroll
            for (int j = 0; j < kP; j++) top[k] = __builtin_fmaxf(top[k], m[k][j]);  // the last one's twice is no harm
            const float old = was == top[k] ? 1.0f : __builtin_amdgcn_exp2f(was - top[k]);
            sum[k] *= old;
            o[k] *= old;
#pragma unroll
            for (int j = 0; j < kP; j++) {
                if (i + j >= sp.parts) break;
                const float f = m[k][j] == -INFINITY ? (l[k][j] == 0.0f ? 0.0f : 1.0f) : __builtin_amdgcn_exp2f(m[k][j] - top[k]);
                sum[k] += l[k][j] * f;
                o[k] += v[k][j] * f;
            }
        }
    }
#pragma unroll
    for (int k = 0; k < kE; k++) {
        const uint32_t rr = M::kRows * it.tile + row0 + kStep * k;
        if (rr >= rows) continue;
        const uint32_t tk = rr / a.group, hd = it.h * a.group + rr % a.group;
        if (sum[k] != 0.0f) o[k] /= sum[k];
        *reinterpret_cast<v4f*>(a.out + (static_cast<size_t>(w.row0 + tk) * a.n_heads + hd) * HD + d) = o[k];
    }
}

}  // namespace

#define ZLM_PAGED(HD, NAME, Q4)                                                                               \
    extern "C" __global__ void __launch_bounds__(256) zlm_paged_append_##NAME##_##HD(AppendArgs a) {          \
        append<HD, Q4>(a);                                                                                    \
    }                                                                                                         \
    extern "C" __global__ void __launch_bounds__(256) zlm_paged_read_##NAME##_##HD(ReadArgs a) {              \
        read_rows<HD, Q4>(a);                                                                                 \
    }                                                                                                         \
    extern "C" __global__ void __launch_bounds__(256, HD == 256 ? 1 : 2) zlm_paged_attend_few_##NAME##_##HD(AttnArgs a) { \
        attend_few<HD, Q4>(a);                                                                                \
    }                                                                                                         \
    extern "C" __global__ void __launch_bounds__(64 * Many<HD>::kWaves, 2) zlm_paged_attend_many_##NAME##_##HD(AttnArgs a) { \
        attend_many<HD, Q4, false>(a);                                                                               \
    }                                                                                                         \
    extern "C" __global__ void __launch_bounds__(256) zlm_paged_merge_many_##NAME##_##HD(AttnArgs a) {        \
        merge_many<HD, Q4>(a);                                                                                \
    }

ZLM_PAGED(64, f16, false)
ZLM_PAGED(64, q4_0, true)
ZLM_PAGED(128, f16, false)
ZLM_PAGED(128, q4_0, true)
ZLM_PAGED(256, f16, false)
ZLM_PAGED(256, q4_0, true)

#define ZLM_PAGED_HALVED(HD, NAME, Q4)                                                                         \
    extern "C" __global__ void __launch_bounds__(512, 2) zlm_paged_attend_halved_##NAME##_##HD(AttnArgs a) { \
        attend_many<HD, Q4, true>(a);                                                                         \
    }
ZLM_PAGED_HALVED(256, f16, false)
ZLM_PAGED_HALVED(256, q4_0, true)
