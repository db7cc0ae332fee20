// Attention over a paged cache held in 8 bits (pages of e4m3 with a power of two for each page and key head).
//
//   out = softmax(scale q . k) v,   k = 2^Ek[page] e4m3,   v = 2^Ev[page] e4m3
//
// An e4m3 value times a power of two is exact in bfloat16 (but for the last sixteenth below the type's largest, which pages may have rounded up past it), so keys and values become bfloat16 in one instruction for two of them
// (v_cvt_scalef32_pk_bf16_fp8) and both products run on the matrix cores' bfloat16 instruction with 32-bit sums.  Queries and weights in bfloat16 are one operand; in 32 bits a number is
// three bfloat16 numbers (8 + 8 + 8 bits of it) whose products with the cache are exact, so the 32-bit path is three products of bfloat16 and not
// one of the 32-bit instruction, which is sixteen times slower.
//
// The rows of a request and a key head are its tokens times the query heads of that key head, token by token; a wave takes 32 of them:
//
//   S^T = K . Q^T     v_mfma_f32_32x32x16_bf16, A = 32 keys, B = the rows.  A lane holds for one row (lane % 32) 16 of 32 scores, so maximum and sum
//                     are a reduction inside the lane and one exchange with lane ^ 32.
//   O^T += V^T . P^T  the lane's weights are the B operand as they stand: V^T is read from LDS in the order in which the scores lie in the registers.
//
// Maximum, sum and output are 32-bit.  In bfloat16 the weights of the second product are rounded to bfloat16 (2^-8 at most each), as in the other attention kernels here, since that product would take twice as long with two
// numbers a weight: outputs are 0.0018 of their size from 64 bits, 0.0022 in the kernel of many rows, whose largest weight may be anything up to 2^8 and is rounded too; their own rounding to bfloat16 alone is 0.0017.
// In 32 bits weights lose nothing.  Exponentials are base 2 with log2(e) folded into the scale.
#include "common.hpp"

typedef __bf16 a8_bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 a8_bf16x8 __attribute__((ext_vector_type(8)));
typedef float a8_f32x2 __attribute__((ext_vector_type(2)));
typedef float a8_f32x4 __attribute__((ext_vector_type(4)));
typedef float a8_f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t a8_u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t a8_u32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((__vector_size__(4 * sizeof(__bf16)))) __bf16 a8_bf16x4;
typedef __attribute__((address_space(3))) a8_bf16x4 a8_lds_bf16x4;

#define A8_KEYS 32       // keys a wave's tile where every wave has keys of its own
#define A8_WAVES 4
#define A8_MOST_KEYS 2048   // of a share of few rows as the caller cuts them, and as the kernel itself may (a8_balance):
#define A8_MOST_BALANCED 4096

union a8_frag {
    a8_bf16x8 vec;
    a8_u32x2 half[2];
    a8_u32x4 raw;
    uint32_t w[4];
};

struct A8Args {
    const void* q;
    int q_stride;
    void* out;
    const int *q_start, *q_len, *ctx_len;
    int S;
    const int* table;
    int width, block;
    uint32_t magic;           // of the division by `block` (a8_page_index)
    int shift, pages;
    const uint8_t *k_pool, *v_pool, *k_scale, *v_scale;
    int nq, nkv, d;
    int beside;               // key heads whose rows share lines of memory (a8_beside)
    float scale;              // times log2(e)
    int window;
    int n, chunk, chunks;     // rows of the step; keys a workgroup, and how many such shares the longest context has
    int most, places;         // few rows: the most keys a workgroup, and how many workgroups the chip holds at once (a8_balance)
    float *part_acc, *part_ml;
    int parts;                // shares that a row has room for there
    int rows_each;            // few rows: the room is numbered by request and key head with so many rows for each, or (0) by the step's rows and heads
    int* cut;                 // behind them: the shares of each request as a8_balance cut them, more than `chunks` for a context longer than the caller said
};

__device__ __forceinline__ uint32_t a8_pack2(float lo, float hi) {
    const a8_f32x2 pair = {lo, hi};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(pair, a8_bf16x2));
}

// Four e4m3 bytes times `unit` (a power of two) as bfloat16.
__device__ __forceinline__ a8_u32x2 a8_widen4(uint32_t bytes, float unit) {
    const a8_bf16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(bytes, unit, false), hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(bytes, unit, true);
    return a8_u32x2{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
}

// The transposing read of gfx950: among 16 neighbouring lanes, lane 4e + q points at row e, columns 4q .. 4q+3; lane i gets column i of the rows 0 .. 3.
__device__ __forceinline__ a8_u32x2 a8_read_transposed(const uint16_t* at) {
    return __builtin_bit_cast(a8_u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4bf16((a8_lds_bf16x4*)(at)));
}

template <int PIECES>
struct A8Type;
template <>
struct A8Type<1> {
    typedef bf16_t type;
};
template <>
struct A8Type<3> {
    typedef float type;
};

// Eight 32-bit numbers as PIECES bfloat16 operands whose sum they are (with one: rounded).
template <int PIECES>
__device__ __forceinline__ void a8_split(const float (&x)[8], a8_frag (&to)[PIECES]) {
    float rest[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) rest[e] = x[e];
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            to[p].w[e] = a8_pack2(rest[2 * e], rest[2 * e + 1]);
            if (p + 1 < PIECES) {
                rest[2 * e] -= __uint_as_float(to[p].w[e] << 16);
                rest[2 * e + 1] -= __uint_as_float(to[p].w[e] & 0xffff0000u);
            }
        }
    }
}

// Where the shares of a row are, in rows of the room: of a step in which few rows stand beside portions there is room for those few alone.
__device__ __forceinline__ size_t a8_place(const A8Args& a, int seq, int kvh, int row, size_t out_row) {
    return a.rows_each > 0 ? (static_cast<size_t>(seq) * a.nkv + kvh) * a.rows_each + row : out_row;
}

// Whether keys are more than the caller's longest context has.
__device__ __forceinline__ bool a8_late(const A8Args& a, int keys) { return keys > static_cast<long>(a.chunk) * a.chunks; }

// Whether request s brings rows.  (One whose context is shorter than what it brings holds the rows of a padded step.)
__device__ __forceinline__ bool a8_brings(const A8Args& a, int s) {
    const int q = a.q_len[s], c = a.ctx_len[s], at = a.q_start[s];         // (all three at once)
    return (q > 0) & (c >= q) & (at >= 0) & (at <= a.n - q);
}

// Rows that a request and key head bring are at most this many for the kernel of few rows (so many of its blocks of 16 as the registers hold, see A8Few), more for the kernel of many.
template <int PIECES, int DQ>
struct A8Few {
    static constexpr int BLOCKS = PIECES == 1 ? (DQ <= 2 ? 4 : 2) : (DQ == 1 ? 4 : DQ == 2 ? 2 : 1);
    // waves a SIMD: two where 256 registers hold a wave's
    static constexpr int WAVES(int blocks) { return PIECES * blocks * DQ > 6 || (DQ == 3 && blocks == 2) || (PIECES == 3 && blocks * DQ > 1) ? 1 : 2; }
};

// Workgroups go to the chip's eight XCDs in turn, and each XCD has an L2 of its own: where a line of 128 bytes holds several key heads' values, those heads' workgroups (`beside` of them) are dealt to one
// XCD, one turn behind the other, so the line is read from memory once (16 tokens at 4,000 keys, 8 key heads of 64: 27 us with neighbours on eight XCDs, 21 with them on one; 12 heads of 96: 55 and 38).
// Number `block` of a grid of a8_grid(...) is a unit (a request, or a block of rows), a key head and a share of the keys; false: there is no such unit.
#define A8_XCDS 8
__device__ __forceinline__ bool a8_deal(const A8Args& a, int block, int units, int& unit, int& kvh, int& share) {
    const int groups = a.nkv / a.beside, turn = block / A8_XCDS;
    const int at = turn / a.beside * A8_XCDS + block % A8_XCDS, rest = at / groups;
    kvh = at % groups * a.beside + turn % a.beside;
    share = rest / units;
    unit = rest - share * units;
    return share < a.chunks;
}
static long a8_grid(const A8Args& a, long units, int chunks) { return (units * chunks * (a.nkv / a.beside) + A8_XCDS - 1) / A8_XCDS * A8_XCDS * a.beside; }
// The fewest heads (at most eight, that divide their number) that fill whole lines together.
static int a8_beside(int nkv, int d) {
    int heads = 1;
    while (heads < 8 && heads * d % 128 != 0 && nkv % (2 * heads) == 0) heads *= 2;
    return heads;
}

// Inclusive sums over a wave: within rows of 16 lanes, then the rows before.  (In the registers: a shuffle through LDS is some 50 ns a step.)
__device__ __forceinline__ int a8_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);         // from one lane below, two, four, eight
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);         // the last of a row to the row behind it (the second and the fourth)
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);         // the last of the first half to the second half
    return v;
}

// Few rows of up to 64 requests whose shares are more than the chip holds at once: shares are made as much longer as brings them into the fewest rounds of the chip (a few workgroups in a round of their own take as
// long as all those of a full one), and a request's are equally long.  By a whole wave; lane s says what request s has (its first key, its keys, its shares, the keys of one).  No two shares stand under one number, and numbers have no
// gaps: workgroups without work between the others leave the shader engines, to which they go in turn, with more than they hold.
// 8 requests of 40 rows at 9,000 to 24,000 keys, 64 heads over 8: 70 us, 97 in shares of 2,048; single tokens of 32 heads over 8: 32 at 1,500 to 8,000 keys 74 and 87, 16 at 1,500 to 16,000 66 and 70.
struct A8Cut {
    int start, q_len, q_start, lo, keys, shares, size;
};
__device__ __forceinline__ A8Cut a8_balance(const A8Args& a, int group, int few) {
    const int s = threadIdx.x % PL_WAVE;
    A8Cut cut{0, 0, 0, 0, 0, 0, 0};
    if (s < a.S && a8_brings(a, s) && a.q_len[s] * group <= few) {
        cut.q_len = a.q_len[s];
        cut.q_start = a.q_start[s];
        cut.start = a.ctx_len[s] - cut.q_len;
        cut.lo = pl_first_visible(cut.start, a.window);
        // (of a context longer than the caller said so much as there is room for: its outputs become NaN)
        cut.keys = static_cast<int>(min(static_cast<long>(cut.start + cut.q_len - cut.lo), static_cast<long>(a.chunk) * a.chunks));
    }
    auto shares = [&](int size) { return cut.keys > 0 ? (cut.keys - 1) / size + 1 : 0; };
    auto all = [&](int size) { return __builtin_amdgcn_readlane(a8_scan(shares(size)), PL_WAVE - 1) * a.nkv; };
    int size = a.chunk;
    if (all(size) > a.places) {
        const int room = pl_ceil_div(all(a.most), a.places) * a.places;
        int low = size / A8_KEYS, high = a.most / A8_KEYS;
        while (low < high) {
            const int mid = (low + high) / 2;
            if (all(mid * A8_KEYS) <= room) high = mid;
            else low = mid + 1;
        }
        size = high * A8_KEYS;
    }
    cut.shares = shares(size);
    cut.size = cut.shares == 0 ? size : ((cut.keys - 1) / cut.shares / A8_KEYS + 1) * A8_KEYS;
    return cut;
}

// Which request and which of its blocks of rows is number `slot`, counted over the requests of more than `few` rows one after the other; by a whole wave.
__device__ __forceinline__ bool a8_find(const A8Args& a, int slot, int group, int rows, int few, int& seq, int& block) {
    const int lane = threadIdx.x % PL_WAVE;
    for (int base = 0; base < a.S; base += PL_WAVE) {
        const int s = base + lane;
        int blocks = 0;
        if (s < a.S && a8_brings(a, s) && a.q_len[s] * group > few) blocks = pl_ceil_div(a.q_len[s] * group, rows);
        const int end = a8_scan(blocks);
        const uint64_t past = __ballot(end > slot);
        if (past != 0) {
            const int first = __ffsll(static_cast<unsigned long long>(past)) - 1;
            seq = __builtin_amdgcn_readfirstlane(base + first);
            // (the last rows, which see the most keys, first)
            block = __builtin_amdgcn_readlane(end, first) - 1 - slot;
            return true;
        }
        slot -= __builtin_amdgcn_readlane(end, PL_WAVE - 1);
    }
    return false;
}

// The keys [lo, hi) that a block of rows sees, cut into shares of `chunk` that begin at whole chunks: how many there are.
__device__ __forceinline__ int a8_shares(int lo, int hi, int chunk) { return hi > lo ? (hi - 1) / chunk - lo / chunk + 1 : 0; }

// Which of its request's pages a key is in: a division by the page size, as a product with ceil(2^shift / block), shift = 31 + ceil(log2(block)), exact below 2^31.
__device__ __forceinline__ int a8_page_index(const A8Args& a, int key) { return static_cast<int>(static_cast<uint64_t>(static_cast<uint32_t>(key)) * a.magic >> a.shift); }
// A page's power, a byte, as the number.
__device__ __forceinline__ float a8_unit(uint32_t power) { return __uint_as_float(power << 23); }

// Four neighbouring results of one row, as the caller's type.
template <int PIECES>
__device__ __forceinline__ void a8_store4(const A8Args& a, size_t at, float x0, float x1, float x2, float x3) {
    if constexpr (PIECES == 1) *reinterpret_cast<a8_u32x2*>(static_cast<bf16_t*>(a.out) + at) = a8_u32x2{a8_pack2(x0, x1), a8_pack2(x2, x3)};
    else *reinterpret_cast<a8_f32x4*>(static_cast<float*>(a.out) + at) = a8_f32x4{x0, x1, x2, x3};
}

// Eight neighbouring values of a query's head, or zeros.
template <int PIECES>
__device__ __forceinline__ void a8_query8(const A8Args& a, size_t at, bool there, a8_frag (&to)[PIECES]) {
    if constexpr (PIECES == 1) {
        to[0].raw = there ? *reinterpret_cast<const a8_u32x4*>(static_cast<const bf16_t*>(a.q) + at) : a8_u32x4{0u, 0u, 0u, 0u};
    } else {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = there ? static_cast<const float*>(a.q)[at + e] : 0.f;
        a8_split<PIECES>(x, to);
    }
}

// The maximum of a lane's number and that of lane ^ 32.
__device__ __forceinline__ float a8_max_half(float v) {
    const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1]));
}
// And of those of lanes ^ 16, ^ 32 and ^ 48.
__device__ __forceinline__ float a8_max_quarters(float v) {
    v = a8_max_half(v);
    const auto both = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1]));
}

// ---- a row by itself ----------------------------------------------------------------------------------------------------
// A weight of zero does not hide a value that is not finite, and a tile's values meet the rows of several tokens, which need not all see its keys.  So where the rows of a workgroup do not all see its keys,
// and a row's result is not finite, a wave works that row out again from the keys [lo, hi) that it sees, one by one, and the row is what these make it.  (Looking at every tile's values among the work on it
// cost 2 to 15%, whether or not there are any.)  Only where that would change something: where one of the other keys that met the row, which are in [met_from, met_to), has such a value in a column that is
// not finite, and none of those that the row sees has, looked for from the nearest one back.  (8,100 tokens of 32 heads take 4.8 ms where all values are NaN, 4.4 where one token's
// are, 9.3 where every 500th's are, 0.6 where none is.)
// A function that is called, and that reads the launch's arguments anew: worked into the kernels it takes registers from their loops (184 instead of 148 for single tokens, a third of their workgroups).
__device__ __forceinline__ const A8Args& a8_args_again() {
    uint64_t at = reinterpret_cast<uint64_t>(__builtin_amdgcn_kernarg_segment_ptr());          // (their first argument in both)
    asm volatile("" : "+s"(at));
    return *reinterpret_cast<const A8Args*>(at);
}
template <int PIECES>
__device__ __attribute__((noinline)) void a8_row_alone(const A8Args& a, int seq, int kvh, int lo, int hi, int met_from, int met_to, size_t row, size_t place, bool whole, int head) {
    typedef typename A8Type<PIECES>::type T;
    const int lane = threadIdx.x % PL_WAVE;
    const T* q = static_cast<const T*>(a.q) + row * a.q_stride + static_cast<size_t>(head) * a.d;
    const size_t out_row = row * a.nq + head;
    // Where a key is, and the place of its powers.
    auto place_of = [&](int key, int& slot, size_t& power) {
        const int index = a8_page_index(a, key), found = a.table[static_cast<size_t>(seq) * a.width + min(index, a.width - 1)];
        const int page = static_cast<unsigned>(found) < static_cast<unsigned>(a.pages) ? found : 0;
        slot = page * a.block + key - index * a.block;
        power = static_cast<size_t>(page) * a.nkv + kvh;
    };
    // Which of the lane's columns (lane, lane + 64, ...), a bit each, have a value that is not finite among the keys [from, to), at most 64.
    auto wild_among = [&](int from, int to) {
        uint32_t wild = 0;
        if (from >= to) return wild;
        int slot;
        size_t power;
        place_of(min(from + lane, to - 1), slot, power);
        const float unit = a8_unit(a.v_scale[power]);
#pragma unroll 4
        for (int j = 0; j < to - from; ++j) {
            const float u = __shfl(unit, j, PL_WAVE);
            const uint8_t* v = a.v_pool + (static_cast<size_t>(__shfl(slot, j, PL_WAVE)) * a.nkv + kvh) * a.d;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (lane + PL_WAVE * i < a.d && !(fabsf(__builtin_amdgcn_cvt_f32_fp8(v[lane + PL_WAVE * i], 0) * u) < INFINITY)) wild |= 1u << i;
        }
        return wild;
    };
    uint32_t spoilt = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int c = lane + PL_WAVE * i;
        if (c < a.d && !(fabsf(whole ? to_float(static_cast<const T*>(a.out)[out_row * a.d + c]) : a.part_acc[place * a.d + c]) < INFINITY)) spoilt |= 1u << i;
    }
    uint32_t others = 0;
#pragma unroll 1
    for (int from = met_from; from < lo; from += PL_WAVE) others |= wild_among(from, min(from + PL_WAVE, lo));
#pragma unroll 1
    for (int from = hi; from < met_to; from += PL_WAVE) others |= wild_among(from, min(from + PL_WAVE, met_to));
    spoilt &= others;
#pragma unroll 1
    for (int to = hi; to > lo && __any(spoilt != 0); to -= PL_WAVE) spoilt &= ~wild_among(max(to - PL_WAVE, lo), to);
    if (!__any(spoilt != 0)) return;

    float m = -INFINITY, l = 0.f, out[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int base = lo; base < hi; base += PL_WAVE) {
        int slot;
        size_t power;
        place_of(min(base + lane, hi - 1), slot, power);
        const size_t at = (static_cast<size_t>(slot) * a.nkv + kvh) * a.d;
        float score = 0.f;
#pragma unroll 1
        for (int c = 0; c < a.d; c += 4) {
            const uint32_t bytes = *reinterpret_cast<const uint32_t*>(a.k_pool + at + c);
            const a8_f32x2 k01 = __builtin_amdgcn_cvt_pk_f32_fp8(bytes, false), k23 = __builtin_amdgcn_cvt_pk_f32_fp8(bytes, true);
            score = fmaf(to_float(q[c]), k01[0], fmaf(to_float(q[c + 1]), k01[1], fmaf(to_float(q[c + 2]), k23[0], fmaf(to_float(q[c + 3]), k23[1], score))));
        }
        score = base + lane < hi ? score * a8_unit(a.k_scale[power]) * a.scale : -INFINITY;
        const float grown = fmaxf(m, wave_max(score)), from = grown == -INFINITY ? 0.f : grown;
        const float alpha = __builtin_amdgcn_exp2f(m - from), weight = __builtin_amdgcn_exp2f(score - from);
        const float unit = a8_unit(a.v_scale[power]);
        m = grown;
        l = l * alpha + weight;
#pragma unroll
        for (int i = 0; i < 4; ++i) out[i] *= alpha;
        const int here = min(hi - base, PL_WAVE);
#pragma unroll 1
        for (int eight = 0; eight < here; eight += 8) {                // (eight keys among themselves first: fewer roundings behind each other)
            float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
            for (int j = eight; j < min(eight + 8, here); ++j) {
                const float w = __shfl(weight, j, PL_WAVE), u = __shfl(unit, j, PL_WAVE);
                const uint8_t* v = a.v_pool + (static_cast<size_t>(__shfl(slot, j, PL_WAVE)) * a.nkv + kvh) * a.d;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (lane + PL_WAVE * i < a.d) x[i] = fmaf(w, __builtin_amdgcn_cvt_f32_fp8(v[lane + PL_WAVE * i], 0) * u, x[i]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) out[i] += x[i];
        }
    }
    l = wave_sum(l);
    const float inv = l != 0.f ? 1.f / l : 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int c = lane + PL_WAVE * i;
        if (c >= a.d) continue;
        if (whole) static_cast<T*>(a.out)[out_row * a.d + c] = from_float<T>(out[i] * inv);
        else a.part_acc[place * a.d + c] = out[i];
    }
    if (!whole && lane == 0) {
        a.part_ml[2 * place] = m;
        a.part_ml[2 * place + 1] = l;
    }
}

// ---- few rows: every wave has keys of its own ------------------------------------------------------------------------------
// A workgroup takes the RB blocks of 16 rows of one request and key head and one share of the keys; its waves take tiles of 32 keys in turn, each with a running maximum and sum, and meet at the end.
// Keys go from memory into the registers that the product reads (a lane reads 16 bytes of one key: the contraction may go through a head's values in any order, so the
// queries are laid out to match); values go through a piece of LDS that belongs to the wave, so the loop has no barrier.  The next tile's bytes are on their way while a tile is worked on.
// Bound by memory: 64 single tokens of 32 heads over 8 at contexts of 1,000 to 12,000 read 857 MB in 190 us, 4.5 TB/s (a copy of 4 GB moves 4.6, pieces of 128 bytes as these are read at 5.3), and their shares are
// put together in another 6.  A wave has one key head: four heads' pieces side by side would be read at 6.2 TB/s, but with four times the shares to put together.
//   S^T = K . Q^T: v_mfma_f32_16x16x32_bf16, twice for 32 keys; a lane has for row lane % 16 the keys 4 (lane / 16) .. + 3 of both.  DQ: the head is padded to 64 DQ values.
//   BALANCED: with the shares of a8_balance.  (A build of its own: the one for shares as the caller cut them loses 0.4 to 1 us of 12 to 20 to what is only compiled in.)
template <int PIECES, int DQ, int RB, bool BALANCED>
__global__ __launch_bounds__(A8_WAVES * PL_WAVE, (A8Few<PIECES, DQ>::WAVES(RB))) void attention_8bit_few_kernel(A8Args a) {
    constexpr int DP = 64 * DQ, VROW = DP + 16;              // (16 more: eight rows read transposed fall on every bank once)
    constexpr int MROW = DP + 4;
    constexpr int VALUES = A8_WAVES * A8_KEYS * VROW * 2, MEET = 2 * 16 * MROW * 4;
    static_assert(MEET <= VALUES, "the waves meet where their values were");
    extern __shared__ __attribute__((aligned(16))) char lds[];
    uint16_t* values = reinterpret_cast<uint16_t*>(lds);
    float* stats = reinterpret_cast<float*>(lds + VALUES);   // [waves][2][rows]
    int* slots = reinterpret_cast<int*>(stats + A8_WAVES * 2 * 16 * RB);
    uint16_t* units = reinterpret_cast<uint16_t*>(slots + (BALANCED ? a.most : a.chunk));           // (the two powers of a key, a byte each)

    const int tid = threadIdx.x, lane = tid % PL_WAVE, wave = tid / PL_WAVE;
    const int col = lane % 16, quarter = lane / 16;
    const int group = a.nq / a.nkv;
    int kvh, seq, share, q_len, q_start, start, lo, hi, shares, size, k_base;
    if (!a8_deal(a, blockIdx.x, a.S, seq, kvh, share)) return;
    if constexpr (BALANCED) {
        const A8Cut cut = a8_balance(a, group, 16 * RB);
        const int number = share * a.S + seq, end = a8_scan(cut.shares);
        const uint64_t past = __ballot(end > number);
        if (past == 0) return;
        seq = __ffsll(static_cast<unsigned long long>(past)) - 1;
        q_len = __builtin_amdgcn_readlane(cut.q_len, seq);
        q_start = __builtin_amdgcn_readlane(cut.q_start, seq);
        start = __builtin_amdgcn_readlane(cut.start, seq);
        lo = __builtin_amdgcn_readlane(cut.lo, seq);
        shares = __builtin_amdgcn_readlane(cut.shares, seq);
        size = __builtin_amdgcn_readlane(cut.size, seq);
        share = number - (__builtin_amdgcn_readlane(end, seq) - shares);
        hi = start + q_len;
        k_base = lo + share * size;
        const bool first = share == 0 && kvh == 0 && tid == 0;
        if (a8_late(a, hi - lo)) shares = a.chunks + 1;
        if (first) a.cut[seq] = shares;
    } else {
        if (!a8_brings(a, seq) || a.q_len[seq] * group > 16 * RB) return;
        q_len = a.q_len[seq];
        q_start = a.q_start[seq];
        start = a.ctx_len[seq] - q_len;
        lo = pl_first_visible(start, a.window);
        hi = start + q_len;
        size = a.chunk;
        shares = a8_shares(lo, hi, size);
        if (share >= shares) return;
        k_base = (lo / size + share) * size;
    }
    const int rows = q_len * group;
    const int k_begin = max(lo, k_base), k_end = k_base + min(hi - k_base, size);
    const int last_from = pl_first_visible(start + q_len - 1, a.window);     // (the last token's first key: no token's is later)

    // Where the keys of the share are, and in what units.  (Keys that no row sees are read at the nearest one's place.)  All pages are asked for, then all powers: one behind the other they would be a
    // wait each for every 256 keys.
    constexpr int EACH = (BALANCED ? A8_MOST_BALANCED : A8_MOST_KEYS) / (A8_WAVES * PL_WAVE);
    const int keys = min(pl_ceil_div(k_end - k_base, A8_KEYS) * A8_KEYS, size);
    int page[EACH];
    const int* row_table = a.table + static_cast<size_t>(seq) * a.width;
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        const int i = tid + e * A8_WAVES * PL_WAVE;
        if (e * A8_WAVES * PL_WAVE < keys) page[e] = row_table[min(a8_page_index(a, min(max(k_base + i, k_begin), k_end - 1)), a.width - 1)];
    }
    uint32_t k_power[EACH], v_power[EACH];
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        if (e * A8_WAVES * PL_WAVE < keys) {
            page[e] = static_cast<unsigned>(page[e]) < static_cast<unsigned>(a.pages) ? page[e] : 0;
            const size_t at = static_cast<size_t>(page[e]) * a.nkv + kvh;
            k_power[e] = a.k_scale[at];
            v_power[e] = a.v_scale[at];
        }
    }
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        const int i = tid + e * A8_WAVES * PL_WAVE;
        if (i < keys) {
            const int key = min(max(k_base + i, k_begin), k_end - 1);
            slots[i] = page[e] * a.block + key - a8_page_index(a, key) * a.block;
            units[i] = static_cast<uint16_t>(k_power[e] | v_power[e] << 8);
        }
    }

    // The rows: what a lane reads of a key with its j-th load are the values 64 j + 16 quarter .. + 15, two operands
    int seen_from[RB], seen[RB], out_row[RB];        // the keys of the share that a row sees: the first and how many
    a8_frag qf[RB][2 * DQ][PIECES];
#pragma unroll
    for (int b = 0; b < RB; ++b) {
        const int row = 16 * b + col;
        const bool live = row < rows;
        const int token = live ? row / group : 0, head = kvh * group + (live ? row % group : 0);
        seen_from[b] = max(pl_first_visible(start + token, a.window), k_begin);
        seen[b] = max(min(start + token + 1, k_end) - seen_from[b], 0);
        out_row[b] = live ? (q_start + token) * a.nq + head : -1;
#pragma unroll
        for (int j = 0; j < 2 * DQ; ++j) {
            const int at = 64 * (j / 2) + 16 * quarter + 8 * (j % 2);
            a8_query8<PIECES>(a, static_cast<size_t>(q_start + token) * a.q_stride + static_cast<size_t>(head) * a.d + at, live && at < a.d, qf[b][j]);
        }
    }
    __syncthreads();

    uint16_t* mine = values + wave * A8_KEYS * VROW;
    a8_f32x4 acc[RB][4 * DQ];
    float m[RB], l[RB];
#pragma unroll
    for (int b = 0; b < RB; ++b) {
        m[b] = -INFINITY;
        l[b] = 0.f;
#pragma unroll
        for (int t = 0; t < 4 * DQ; ++t) acc[b][t] = a8_f32x4{0.f, 0.f, 0.f, 0.f};
    }

    // A tile on its way: keys in two halves of 16, values 16 bytes a lane, 4 DQ lanes a key.  Where they are is read from LDS a tile before their bytes are asked for, and no load stands under a condition
    // (a lane without a piece of a head reads the last one: the queries' zeros take its products out, and nothing keeps its results), so a tile has no wait but for its bytes.
    constexpr int VP = 4 * DQ, LOADS = 2 * DQ;
    a8_u32x4 kraw[LOADS], vraw[LOADS];
    int k_slot[2], v_slot[LOADS];
    uint32_t k_unit[2], v_unit[LOADS];
    const uint32_t row_bytes = a.nkv * a.d;
    const int last_piece = a.d / 16 - 1;
    const uint8_t *k_from = a.k_pool + kvh * a.d, *v_from = a.v_pool + kvh * a.d;
    auto look = [&](int base) {
#pragma unroll
        for (int half = 0; half < 2; ++half) k_slot[half] = slots[base + 16 * half + col];
#pragma unroll
        for (int i = 0; i < LOADS; ++i) v_slot[i] = slots[base + (i * PL_WAVE + lane) / VP];
    };
    auto fetch = [&](int base) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) vraw[i] = *reinterpret_cast<const a8_u32x4*>(v_from + static_cast<size_t>(v_slot[i]) * row_bytes + 16 * min((i * PL_WAVE + lane) % VP, last_piece));
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int j = 0; j < DQ; ++j)
                kraw[half * DQ + j] = *reinterpret_cast<const a8_u32x4*>(k_from + static_cast<size_t>(k_slot[half]) * row_bytes + 16 * min(4 * j + quarter, last_piece));
#pragma unroll
        for (int half = 0; half < 2; ++half) k_unit[half] = units[base + 16 * half + col];
#pragma unroll
        for (int i = 0; i < LOADS; ++i) v_unit[i] = units[base + (i * PL_WAVE + lane) / VP];
    };
    // this wave's first and last tiles with keys (past the share's last tile that one is read once more)
    const int first_tile = (k_begin - k_base) / A8_KEYS, end_tile = pl_ceil_div(k_end - k_base, A8_KEYS);
    int tile = first_tile + wave;
    if (tile < end_tile) {
        look(tile * A8_KEYS);
        fetch(tile * A8_KEYS);
        look(min(tile + A8_WAVES, end_tile - 1) * A8_KEYS);
    }
    for (; tile < end_tile; tile += A8_WAVES) {
        const int k0 = k_base + tile * A8_KEYS;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int at = i * PL_WAVE + lane, key = at / VP, piece = at % VP;
            const float unit = a8_unit(v_unit[i] >> 8);
            a8_frag to[2];
#pragma unroll
            for (int e = 0; e < 4; ++e) to[e / 2].half[e % 2] = a8_widen4(vraw[i][e], unit);
            // (the first eight of 16 values stand in the row's first half, the others in its second: neighbouring lanes write neighbouring pieces)
            *reinterpret_cast<a8_u32x4*>(mine + key * VROW + 8 * piece) = to[0].raw;
            *reinterpret_cast<a8_u32x4*>(mine + key * VROW + DP / 2 + 8 * piece) = to[1].raw;
        }
        a8_f32x4 s[RB][2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const float unit = a8_unit(k_unit[half] & 0xff);
#pragma unroll
            for (int b = 0; b < RB; ++b) s[b][half] = a8_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < 2 * DQ; ++j) {
                a8_frag kf;
                kf.half[0] = a8_widen4(kraw[half * DQ + j / 2][2 * (j % 2)], unit);
                kf.half[1] = a8_widen4(kraw[half * DQ + j / 2][2 * (j % 2) + 1], unit);
#pragma unroll
                for (int b = 0; b < RB; ++b)
#pragma unroll
                    for (int p = PIECES - 1; p >= 0; --p) s[b][half] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf.vec, qf[b][j][p].vec, s[b][half], 0, 0, 0);
            }
        }
        fetch(min(tile + A8_WAVES, end_tile - 1) * A8_KEYS);
        look(min(tile + 2 * A8_WAVES, end_tile - 1) * A8_KEYS);
        const bool whole = k0 >= k_begin && k0 >= last_from && k0 + A8_KEYS <= k_end && k0 + A8_KEYS - 1 <= start;
        a8_frag pf[RB][PIECES];
#pragma unroll
        for (int b = 0; b < RB; ++b) {
            // (Chosen value by value: elements of a product's result written under a branch have come out as another element here, in the build for 32 bits.)
            float x[8], top = m[b];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[e] = s[b][e / 4][e % 4] * a.scale;
                if (!whole) {
                    const int key = k0 + 16 * (e / 4) + 4 * quarter + e % 4;
                    x[e] = static_cast<unsigned>(key - seen_from[b]) < static_cast<unsigned>(seen[b]) ? x[e] : -INFINITY;
                }
                top = fmaxf(top, x[e]);
            }
            top = a8_max_quarters(top);
            const float from = top == -INFINITY ? 0.f : top;
            const float alpha = __builtin_amdgcn_exp2f(m[b] - from);
            m[b] = top;
            float sum = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[e] = __builtin_amdgcn_exp2f(x[e] - from);
                sum += x[e];
            }
            l[b] = l[b] * alpha + sum;
            a8_split<PIECES>(x, pf[b]);
#pragma unroll
            for (int t = 0; t < 4 * DQ; ++t) acc[b][t] *= alpha;
        }
        __builtin_amdgcn_wave_barrier();
        const uint16_t* v_at = mine + (4 * quarter + col / 4) * VROW + 4 * (col % 4);
#pragma unroll
        for (int t = 0; t < 4 * DQ; ++t) {
            a8_frag vf;
            vf.half[0] = a8_read_transposed(v_at + 16 * t);
            vf.half[1] = a8_read_transposed(v_at + 16 * VROW + 16 * t);
#pragma unroll
            for (int b = 0; b < RB; ++b)
#pragma unroll
                for (int p = PIECES - 1; p >= 0; --p) acc[b][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf.vec, pf[b][p].vec, acc[b][t], 0, 0, 0);
        }
        __builtin_amdgcn_wave_barrier();
    }

    const bool whole_row = BALANCED ? shares == 1 : a.chunks == 1;       // (nothing to be put together)
    // The waves meet: maximum and sum first, then the outputs in halves, always in the same order.
#pragma unroll
    for (int b = 0; b < RB; ++b) {
        l[b] += __shfl_xor(l[b], 16, PL_WAVE);
        l[b] += __shfl_xor(l[b], 32, PL_WAVE);
        if (quarter == 0) {
            stats[(2 * wave) * 16 * RB + 16 * b + col] = m[b];
            stats[(2 * wave + 1) * 16 * RB + 16 * b + col] = l[b];
        }
    }
    __syncthreads();
    // (not all rows see all keys of the share)
    const bool unlike = k_begin < last_from || k_end - 1 > start;
    uint64_t again = 0;                          // rows that are worked out once more
    float* meet = reinterpret_cast<float*>(lds);
#pragma unroll
    for (int b = 0; b < RB; ++b) {
        float top = -INFINITY, total = 0.f;
#pragma unroll
        for (int w = 0; w < A8_WAVES; ++w) top = fmaxf(top, stats[2 * w * 16 * RB + 16 * b + col]);
        const float from = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int w = 0; w < A8_WAVES; ++w)
            total += stats[(2 * w + 1) * 16 * RB + 16 * b + col] * __builtin_amdgcn_exp2f(stats[2 * w * 16 * RB + 16 * b + col] - from);
        const float weight = __builtin_amdgcn_exp2f(m[b] - from);
#pragma unroll
        for (int t = 0; t < 4 * DQ; ++t) acc[b][t] *= weight;
#pragma unroll
        for (int step = A8_WAVES / 2; step > 0; step /= 2) {
            if (wave >= step && wave < 2 * step && out_row[b] >= 0)
#pragma unroll
                for (int t = 0; t < 4 * DQ; ++t) *reinterpret_cast<a8_f32x4*>(meet + ((wave - step) * 16 + col) * MROW + 16 * t + 4 * quarter) = acc[b][t];
            __syncthreads();
            if (wave < step && out_row[b] >= 0)
#pragma unroll
                for (int t = 0; t < 4 * DQ; ++t) acc[b][t] += *reinterpret_cast<const a8_f32x4*>(meet + (wave * 16 + col) * MROW + 16 * t + 4 * quarter);
            __syncthreads();
        }
        if (wave == 0 && out_row[b] >= 0) {
            if (__builtin_expect(unlike, 0)) {
                float finite = 0.f;              // (or NaN)
#pragma unroll
                for (int t = 0; t < 4 * DQ; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) finite = fmaf(acc[b][t][i], 0.f, finite);
                uint64_t bad = __ballot(finite != finite && total == total);          // (weights that are NaN leave nothing else)
                bad |= bad >> 32;
                again |= ((bad | bad >> 16) & 0xffff) << (16 * b);
            }
            const size_t place = a8_place(a, seq, kvh, 16 * b + col, out_row[b]) * a.parts + share;
            if (whole_row) {
                if (!BALANCED && shares > 1) total = NAN;          // (a context longer than the caller said)
                const float inv = total != 0.f ? 1.f / total : 0.f;
#pragma unroll
                for (int t = 0; t < 4 * DQ; ++t) acc[b][t] *= inv;
            } else if (quarter == 0) {
                a.part_ml[2 * place] = top;
                a.part_ml[2 * place + 1] = total;
            }
#pragma unroll
            for (int t = 0; t < 4 * DQ; ++t) {
                const int c = 16 * t + 4 * quarter;           // (as the values stood in LDS)
                const int at = 16 * (c % (DP / 2) / 8) + 8 * (c / (DP / 2)) + c % 8;
                if (at >= a.d) continue;
                if (whole_row) a8_store4<PIECES>(a, static_cast<size_t>(out_row[b]) * a.d + at, acc[b][t][0], acc[b][t][1], acc[b][t][2], acc[b][t][3]);
                else *reinterpret_cast<a8_f32x4*>(a.part_acc + place * a.d + at) = acc[b][t];
            }
        }
    }
    if (__builtin_expect(!unlike, 1)) return;
    again = static_cast<uint64_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(again >> 32))) << 32 | static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(again)));
    if (again == 0 || wave != 0 || (!BALANCED && whole_row && shares > 1)) return;
    __threadfence_block();
    for (; again != 0; again &= again - 1) {
        const int row = __ffsll(static_cast<unsigned long long>(again)) - 1, token = row / group, head = kvh * group + row % group;
        const size_t place = a8_place(a, seq, kvh, row, static_cast<size_t>(q_start + token) * a.nq + head) * a.parts + share;
        a8_row_alone<PIECES>(a8_args_again(), seq, kvh, max(pl_first_visible(start + token, a.window), k_begin), min(start + token + 1, k_end), k_begin, k_end, q_start + token, place,
                             whole_row, head);
    }
}

// ---- many rows: every wave has rows of its own -----------------------------------------------------------------------------
// A workgroup takes NW blocks of 32 rows of one request and key head and one share of the keys, a block a wave.  Tiles of 32 KB keys come into LDS as bfloat16, so what an e4m3 value costs to widen is
// paid once for all the rows.
//   S^T = K . Q^T: v_mfma_f32_32x32x16_bf16; a lane has for row lane % 32 the keys 8 (i / 4) + 4 (lane / 32) + i % 4 of 32.  DT: the head is padded to 32 DT values.
// What bounds it is what a SIMD can issue: of a tile of 64 keys and 128 values a wave's products take 1,024 cycles, its other vector instructions some 1,060 (an exponential as long as two of the rest), and LDS,
// which every wave reads whole, another 500 a wave and its share of the unit.  So the scores of the next tile are multiplied while the weights of this one are made, and the next maximum is found while
// this tile's weights meet its values: both pipes work in one wave, whatever the other wave of the SIMD does.  For that the keys in LDS are a tile ahead of the values (two lengths of keys, three of
// values), their bytes another tile ahead in registers, and their pages one more.  A round has one barrier.  8,100 tokens of 32 heads over 8 take 0.515 ms, 1,045 TFLOP/s (0.50 to 0.56 as the card clocks;
// a large matrix product of the library reaches 1,450 on the same card); without the overlap they took 0.69 when that was 0.57.  Tried and slower: the two waves of a SIMD half a round apart with a barrier a half (0.64), 64 rows a wave with all 512 registers (0.85: moves
// between the two halves of the register file).
template <int PIECES, int DT>
struct A8Many {
    static constexpr int KB = DT == 8 || (PIECES == 3 && DT != 4) ? 1 : 2;     // (what 160 KB of LDS hold; in 32 bits what leaves two waves a SIMD their registers, where that can be)
    static constexpr int WAVES = PIECES == 1 ? (DT <= 4 ? 2 : 1) : (DT <= 3 ? 2 : 1);   // a SIMD
    static constexpr int KROW = 32 * DT + 8, VROW = 32 * DT + (DT % 2 == 0 ? 32 : 0);
    static constexpr size_t LDS = static_cast<size_t>(32 * KB) * (2 * KROW + 3 * VROW) * 2;
};

template <int PIECES, int DT, int NW>
__global__ __launch_bounds__(NW * PL_WAVE) __attribute__((amdgpu_waves_per_eu(A8Many<PIECES, DT>::WAVES, A8Many<PIECES, DT>::WAVES))) void attention_8bit_many_kernel(A8Args a, int few, int units) {
    constexpr int KB = A8Many<PIECES, DT>::KB, TILE = 32 * KB, KROW = A8Many<PIECES, DT>::KROW, VROW = A8Many<PIECES, DT>::VROW, THREADS = NW * PL_WAVE;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    uint16_t* keys = reinterpret_cast<uint16_t*>(lds);                 // [2][TILE][KROW]
    uint16_t* values = keys + 2 * TILE * KROW;                         // [3][TILE][VROW]

    const int tid = threadIdx.x, lane = tid % PL_WAVE, wave = __builtin_amdgcn_readfirstlane(tid / PL_WAVE);
    const int col = lane % 32, half = lane / 32;
    const int group = a.nq / a.nkv;
    int kvh, unit, share, seq, rb;
    if (!a8_deal(a, blockIdx.x, units, unit, kvh, share) || !a8_find(a, unit, group, 32 * NW, few, seq, rb)) return;
    const int q_len = a.q_len[seq], start = a.ctx_len[seq] - q_len, q_start = a.q_start[seq];
    const int first_row = rb * 32 * NW, rows = min(32 * NW, q_len * group - first_row);
    const int lo = pl_first_visible(start + first_row / group, a.window), hi = start + (first_row + rows - 1) / group + 1;
    const int shares = a8_shares(lo, hi, a.chunk);
    if (share >= shares) return;
    const int k_base = (lo / a.chunk + share) * a.chunk;
    const int k_begin = max(lo, k_base), k_end = min(hi, k_base + a.chunk);

    // This wave's rows.
    const int row = first_row + 32 * wave + col;
    const bool active = 32 * wave < rows, live = 32 * wave + col < rows;
    const int token = live ? row / group : (first_row + (active ? 32 * wave : 0)) / group, head = kvh * group + (live ? row % group : 0);
    // the keys of the share that the lane's row sees: the first and how many
    const int seen_from = max(pl_first_visible(start + token, a.window), k_begin), seen = max(min(start + token + 1, k_end) - seen_from, 0);
    const int first_pos = start + (first_row + (active ? 32 * wave : 0)) / group, last_pos = start + (first_row + min(32 * wave + 32, rows) - 1) / group;
    const int wave_from = pl_first_visible(first_pos, a.window), last_from = pl_first_visible(last_pos, a.window);
    a8_frag qf[2 * DT][PIECES];
#pragma unroll
    for (int j = 0; j < 2 * DT; ++j) {
        const int at = 16 * j + 8 * half;
        a8_query8<PIECES>(a, static_cast<size_t>(q_start + token) * a.q_stride + static_cast<size_t>(head) * a.d + at, live && at < a.d, qf[j]);
    }

    // Tiles on their way: 16 bytes a lane and load, 2 DT lanes a key.  The pages of a tile are asked for a round before its bytes, so that no round waits for one read behind another.
    constexpr int VP = 2 * DT, LOADS = (TILE * VP + THREADS - 1) / THREADS;
    struct Bytes {
        a8_u32x4 k[LOADS], v[LOADS];
        uint32_t k_power[LOADS], v_power[LOADS];      // (as they come: made into a unit where they are read they would be waited for there)
    };
    struct Places {
        int page[LOADS], off[LOADS];
    };
    // (No load stands under a condition: what comes behind one is waited for where the paths meet.  A lane without a piece of a head reads the last one, whose products the queries' zeros take out.)
    const int last_piece = a.d / 16 - 1;
    auto look = [&](int k0, Places& to) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int at = i * THREADS + tid;
            const int key = min(max(k0 + at / VP, k_begin), k_end - 1);      // (keys that no row sees are read at the nearest one's place)
            const int index = a8_page_index(a, key);
            to.off[i] = key - index * a.block;
            to.page[i] = a.table[static_cast<size_t>(seq) * a.width + min(index, a.width - 1)];
        }
    };
    auto fetch = [&](const Places& at, Bytes& to) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int piece = min((i * THREADS + tid) % VP, last_piece);
            const int page = static_cast<unsigned>(at.page[i]) < static_cast<unsigned>(a.pages) ? at.page[i] : 0;
            const size_t from = (static_cast<size_t>(page * a.block + at.off[i]) * a.nkv + kvh) * a.d + 16 * piece;
            to.k[i] = *reinterpret_cast<const a8_u32x4*>(a.k_pool + from);
            to.v[i] = *reinterpret_cast<const a8_u32x4*>(a.v_pool + from);
            to.k_power[i] = a.k_scale[static_cast<size_t>(page) * a.nkv + kvh];
            to.v_power[i] = a.v_scale[static_cast<size_t>(page) * a.nkv + kvh];
        }
    };
    auto put = [&](const Bytes& from, int k_buffer, int v_buffer) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int at = i * THREADS + tid, key = at / VP, piece = at % VP;
            if (TILE * VP % THREADS != 0 && at >= TILE * VP) continue;
            a8_frag to[2];
#pragma unroll
            for (int e = 0; e < 4; ++e) to[e / 2].half[e % 2] = a8_widen4(from.k[i][e], a8_unit(from.k_power[i]));
            uint16_t* k_to = keys + (k_buffer * TILE + key) * KROW + 16 * piece;
            *reinterpret_cast<a8_u32x4*>(k_to) = to[0].raw;
            *reinterpret_cast<a8_u32x4*>(k_to + 8) = to[1].raw;
#pragma unroll
            for (int e = 0; e < 4; ++e) to[e / 2].half[e % 2] = a8_widen4(from.v[i][e], a8_unit(from.v_power[i]));
            uint16_t* v_to = values + (v_buffer * TILE + key) * VROW + 16 * piece;
            *reinterpret_cast<a8_u32x4*>(v_to) = to[0].raw;
            *reinterpret_cast<a8_u32x4*>(v_to + 8) = to[1].raw;
        }
    };

    Bytes bytes;
    Places places;
    a8_f32x16 acc[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[t][i] = 0.f;
    float m = -INFINITY, l = 0.f, top = -INFINITY;

    const int k_first = k_begin / TILE * TILE, tiles = pl_ceil_div(k_end - k_first, TILE);
    // The wave's rows see something of the tile at k0, or all of it.
    auto sees = [&](int k0) { return active && k0 <= last_pos && k0 + TILE > wave_from; };
    auto whole = [&](int k0) { return k0 >= k_begin && k0 >= last_from && k0 + TILE <= k_end && k0 + TILE - 1 <= first_pos; };
    auto scores = [&](a8_f32x16 (&s)[KB], int buffer) {
        const uint16_t* from = keys + (buffer * TILE + col) * KROW + 8 * half;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[kb][i] = 0.f;
#pragma unroll
        for (int j = 0; j < 2 * DT; ++j)
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                a8_frag kf;
                kf.raw = *reinterpret_cast<const a8_u32x4*>(from + 32 * kb * KROW + 16 * j);
#pragma unroll
                for (int p = PIECES - 1; p >= 0; --p) s[kb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf.vec, qf[j][p].vec, s[kb], 0, 0, 0);
            }
    };
    // (Values are chosen under the branch and put back behind it, as in the kernel of few rows: see there.)
    auto mask = [&](a8_f32x16 (&s)[KB], int k0) {
        float x[16 * KB];
#pragma unroll
        for (int i = 0; i < 16 * KB; ++i) x[i] = s[i / 16][i % 16];
        if (!whole(k0)) {
#pragma unroll
            for (int i = 0; i < 16 * KB; ++i) {
                const int key = k0 + 32 * (i / 16) + 8 * (i % 16 / 4) + 4 * half + i % 4;
                x[i] = static_cast<unsigned>(key - seen_from) < static_cast<unsigned>(seen) ? x[i] : -INFINITY;
            }
        }
#pragma unroll
        for (int i = 0; i < 16 * KB; ++i) s[i / 16][i % 16] = x[i];
    };
    auto largest = [&](const a8_f32x16 (&s)[KB]) {
        float most = s[0][0];
#pragma unroll
        for (int i = 1; i < 16 * KB; ++i) most = fmaxf(most, s[i / 16][i % 16]);
        return a8_max_half(most) * a.scale;
    };
    // Round t: this tile's weights and values, the next one's scores, the one's bytes behind that.
    int v_now = 0;
    auto round = [&](a8_f32x16 (&s)[KB], a8_f32x16 (&next)[KB], int t) {
        const int k0 = k_first + t * TILE, v_put = v_now == 0 ? 2 : v_now - 1;
        if (sees(k0)) {
            // Weights are taken relative to a maximum that is at most 2^8 off: sums and outputs are scaled anew only where a row's maximum has grown by more.
            if (__any(top > m + 8.f)) {
                const float grown = fmaxf(m, top);
                const float alpha = __builtin_amdgcn_exp2f(m - (grown == -INFINITY ? 0.f : grown));
                m = grown;
                l *= alpha;
#pragma unroll
                for (int t = 0; t < DT; ++t)
#pragma unroll
                    for (int i = 0; i < 16; ++i) acc[t][i] *= alpha;
            }
            const float from = m == -INFINITY ? 0.f : m;
            scores(next, (t + 1) % 2);
            a8_frag pf[2 * KB][PIECES];
            float sum = 0.f;
#pragma unroll
            for (int g = 0; g < 2 * KB; ++g) {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x[e] = __builtin_amdgcn_exp2f(fmaf(s[g / 2][8 * (g % 2) + e], a.scale, -from));
                    sum += x[e];
                }
                a8_split<PIECES>(x, pf[g]);
            }
            l += sum;
            // (Both orders of work are put side by side here: between two products on the matrix cores, their operands' read and a share of the weights.  Made by the
            // compiler, the weights follow the products, and even go behind the branch below.)
            __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
            for (int i = 0; i < 2 * DT * KB; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x8, PIECES, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x402, PIECES == 1 ? (28 + 2 * DT - 1) / (2 * DT) : (56 + 2 * DT - 1) / (2 * DT), 0);
            }
#pragma unroll
            for (int g = 0; g < 2 * KB; ++g)
#pragma unroll
                for (int p = 0; p < PIECES; ++p) asm volatile("" : "+v"(pf[g][p].raw));
            mask(next, k0 + TILE);
            top = largest(next);
            const uint16_t* v_from = values + (v_now * TILE + 4 * half + lane % 16 / 4) * VROW + 16 * (lane / 16 % 2) + 4 * (lane % 4);
            // (In this order, AHEAD reads before the product that needs the first: left to itself the compiler waits for every pair of them.  Other instructions may move across.)
            constexpr int PRODUCTS = 2 * KB * DT, AHEAD = PRODUCTS < 6 ? PRODUCTS : 6;
            a8_frag vf[AHEAD];
            auto read_values = [&](int i) {
                const uint16_t* at = v_from + 16 * (i / DT) * VROW + 32 * (i % DT);
                vf[i % AHEAD].half[0] = a8_read_transposed(at);
                vf[i % AHEAD].half[1] = a8_read_transposed(at + 8 * VROW);
            };
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) read_values(i);
#pragma unroll
            for (int i = 0; i < PRODUCTS; ++i) {
                __builtin_amdgcn_sched_barrier(0x6);
#pragma unroll
                for (int p = PIECES - 1; p >= 0; --p) acc[i % DT] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[i % AHEAD].vec, pf[i / DT][p].vec, acc[i % DT], 0, 0, 0);
                if (i + AHEAD < PRODUCTS) read_values(i + AHEAD);
            }
            __builtin_amdgcn_sched_barrier(0x6);
        } else if (sees(k0 + TILE)) {
            scores(next, (t + 1) % 2);
            mask(next, k0 + TILE);
            top = largest(next);
        }
        put(bytes, t % 2, v_put);
        fetch(places, bytes);
        look(k0 + 4 * TILE, places);
        v_now = v_now == 2 ? 0 : v_now + 1;
        __syncthreads();
    };

    // (beyond the last tile the nearest key is read once more: no round goes by whether there is a next one)
    {
        Places second;
        Bytes first;
        look(k_first, places);
        look(k_first + TILE, second);
        fetch(places, first);
        look(k_first + 2 * TILE, places);
        fetch(second, bytes);
        put(first, 0, 0);
        put(bytes, 1, 1);
        fetch(places, bytes);
        look(k_first + 3 * TILE, places);
    }
    __syncthreads();
    a8_f32x16 s[2][KB];
    if (sees(k_first)) {
        scores(s[0], 0);
        mask(s[0], k_first);
        top = largest(s[0]);
    }
    __syncthreads();
    for (int t = 0; t < tiles; t += 2) {
        round(s[0], s[1], t);
        if (t + 1 < tiles) round(s[1], s[0], t + 1);
    }
    l += __shfl_xor(l, 32, PL_WAVE);
    uint32_t again = 0;                       // rows that are worked out once more
    if (k_begin < last_from || k_end - 1 > first_pos) {          // (not all of the wave's rows see all keys of the share)
        float finite = 0.f;                   // (or NaN)
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) finite = fmaf(acc[t][i], 0.f, finite);
        const uint64_t bad = __ballot(live && finite != finite && l == l);          // (weights that are NaN leave nothing else)
        again = static_cast<uint32_t>(bad | bad >> 32);
    }
    if (!active) return;

    const size_t out_row = static_cast<size_t>(q_start + token) * a.nq + head, place = out_row * a.parts + share;
    if (live) {
        float inv = 1.f;
        if (a.chunks == 1) {
            if (shares > 1) l = NAN;              // (a context longer than the caller said)
            inv = l != 0.f ? 1.f / l : 0.f;
        } else if (half == 0) {
            a.part_ml[2 * place] = m;
            a.part_ml[2 * place + 1] = l;
        }
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int at = 32 * t + 8 * i + 4 * half;
                if (at >= a.d) continue;
                if (a.chunks == 1) a8_store4<PIECES>(a, out_row * a.d + at, acc[t][4 * i] * inv, acc[t][4 * i + 1] * inv, acc[t][4 * i + 2] * inv, acc[t][4 * i + 3] * inv);
                else *reinterpret_cast<a8_f32x4*>(a.part_acc + place * a.d + at) = a8_f32x4{acc[t][4 * i], acc[t][4 * i + 1], acc[t][4 * i + 2], acc[t][4 * i + 3]};
            }
    }
    if (again == 0 || (a.chunks == 1 && shares > 1)) return;
    __threadfence_block();
    for (; again != 0; again &= again - 1) {
        const int r = first_row + 32 * wave + __ffs(again) - 1, of = r / group, query = kvh * group + r % group;
        a8_row_alone<PIECES>(a8_args_again(), seq, kvh, max(pl_first_visible(start + of, a.window), k_begin), min(start + of + 1, k_end), max(k_begin, wave_from - TILE), min(k_end, last_pos + TILE + 1), q_start + of,
                             (static_cast<size_t>(q_start + of) * a.nq + query) * a.parts + share, a.chunks == 1, query);
    }
}

// ---- shares put together ---------------------------------------------------------------------------------------------------
// A wave a row and query head: the shares that its block of rows had, in their order.  (A request of few rows is one block.)
// Rows of either kernel, those of many (`tall` workgroups, `many_groups` for a block of `per` rows and a key head) before those of few (`few_groups` for a request and key head): side by side, since each is
// a chain of reads (512 tokens behind 4,100 beside 15 single ones: 11 us in one launch, 12 and 5 in two).
struct A8Merge {
    A8Args many, few;
    int tall, per, many_groups, few_groups;
    int above, few_rows;      // rows of a request that are too few for the kernel of many, and as many as the kernel of few took
};

template <typename T>
__global__ __launch_bounds__(A8_WAVES * PL_WAVE) void attention_8bit_merge_kernel(A8Merge g) {
    const int lane = threadIdx.x % PL_WAVE;
    const bool tall = static_cast<int>(blockIdx.x) < g.tall;
    const A8Args& a = tall ? g.many : g.few;
    const int group = a.nq / a.nkv, few = tall ? g.above : g.few_rows, per = tall ? g.per : 0;
    const int every = tall ? g.many_groups : g.few_groups, block = static_cast<int>(blockIdx.x) - (tall ? 0 : g.tall);
    const int kvh = block / every % a.nkv;
    int seq = block / every / a.nkv, rb = 0;
    if (tall) {
        if (!a8_find(a, seq, group, per, few, seq, rb)) return;
    } else if (!a8_brings(a, seq) || a.q_len[seq] * group > few) {
        return;
    }
    const int q_len = a.q_len[seq], start = a.ctx_len[seq] - q_len;
    const int first_row = rb * per, rows = min(tall ? per : few, q_len * group - first_row);
    const int lo = pl_first_visible(start + first_row / group, a.window), hi = start + (first_row + rows - 1) / group + 1;
    int all = a8_shares(lo, hi, a.chunk);
    if (!tall && a.most > a.chunk) {
        all = a.cut[seq];
        if (all == 1) return;             // (written as they are)
    }
    const int shares = min(all, a.chunks);
    const int waves = A8_WAVES * every;
    const int lanes = a.d <= 32 ? 8 : a.d <= 64 ? 16 : a.d <= 128 ? 32 : 64;        // of a share's row; the wave takes several shares at a time
    for (int r = threadIdx.x / PL_WAVE + A8_WAVES * (block % every); r < rows; r += waves) {
        const int row = first_row + r;
        const size_t out_row = static_cast<size_t>(a.q_start[seq] + row / group) * a.nq + kvh * group + row % group;
        const size_t place = a8_place(a, seq, kvh, row, out_row) * a.parts;
        const float *ml = a.part_ml + 2 * place, *acc = a.part_acc + place * a.d;
        float top = -INFINITY, total = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
        const int at = 4 * (lane % lanes), from_at = min(at, a.d - 4);
        for (int base = 0; base < shares; base += PL_WAVE) {
            // (a lane has one share's maximum and sum; the shares' rows are asked for without regard to them, eight reads at once)
            const int here = min(shares - base, PL_WAVE), own = min(lane, here - 1);
            const float m = lane < here ? ml[2 * (base + own)] : -INFINITY, l = ml[2 * (base + own) + 1];
            const float grown = fmaxf(top, wave_max(m)), from = grown == -INFINITY ? 0.f : grown;
            const float weight = __builtin_amdgcn_exp2f(m - from), alpha = __builtin_amdgcn_exp2f(top - from);
            top = grown;
            total = total * alpha + (lane < here ? weight * l : 0.f);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] *= alpha;
#pragma unroll 8
            for (int i = 0; i < here; i += PL_WAVE / lanes) {
                const int s = i + lane / lanes;
                const a8_f32x4 y = *reinterpret_cast<const a8_f32x4*>(acc + static_cast<size_t>(base + min(s, here - 1)) * a.d + from_at);
                const float w = __shfl(weight, s % PL_WAVE, PL_WAVE);
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] += s < here ? w * y[e] : 0.f;
            }
        }
        total = wave_sum(total);
        for (int off = lanes; off < PL_WAVE; off <<= 1) {
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] += __shfl_xor(x[e], off, PL_WAVE);
        }
        if (all > shares) total = NAN;        // (a context longer than the caller said)
        const float inv = total != 0.f ? 1.f / total : 0.f;
        if (lane < lanes && at < a.d) {
            struct __attribute__((aligned(4 * sizeof(T)))) Piece {
                T v[4];
            } to;
#pragma unroll
            for (int e = 0; e < 4; ++e) to.v[e] = from_float<T>(x[e] * inv);
            *reinterpret_cast<Piece*>(static_cast<T*>(a.out) + out_row * a.d + at) = to;
        }
    }
}

static int a8_lds(const void* kernel, size_t lds) {
    if (lds <= 64 * 1024) return 0;
    hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds));
    PL_REQUIRE(e == hipSuccess, "8-bit attention: %zu bytes of LDS refused: %s", lds, hipGetErrorString(e));
    return 0;
}

// Workgroups of the kernel of few rows that a compute unit's registers hold.
static int a8_held(const void* kernel) {
    int held = 0;
    return hipOccupancyMaxActiveBlocksPerMultiprocessor(&held, kernel, A8_WAVES * PL_WAVE, 0) == hipSuccess && held > 0 ? held : 1;
}

template <int PIECES, int DQ, int RB>
static int launch_few(A8Args& a, int rows, A8Merge& merge, hipStream_t stream) {
    PL_REQUIRE(a8_grid(a, a.S, a.chunks) < (1l << 31), "8-bit attention: %d requests in %d shares are too many for a launch", a.S, a.chunks);
    auto room = [](int keys) { return static_cast<size_t>(A8_WAVES) * A8_KEYS * (64 * DQ + 16) * 2 + A8_WAVES * 2 * 16 * RB * 4 + static_cast<size_t>(keys) * 6; };
    a.most = a.chunk;
    const long longest = static_cast<long>(a.chunk) * a.chunks;
    if (a.S <= PL_WAVE && a.chunks > 1) {
        // (as many workgroups a unit as its registers hold, and fewer only where LDS could not hold longer shares of so many)
        static const int by_registers = a8_held(reinterpret_cast<const void*>(&attention_8bit_few_kernel<PIECES, DQ, RB, true>));
        int held = by_registers;
        // (LDS is given out in pieces of 1,280 bytes: three of 54,080, which are less than 160 KB, do not fit)
        auto fits = [&](int held) { return (160l * 1024 / held / 2560 * 2560 - static_cast<long>(room(0))) / 6 / A8_KEYS * A8_KEYS; };
        while (held > 1 && fits(held) <= a.chunk) --held;
        a.places = pl_compute_units() * held;
        if (static_cast<long>(a.S) * a.nkv * a.chunks > a.places) a.most = static_cast<int>(max(static_cast<long>(a.chunk), min(longest, min(fits(held), static_cast<long>(A8_MOST_BALANCED)))));
    }
    long grid = a8_grid(a, a.S, a.chunks);
    if (a.most > a.chunk) {
        // (no more workgroups than the rounds that the longest contexts could take: thousands without work would take turns on the chip)
        const long rounds = (a.S * ((longest + a.most - 1) / a.most) * a.nkv + a.places - 1) / a.places, shares = min(static_cast<long>(a.S) * a.chunks, rounds * a.places / a.nkv);
        grid = a8_grid(a, shares, 1);
    }
    const size_t lds = room(a.most);
    auto launch = [&](auto kernel) {
        if (int e = a8_lds(reinterpret_cast<const void*>(kernel), lds)) return e;
        kernel<<<static_cast<unsigned>(grid), A8_WAVES * PL_WAVE, lds, stream>>>(a);
        return 0;
    };
    if (int e = a.most > a.chunk ? launch(&attention_8bit_few_kernel<PIECES, DQ, RB, true>) : launch(&attention_8bit_few_kernel<PIECES, DQ, RB, false>)) return e;
    PL_CHECK_LAUNCH("attention_8bit_few");
    merge.few_groups = pl_ceil_div(rows, A8_WAVES);
    merge.few_rows = 16 * RB;
    return 0;
}

template <int PIECES, int DQ>
static int launch_few(A8Args& a, int rows, A8Merge& merge, hipStream_t stream) {
    constexpr int MOST = A8Few<PIECES, DQ>::BLOCKS;
    if (rows <= 16 || MOST == 1) return launch_few<PIECES, DQ, 1>(a, rows, merge, stream);
    if constexpr (MOST >= 2)
        if (rows <= 32 || MOST == 2) return launch_few<PIECES, DQ, 2>(a, rows, merge, stream);
    if constexpr (MOST >= 4) {
        if (rows <= 48) return launch_few<PIECES, DQ, 3>(a, rows, merge, stream);
        return launch_few<PIECES, DQ, 4>(a, rows, merge, stream);
    }
    return 0;
}

template <int PIECES>
static int launch_few(A8Args& a, int rows, A8Merge& merge, hipStream_t stream) {
    switch (pl_ceil_div(a.d, 64)) {
        case 1: return launch_few<PIECES, 1>(a, rows, merge, stream);
        case 2: return launch_few<PIECES, 2>(a, rows, merge, stream);
        case 3: return launch_few<PIECES, 3>(a, rows, merge, stream);
        default: return launch_few<PIECES, 4>(a, rows, merge, stream);
    }
}

template <int PIECES, int DT, int NW>
static int launch_many(const A8Args& a, int few, long blocks, A8Merge& merge, hipStream_t stream) {
    const size_t lds = A8Many<PIECES, DT>::LDS;
    if (int e = a8_lds(reinterpret_cast<const void*>(&attention_8bit_many_kernel<PIECES, DT, NW>), lds)) return e;
    PL_REQUIRE(a8_grid(a, blocks, a.chunks) < (1l << 31) && blocks * a.nkv * 4 * NW < (1l << 31), "8-bit attention: %ld blocks of rows in %d shares are too many for a launch", blocks, a.chunks);
    attention_8bit_many_kernel<PIECES, DT, NW><<<static_cast<unsigned>(a8_grid(a, blocks, a.chunks)), NW * PL_WAVE, lds, stream>>>(a, few, static_cast<int>(blocks));
    PL_CHECK_LAUNCH("attention_8bit_many");
    if (a.chunks > 1) {
        merge.per = 32 * NW;
        merge.many_groups = 4 * NW;
        merge.tall = static_cast<int>(blocks * a.nkv * merge.many_groups);
    }
    return 0;
}

template <int PIECES, int DT, int NW>
static int launch_many_blocks(const A8Args& a, int few, int max_q_len, A8Merge& merge, hipStream_t stream) {
    const int group = a.nq / a.nkv;
    // blocks of rows: one a request for what is left over, and the whole ones
    const long most = static_cast<long>(a.S) * ((static_cast<long>(max_q_len) * group + 32 * NW - 1) / (32 * NW)), all = a.S + static_cast<long>(a.n) * group / (32 * NW);
    return launch_many<PIECES, DT, NW>(a, few, most < all ? most : all, merge, stream);
}

// Four waves a workgroup where eight's registers or LDS leave no second one beside it anyway (32 bits, heads of more than 128) or where two of four fit a unit (heads of up to 64: 2 prompts of 1,500 to 2,000 tokens,
// 16 heads over 8, 45 us with eight, 40 with four); else eight, which widen a tile for 256 rows, but for so few rows that workgroups of 128 do not fill the chip either (512 tokens of 16 heads over 8: 23.5 and 20.8 us).
static int a8_waves(int n, int nq, int nkv, int d, int chunks, int dtype) {
    const long blocks = (static_cast<long>(n) * (nq / nkv) + 127) / 128 * nkv * chunks;
    return dtype == PL_DTYPE_BF16 && d > 64 && d <= 128 && blocks > 256 ? 8 : 4;
}

template <int PIECES, int DT>
static int launch_many(const A8Args& a, int few, int max_q_len, A8Merge& merge, hipStream_t stream) {
    if constexpr (PIECES == 1 && (DT == 3 || DT == 4))
        if (a8_waves(a.n, a.nq, a.nkv, a.d, a.chunks, PL_DTYPE_BF16) == 8) return launch_many_blocks<PIECES, DT, 8>(a, few, max_q_len, merge, stream);
    return launch_many_blocks<PIECES, DT, 4>(a, few, max_q_len, merge, stream);
}

template <int PIECES>
static int launch_many(const A8Args& a, int few, int max_q_len, A8Merge& merge, hipStream_t stream) {
    switch (pl_ceil_div(a.d, 32)) {
        case 1: return launch_many<PIECES, 1>(a, few, max_q_len, merge, stream);
        case 2: return launch_many<PIECES, 2>(a, few, max_q_len, merge, stream);
        case 3: return launch_many<PIECES, 3>(a, few, max_q_len, merge, stream);
        case 4: return launch_many<PIECES, 4>(a, few, max_q_len, merge, stream);
        case 5:
        case 6: return launch_many<PIECES, 6>(a, few, max_q_len, merge, stream);
        default: return launch_many<PIECES, 8>(a, few, max_q_len, merge, stream);
    }
}

// The most rows (tokens times query heads a key head) of a request that the kernel of few rows takes.
extern "C" int pl_paged_attention_8bit_few(int d, int dtype) {
    const int dq = pl_ceil_div(d, 64);
    if (dtype == PL_DTYPE_F32) return 16 * (dq == 1 ? A8Few<3, 1>::BLOCKS : dq == 2 ? A8Few<3, 2>::BLOCKS : A8Few<3, 3>::BLOCKS);
    return 16 * (dq <= 2 ? A8Few<1, 2>::BLOCKS : A8Few<1, 3>::BLOCKS);
}

// The waves of a workgroup of the kernel of many rows, for `chunks` shares.
extern "C" int pl_paged_attention_8bit_waves(int n, int nq, int nkv, int d, int chunks, int dtype) { return nkv >= 1 ? a8_waves(n, nq, nkv, d, chunks, dtype) : 0; }

// Which kernels a step needs and what room their shares take, in rows of d values (and two numbers more): nothing for a kernel that does not run or has one share.
struct A8Plan {
    bool few_runs, many_runs;
    int few;                  // a request's rows (tokens times query heads a key head) that the kernel of few takes, at most
    int rows, rows_each;      // and may bring; A8Args::rows_each
    long few_places, many_places;
};
static A8Plan a8_plan(int S, int n, int max_q_len, int min_q_len, int nq, int nkv, int d, int few_chunks, int many_chunks, int dtype) {
    const long group = nq / nkv, longest = max_q_len * group, all = static_cast<long>(n) * nq;
    A8Plan p{};
    // In a step of portions only what 16 rows hold goes to the kernel of few: those are the single tokens beside them, for which its smallest form is the fastest
    // (15 single tokens at up to 4,600 keys beside a portion: 32 us with it, 91 with the form for 64 rows).
    p.few = pl_paged_attention_8bit_few(d, dtype);
    p.many_runs = longest > p.few;
    if (p.many_runs) p.few = 16;
    p.few_runs = min_q_len * group <= p.few;
    p.rows = static_cast<int>(longest < p.few ? longest : p.few);
    // (as many as the build for so many rows holds: a request that brings more than it was said to stays inside its own)
    const int held = pl_ceil_div(p.rows, 16) * 16;
    const long each = static_cast<long>(S) * nkv * held;
    if (each < all) p.rows_each = held;
    if (p.few_runs && few_chunks > 1) p.few_places = (each < all ? each : all) * few_chunks;
    if (p.many_runs && many_chunks > 1) p.many_places = all * many_chunks;
    return p;
}

// How many rows of room pl_paged_attention_8bit needs for a step's shares.
extern "C" long long pl_paged_attention_8bit_places(int S, int n, int max_q_len, int min_q_len, int nq, int nkv, int d, int few_chunks, int many_chunks, int dtype) {
    if (nkv < 1 || nq < nkv || d < 1) return 0;
    const A8Plan plan = a8_plan(S, n, max_q_len, min_q_len, nq, nkv, d, few_chunks, many_chunks, dtype);
    return plan.few_places + plan.many_places;
}

// The kernel of few rows and that of many have shares of their own size.  `part_acc` has room for d floats for each of pl_paged_attention_8bit_places(...), those of many rows first;
// `part_ml` for two, and for S more behind those.
extern "C" int pl_paged_attention_8bit(const void* q, int q_stride, void* out, const void* q_start, const void* q_len, const void* ctx_len, int S, int n, int max_q_len, int min_q_len,
                                       const void* table, int width, int block, int pool_rows, const void* k_pool, const void* v_pool, const void* k_scale,
                                       const void* v_scale, int nq, int nkv, int d, float scale, int window, int few_chunk, int few_chunks, int many_chunk, int many_chunks,
                                       void* part_acc, void* part_ml, int dtype, void* stream) {
    PL_REQUIRE(d >= 16 && d <= 256 && d % 16 == 0, "8-bit attention: head size %d, the kernels take multiples of 16 up to 256", d);
    PL_REQUIRE(nkv >= 1 && nq >= nkv && nq % nkv == 0, "8-bit attention: %d query heads over %d key heads", nq, nkv);
    PL_REQUIRE(S >= 1 && n >= 1 && max_q_len >= 1 && min_q_len <= max_q_len && width >= 1 && block >= 1 && pool_rows >= block,
               "8-bit attention: %d requests, %d rows, %d to %d of one request, tables of %d pages of %d, %d rows", S, n, min_q_len, max_q_len, width, block, pool_rows);
    PL_REQUIRE(static_cast<long>(n) * nq < (1l << 31) && (static_cast<long>(S) + 8) * nkv < (1l << 31), "8-bit attention: %d rows of %d heads, %d requests are too many for a launch", n, nq, S);
    PL_REQUIRE(few_chunk >= A8_KEYS && few_chunk % A8_KEYS == 0 && few_chunk <= A8_MOST_KEYS && few_chunks >= 1 && few_chunks < 65536,
               "8-bit attention: %d shares of %d keys", few_chunks, few_chunk);
    PL_REQUIRE(many_chunk >= 64 && many_chunk % 64 == 0 && many_chunks >= 1 && many_chunks < 65536,
               "8-bit attention: %d shares of %d keys", many_chunks, many_chunk);
    const A8Plan plan = a8_plan(S, n, max_q_len, min_q_len, nq, nkv, d, few_chunks, many_chunks, dtype);
    PL_REQUIRE(plan.few_places + plan.many_places == 0 || (part_acc && part_ml), "8-bit attention: no room for %ld rows of shares", plan.few_places + plan.many_places);
    const int shift = 31 + (block > 1 ? 32 - __builtin_clz(block - 1) : 0);
    const uint32_t magic = static_cast<uint32_t>(((uint64_t{1} << shift) + block - 1) / block);
    A8Args a{q, q_stride, out, static_cast<const int*>(q_start), static_cast<const int*>(q_len), static_cast<const int*>(ctx_len), S, static_cast<const int*>(table), width, block, magic, shift, pool_rows / block,
             static_cast<const uint8_t*>(k_pool), static_cast<const uint8_t*>(v_pool), static_cast<const uint8_t*>(k_scale), static_cast<const uint8_t*>(v_scale),
             nq, nkv, d, a8_beside(nkv, d), scale * 1.4426950408889634f, window, n, few_chunk, few_chunks, few_chunk, 0, static_cast<float*>(part_acc), static_cast<float*>(part_ml), few_chunks, 0, nullptr};
    const hipStream_t on = static_cast<hipStream_t>(stream);
    const bool f32 = dtype == PL_DTYPE_F32;
    A8Merge merge{a, a, 0, 0, 1, 1, plan.few, 0};
    long groups = 0;
    if (plan.few_runs) {
        merge.few.rows_each = plan.rows_each;
        if (plan.few_places > 0) {
            merge.few.part_acc += plan.many_places * d;
            merge.few.part_ml += plan.many_places * 2;
            merge.few.cut = reinterpret_cast<int*>(merge.few.part_ml + plan.few_places * 2);
        }
        if (int e = f32 ? launch_few<3>(merge.few, plan.rows, merge, on) : launch_few<1>(merge.few, plan.rows, merge, on)) return e;
        if (few_chunks > 1) groups = static_cast<long>(S) * nkv * merge.few_groups;
    }
    if (plan.many_runs) {
        merge.many.chunk = many_chunk;
        merge.many.chunks = merge.many.parts = many_chunks;
        if (int e = f32 ? launch_many<3>(merge.many, plan.few, max_q_len, merge, on) : launch_many<1>(merge.many, plan.few, max_q_len, merge, on)) return e;
        groups += merge.tall;
    }
    if (groups == 0) return 0;
    PL_REQUIRE(groups < (1l << 31), "8-bit attention: shares of %d requests are too many for a launch", S);
    if (f32) attention_8bit_merge_kernel<float><<<static_cast<unsigned>(groups), A8_WAVES * PL_WAVE, 0, on>>>(merge);
    else attention_8bit_merge_kernel<bf16_t><<<static_cast<unsigned>(groups), A8_WAVES * PL_WAVE, 0, on>>>(merge);
    PL_CHECK_LAUNCH("attention_8bit_merge");
    return 0;
}
