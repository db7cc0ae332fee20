// Attention over a paged cache held in 8 bits (pages of e4m3 with a power of two for each page and key head).
//
//   out = softmax(scale q . k) v,   k = 2^Ek[page] e4m3,   v = 2^Ev[page] e4m3
//
// An e4m3 value times a power of two is exact in bfloat16, so keys and values become bfloat16 in one instruction for two of them
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
// Maximum, sum, weights and output are 32-bit; exponentials are base 2 with log2(e) folded into the scale.
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

#define A8_ROWS 32       // rows a wave
#define A8_KEYS 32       // keys a tile
#define A8_WAVES 4

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
    int width, block, pool_rows;
    const uint8_t *k_pool, *v_pool, *k_scale, *v_scale;
    int nq, nkv, d;
    float scale;              // times log2(e)
    int window;
    int n, chunk, chunks;     // rows of the step; keys a workgroup, and how many such shares the longest context has
    float *part_acc, *part_ml;
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

// Elements that a row of values in LDS is padded by: a row then begins 16 banks (of 64) further than the one before, so the four rows of 64 bytes
// that 32 lanes read transposed fall on every bank once.
__host__ __device__ constexpr int a8_pad(int dt) { return dt % 2 == 0 ? 32 : 0; }

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

// Which request and which of its blocks of rows is number `slot`, counted over the requests one after the other; by a whole wave.
__device__ __forceinline__ bool a8_find(const A8Args& a, int slot, int group, int rows, int& seq, int& block) {
    const int lane = threadIdx.x % PL_WAVE;
    for (int base = 0; base < a.S; base += PL_WAVE) {
        const int s = base + lane;
        int blocks = 0;
        // (a request whose context is shorter than what it brings holds the rows of a padded step)
        if (s < a.S && a.q_len[s] > 0 && a.ctx_len[s] >= a.q_len[s] && a.q_start[s] >= 0 && a.q_start[s] <= a.n - a.q_len[s]) blocks = pl_ceil_div(a.q_len[s] * group, rows);
        int end = blocks;
#pragma unroll
        for (int off = 1; off < PL_WAVE; off <<= 1) {
            const int up = __shfl_up(end, off, PL_WAVE);
            if (lane >= off) end += up;
        }
        const uint64_t past = __ballot(end > slot);
        if (past != 0) {
            const int first = __ffsll(static_cast<unsigned long long>(past)) - 1;
            seq = base + first;
            block = slot - (__shfl(end, first, PL_WAVE) - __shfl(blocks, first, PL_WAVE));
            return true;
        }
        slot -= __shfl(end, PL_WAVE - 1, PL_WAVE);
    }
    return false;
}

// The keys [lo, hi) that a block of rows sees, cut into shares of `chunk` that begin at whole chunks: how many there are.
__device__ __forceinline__ int a8_shares(int lo, int hi, int chunk) { return hi > lo ? (hi - 1) / chunk - lo / chunk + 1 : 0; }

// ---- few rows: every wave has keys of its own ------------------------------------------------------------------------------
// A workgroup takes one block of 32 rows of one key head and one share of the keys; its waves take tiles of 32 keys in turn, each with a running maximum and sum, and meet at the end.
// Keys go from memory into the registers that the product reads (a lane reads 16 bytes of one key: the contraction may go through a head's values in any order, so the
// queries are laid out to match); values go through a piece of LDS that belongs to the wave, so the loop has no barrier.
template <int PIECES, int DT>
__global__ __launch_bounds__(A8_WAVES * PL_WAVE, PIECES * DT >= 8 && DT != 4 ? 1 : 2) void attention_8bit_kernel(A8Args a) {
    typedef typename A8Type<PIECES>::type T;
    constexpr int DP = 32 * DT, VROW = DP + a8_pad(DT);
    constexpr int MEET = 2 * A8_ROWS * (DP + 4) * 4;         // two waves' outputs, behind the loop
    constexpr int VALUES = A8_WAVES * A8_KEYS * VROW * 2;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    uint16_t* values = reinterpret_cast<uint16_t*>(lds);
    int* slots = reinterpret_cast<int*>(lds + (MEET > VALUES ? MEET : VALUES));
    float* k_unit = reinterpret_cast<float*>(slots + a.chunk);
    float* v_unit = k_unit + a.chunk;
    float* stats = v_unit + a.chunk;                         // [waves][2][rows]

    const int tid = threadIdx.x, lane = tid % PL_WAVE, wave = tid / PL_WAVE;
    const int col = lane % 32, half = lane / 32;
    const int group = a.nq / a.nkv;
    const int kvh = blockIdx.x % a.nkv;
    int seq, rb;
    if (!a8_find(a, blockIdx.x / a.nkv, group, A8_ROWS, seq, rb)) return;
    const int q_len = a.q_len[seq], ctx = a.ctx_len[seq], start = ctx - q_len;
    const int first_row = rb * A8_ROWS, rows = min(A8_ROWS, q_len * group - first_row);
    const int first_token = first_row / group, last_token = (first_row + rows - 1) / group;
    const int lo = pl_first_visible(start + first_token, a.window), hi = start + last_token + 1;
    const int share0 = lo / a.chunk, shares = a8_shares(lo, hi, a.chunk);
    const int share = blockIdx.y;
    if (share >= shares) return;
    const int k_begin = max(lo, (share0 + share) * a.chunk), k_end = min(hi, (share0 + share + 1) * a.chunk);
    const int k_base = (share0 + share) * a.chunk;

    // Where the keys of the share are, and in what units.  (Keys that no row sees are read at the last one's place.)
    for (int i = tid; i < a.chunk; i += A8_WAVES * PL_WAVE) {
        const int key = min(max(k_base + i, k_begin), k_end - 1);
        const int index = key / a.block;
        int page = index < a.width ? a.table[static_cast<size_t>(seq) * a.width + index] : 0;
        page = page < 0 || page >= a.pool_rows / a.block ? 0 : page;
        slots[i] = page * a.block + key % a.block;
        k_unit[i] = __uint_as_float(static_cast<uint32_t>(a.k_scale[static_cast<size_t>(page) * a.nkv + kvh]) << 23);
        v_unit[i] = __uint_as_float(static_cast<uint32_t>(a.v_scale[static_cast<size_t>(page) * a.nkv + kvh]) << 23);
    }

    // The rows: piece 2j + e of a lane's keys are the values 32j + 16 half + 8e ..
    const int row = first_row + col;
    const bool live = col < rows;
    const int token = live ? row / group : first_token, head = kvh * group + (live ? row % group : 0);
    const int position = start + token, seen_from = pl_first_visible(position, a.window);
    a8_frag qf[2 * DT][PIECES];
    {
        const T* from = static_cast<const T*>(a.q) + static_cast<size_t>(a.q_start[seq] + token) * a.q_stride + static_cast<size_t>(head) * a.d;
#pragma unroll
        for (int j = 0; j < 2 * DT; ++j) {
            const int at = 32 * (j / 2) + 16 * half + 8 * (j % 2);
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = live && at < a.d ? to_float(from[at + e]) : 0.f;
            a8_split<PIECES>(x, qf[j]);
        }
    }
    __syncthreads();

    uint16_t* mine = values + wave * A8_KEYS * VROW;
    a8_f32x16 acc[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[t][i] = 0.f;
    float m = -INFINITY, l = 0.f;

    for (int base = wave * A8_KEYS; base < a.chunk; base += A8_WAVES * A8_KEYS) {
        const int k0 = k_base + base;
        if (k0 + A8_KEYS <= k_begin || k0 >= k_end) continue;
        // values: 16 bytes a lane, DP / 16 lanes a key
        constexpr int VP = DP / 16, VLOADS = A8_KEYS * VP / PL_WAVE;
#pragma unroll
        for (int i = 0; i < VLOADS; ++i) {
            const int at = i * PL_WAVE + lane, key = at / VP, piece = at % VP;
            a8_u32x4 raw = {0u, 0u, 0u, 0u};
            if (16 * piece < a.d) raw = *reinterpret_cast<const a8_u32x4*>(a.v_pool + (static_cast<size_t>(slots[base + key]) * a.nkv + kvh) * a.d + 16 * piece);
            const float unit = v_unit[base + key];
            a8_frag to[2];
#pragma unroll
            for (int e = 0; e < 4; ++e) to[e / 2].half[e % 2] = a8_widen4(raw[e], unit);
            *reinterpret_cast<a8_u32x4*>(mine + key * VROW + 16 * piece) = to[0].raw;
            *reinterpret_cast<a8_u32x4*>(mine + key * VROW + 16 * piece + 8) = to[1].raw;
        }
        // scores
        const uint8_t* k_from = a.k_pool + (static_cast<size_t>(slots[base + col]) * a.nkv + kvh) * a.d;
        const float unit = k_unit[base + col];
        a8_f32x16 s;
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
        for (int j = 0; j < DT; ++j) {
            a8_u32x4 raw = {0u, 0u, 0u, 0u};
            const int at = 32 * j + 16 * half;
            if (at < a.d) raw = *reinterpret_cast<const a8_u32x4*>(k_from + at);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                a8_frag kf;
                kf.half[0] = a8_widen4(raw[2 * e], unit);
                kf.half[1] = a8_widen4(raw[2 * e + 1], unit);
#pragma unroll
                for (int p = PIECES - 1; p >= 0; --p) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf.vec, qf[2 * j + e][p].vec, s, 0, 0, 0);
            }
        }
        // weights
        float top = m;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int key = k0 + 8 * (i / 4) + 4 * half + i % 4;
            s[i] = key >= k_begin && key < k_end && key <= position && key >= seen_from ? s[i] * a.scale : -INFINITY;
            top = fmaxf(top, s[i]);
        }
        top = fmaxf(top, __shfl_xor(top, 32, PL_WAVE));
        const float base2 = top == -INFINITY ? 0.f : top;
        const float alpha = __builtin_amdgcn_exp2f(m - base2);
        m = top;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            s[i] = __builtin_amdgcn_exp2f(s[i] - base2);
            sum += s[i];
        }
        l = l * alpha + sum;
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[t][i] *= alpha;
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            a8_frag pf[PIECES];
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = s[8 * g + e];
            a8_split<PIECES>(x, pf);
            const int key = 16 * g + 4 * half + (lane % 16) / 4;
#pragma unroll
            for (int t = 0; t < DT; ++t) {
                const int column = 32 * t + 16 * ((lane / 16) % 2) + 4 * (lane % 4);
                a8_frag vf;
                vf.half[0] = a8_read_transposed(mine + key * VROW + column);
                vf.half[1] = a8_read_transposed(mine + (key + 8) * VROW + column);
#pragma unroll
                for (int p = PIECES - 1; p >= 0; --p) acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf.vec, pf[p].vec, acc[t], 0, 0, 0);
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
    l += __shfl_xor(l, 32, PL_WAVE);

    // The waves meet: maximum and sum first, then the outputs in halves, always in the same order.
    if (half == 0) {
        stats[(2 * wave) * A8_ROWS + col] = m;
        stats[(2 * wave + 1) * A8_ROWS + col] = l;
    }
    __syncthreads();
    float top = -INFINITY, total = 0.f;
#pragma unroll
    for (int w = 0; w < A8_WAVES; ++w) top = fmaxf(top, stats[2 * w * A8_ROWS + col]);
    const float base2 = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int w = 0; w < A8_WAVES; ++w) total += stats[(2 * w + 1) * A8_ROWS + col] * __builtin_amdgcn_exp2f(stats[2 * w * A8_ROWS + col] - base2);
    const float mine2 = __builtin_amdgcn_exp2f(m - base2);
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[t][i] *= mine2;
    float* meet = reinterpret_cast<float*>(lds);
#pragma unroll
    for (int step = A8_WAVES / 2; step > 0; step /= 2) {
        if (wave >= step && wave < 2 * step && live)
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<a8_f32x4*>(meet + ((wave - step) * A8_ROWS + col) * (DP + 4) + 32 * t + 8 * i + 4 * half) =
                        a8_f32x4{acc[t][4 * i], acc[t][4 * i + 1], acc[t][4 * i + 2], acc[t][4 * i + 3]};
        __syncthreads();
        if (wave < step && live)
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const a8_f32x4 other = *reinterpret_cast<const a8_f32x4*>(meet + (wave * A8_ROWS + col) * (DP + 4) + 32 * t + 8 * i + 4 * half);
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[t][4 * i + e] += other[e];
                }
        __syncthreads();
    }
    if (wave != 0 || !live) return;

    const size_t out_row = static_cast<size_t>(a.q_start[seq] + token) * a.nq + head;
    if (a.chunks == 1) {
        if (shares > 1) total = NAN;          // (a context longer than the caller said)
        const float inv = total != 0.f ? 1.f / total : 0.f;
        T* to = static_cast<T*>(a.out) + out_row * a.d;
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int at = 32 * t + 8 * i + 4 * half;
                if (at < a.d) {
                    if constexpr (PIECES == 1) {
                        *reinterpret_cast<a8_u32x2*>(to + at) =
                            a8_u32x2{a8_pack2(acc[t][4 * i] * inv, acc[t][4 * i + 1] * inv), a8_pack2(acc[t][4 * i + 2] * inv, acc[t][4 * i + 3] * inv)};
                    } else {
                        *reinterpret_cast<a8_f32x4*>(to + at) = a8_f32x4{acc[t][4 * i] * inv, acc[t][4 * i + 1] * inv, acc[t][4 * i + 2] * inv, acc[t][4 * i + 3] * inv};
                    }
                }
            }
        return;
    }
    const size_t place = out_row * a.chunks + share;
    if (half == 0) {
        a.part_ml[2 * place] = top;
        a.part_ml[2 * place + 1] = total;
    }
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = 32 * t + 8 * i + 4 * half;
            if (at < a.d) *reinterpret_cast<a8_f32x4*>(a.part_acc + place * a.d + at) = a8_f32x4{acc[t][4 * i], acc[t][4 * i + 1], acc[t][4 * i + 2], acc[t][4 * i + 3]};
        }
}

// ---- shares put together ---------------------------------------------------------------------------------------------------
// A wave a row and query head: the shares that its block of rows had, in their order.
template <typename T>
__global__ __launch_bounds__(A8_WAVES * PL_WAVE) void attention_8bit_merge_kernel(A8Args a) {
    const int lane = threadIdx.x % PL_WAVE;
    const int group = a.nq / a.nkv;
    const int kvh = blockIdx.x % a.nkv;
    int seq, rb;
    if (!a8_find(a, blockIdx.x / a.nkv, group, A8_ROWS, seq, rb)) return;
    const int q_len = a.q_len[seq], start = a.ctx_len[seq] - q_len;
    const int first_row = rb * A8_ROWS, rows = min(A8_ROWS, q_len * group - first_row);
    const int lo = pl_first_visible(start + first_row / group, a.window), hi = start + (first_row + rows - 1) / group + 1;
    const int all = a8_shares(lo, hi, a.chunk), shares = min(all, a.chunks);
    for (int r = threadIdx.x / PL_WAVE; r < rows; r += A8_WAVES) {
        const int row = first_row + r;
        const size_t out_row = static_cast<size_t>(a.q_start[seq] + row / group) * a.nq + kvh * group + row % group;
        const float* ml = a.part_ml + 2 * out_row * a.chunks;
        const float* acc = a.part_acc + out_row * a.chunks * a.d;
        float top = -INFINITY;
        for (int s = lane; s < shares; s += PL_WAVE) top = fmaxf(top, ml[2 * s]);
        top = wave_max(top);
        const float base2 = top == -INFINITY ? 0.f : top;
        float total = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
        for (int s = 0; s < shares; ++s) {
            const float w = __builtin_amdgcn_exp2f(ml[2 * s] - base2);
            total += w * ml[2 * s + 1];
            if (4 * lane < a.d) {
                const a8_f32x4 y = *reinterpret_cast<const a8_f32x4*>(acc + static_cast<size_t>(s) * a.d + 4 * lane);
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] += w * y[e];
            }
        }
        if (all > shares) total = NAN;        // (a context longer than the caller said)
        const float inv = total != 0.f ? 1.f / total : 0.f;
        if (4 * lane < a.d) {
            struct __attribute__((aligned(4 * sizeof(T)))) Piece {
                T v[4];
            } to;
#pragma unroll
            for (int e = 0; e < 4; ++e) to.v[e] = from_float<T>(x[e] * inv);
            *reinterpret_cast<Piece*>(static_cast<T*>(a.out) + out_row * a.d + 4 * lane) = to;
        }
    }
}

template <int PIECES, int DT>
static int launch_attention(const A8Args& a, long blocks, hipStream_t stream) {
    constexpr int DP = 32 * DT, VROW = DP + a8_pad(DT);
    constexpr int MEET = 2 * A8_ROWS * (DP + 4) * 4, VALUES = A8_WAVES * A8_KEYS * VROW * 2;
    const size_t lds = (MEET > VALUES ? MEET : VALUES) + static_cast<size_t>(a.chunk) * 12 + A8_WAVES * 2 * A8_ROWS * 4;
    const dim3 grid(static_cast<unsigned>(blocks * a.nkv), static_cast<unsigned>(a.chunks));
    if (lds > 48 * 1024) {
        hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&attention_8bit_kernel<PIECES, DT>), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds));
        PL_REQUIRE(e == hipSuccess, "8-bit attention: %zu bytes of LDS refused: %s", lds, hipGetErrorString(e));
    }
    attention_8bit_kernel<PIECES, DT><<<grid, A8_WAVES * PL_WAVE, lds, stream>>>(a);
    PL_CHECK_LAUNCH("attention_8bit");
    if (a.chunks > 1) {
        attention_8bit_merge_kernel<typename A8Type<PIECES>::type><<<static_cast<unsigned>(blocks * a.nkv), A8_WAVES * PL_WAVE, 0, stream>>>(a);
        PL_CHECK_LAUNCH("attention_8bit_merge");
    }
    return 0;
}

template <int PIECES>
static int launch_attention(const A8Args& a, long blocks, hipStream_t stream) {
    switch (pl_ceil_div(a.d, 32)) {
        case 1: return launch_attention<PIECES, 1>(a, blocks, stream);
        case 2: return launch_attention<PIECES, 2>(a, blocks, stream);
        case 3: return launch_attention<PIECES, 3>(a, blocks, stream);
        case 4: return launch_attention<PIECES, 4>(a, blocks, stream);
        case 5:
        case 6: return launch_attention<PIECES, 6>(a, blocks, stream);
        default: return launch_attention<PIECES, 8>(a, blocks, stream);
    }
}

extern "C" int pl_paged_attention_8bit(const void* q, int q_stride, void* out, const void* q_start, const void* q_len, const void* ctx_len, int S, int n, int max_q_len,
                                       const void* table, int width, int block, int pool_rows, const void* k_pool, const void* v_pool, const void* k_scale,
                                       const void* v_scale, int nq, int nkv, int d, float scale, int window, int chunk, int chunks, void* part_acc, void* part_ml, int dtype,
                                       void* stream) {
    PL_REQUIRE(d >= 16 && d <= 256 && d % 16 == 0, "8-bit attention: head size %d, the kernel takes multiples of 16 up to 256", d);
    PL_REQUIRE(nkv >= 1 && nq >= nkv && nq % nkv == 0, "8-bit attention: %d query heads over %d key heads", nq, nkv);
    PL_REQUIRE(S >= 1 && n >= 1 && max_q_len >= 1 && width >= 1 && block >= 1 && pool_rows >= block, "8-bit attention: %d requests, %d rows, %d of one request, tables of %d pages of %d, %d rows",
               S, n, max_q_len, width, block, pool_rows);
    PL_REQUIRE(chunk >= A8_KEYS && chunk % A8_KEYS == 0 && chunk <= 2048 && chunks >= 1 && chunks < 65536 && (chunks == 1 || (part_acc && part_ml)), "8-bit attention: %d shares of %d keys", chunks, chunk);
    const A8Args a{q, q_stride, out, static_cast<const int*>(q_start), static_cast<const int*>(q_len), static_cast<const int*>(ctx_len), S, static_cast<const int*>(table), width, block, pool_rows,
                   static_cast<const uint8_t*>(k_pool), static_cast<const uint8_t*>(v_pool), static_cast<const uint8_t*>(k_scale), static_cast<const uint8_t*>(v_scale),
                   nq, nkv, d, scale * 1.4426950408889634f, window, n, chunk, chunks, static_cast<float*>(part_acc), static_cast<float*>(part_ml)};
    const int group = nq / nkv;
    // blocks of rows: one a request for what is left over, and the whole ones
    const long most = static_cast<long>(S) * pl_ceil_div(max_q_len * group, A8_ROWS);
    const long all = S + static_cast<long>(n) * group / A8_ROWS;
    const long blocks = most < all ? most : all;
    PL_REQUIRE(blocks * nkv < (1l << 31), "8-bit attention: %ld blocks of rows are too many for a launch", blocks);
    return dtype == PL_DTYPE_F32 ? launch_attention<3>(a, blocks, static_cast<hipStream_t>(stream)) : launch_attention<1>(a, blocks, static_cast<hipStream_t>(stream));
}
