// A paged cache held in 8 bits: where a step's tokens go, and how they get there.
//
// A page keeps, for each key head, `block` rows of d values of type e4m3 and one power of two E for the keys and one for the values: the row stands for
// 2^E times what its bytes say.  E is the least power whose 448-fold (the largest e4m3) holds the largest finite value of the head's rows in the page, so it can grow
// while the page fills; what the page holds then is expressed in the new unit and rounded again (a value that has been through n growths of one is off by at most half a
// step of the last unit plus half a step of every finer one before, less than a whole step).  It never shrinks before the page is begun anew.
// A power of two and not any scale: e4m3 times a power of two is exact in bfloat16 and in 32 bits, so reading rounds nothing.
#include "common.hpp"
#include "head_rows.hpp"

#define P8_LARGEST_SEQS 8192      // two words of LDS a request: 64 KB
#define P8_TABLE_THREADS 256
#define P8_HEADS 4                // query heads a group of lanes
#define P8_WAVES 4
#define P8_SINGLE_UNITS 16384     // up to so many rows times heads of keys and values every row is looked at by a wave of its own

// ---- block tables and slots ---------------------------------------------------------------------------------------------
// Request s brings q_len[s] tokens, its context behind the step is ctx_len[s]; it holds ceil((ctx - q) / block) pages and needs ceil(ctx / block).  Where new pages
// begin in the list of free ones, and where rows begin, are sums over the requests before.  Every workgroup works these sums out for itself in LDS: a few hundred words read from L2 take less
// than a second launch, and then it serves its share of rows and of table entries with no word to the other workgroups.  Bound by the launch: 512 requests of one token are 30 KB.
struct P8Request {
    int q_end, held, need, new_end;
};

__global__ __launch_bounds__(P8_TABLE_THREADS) void step_tables_kernel(const int* __restrict__ q_len, const int* __restrict__ ctx_len, int S, int* table, int width,
                                                                       int block, const int* __restrict__ free_pages, int num_free, int rows, int* __restrict__ q_start,
                                                                       int* __restrict__ positions, int* __restrict__ seq_of, int* __restrict__ slots,
                                                                       int* __restrict__ pages) {
    extern __shared__ int lds[];
    int* q_end = lds;                // rows up to and with request s
    int* new_end = lds + S;          // new pages up to and with request s
    __shared__ int wave_rows[P8_TABLE_THREADS / PL_WAVE], wave_pages[P8_TABLE_THREADS / PL_WAVE];
    const int tid = threadIdx.x, lane = tid % PL_WAVE, wave = tid / PL_WAVE;

    // A request whose context is shorter than what it brings holds the rows of a padded step: no position, no page.
    auto request = [&](int s, int& held, int& need) {
        const int q = max(q_len[s], 0), c = ctx_len[s];
        held = need = 0;
        if (c >= q && c > 0) {
            held = min((c - q) / block + ((c - q) % block != 0), width);
            need = min(c / block + (c % block != 0), width);
        }
        return q;
    };

    int rows_before = 0, pages_before = 0;
    for (int base = 0; base < S; base += P8_TABLE_THREADS) {
        const int s = base + tid;
        int q = 0, held = 0, need = 0;
        if (s < S) q = request(s, held, need);
        int sum_q = q, sum_new = free_pages != nullptr ? need - held : 0;
#pragma unroll
        for (int off = 1; off < PL_WAVE; off <<= 1) {
            const int a = __shfl_up(sum_q, off, PL_WAVE), b = __shfl_up(sum_new, off, PL_WAVE);
            if (lane >= off) {
                sum_q += a;
                sum_new += b;
            }
        }
        if (lane == PL_WAVE - 1) {
            wave_rows[wave] = sum_q;
            wave_pages[wave] = sum_new;
        }
        __syncthreads();
        int all_rows = 0, all_pages = 0;
        for (int w = 0; w < P8_TABLE_THREADS / PL_WAVE; ++w) {
            if (w == wave) {
                sum_q += all_rows + rows_before;
                sum_new += all_pages + pages_before;
            }
            all_rows += wave_rows[w];
            all_pages += wave_pages[w];
        }
        if (s < S) {
            q_end[s] = sum_q;
            new_end[s] = sum_new;
            if (blockIdx.x == 0) q_start[s] = sum_q - q;
        }
        rows_before += all_rows;
        pages_before += all_pages;
        __syncthreads();
    }
    if (blockIdx.x == 0 && tid == 0) *pages = pages_before;

    // The page of request s that is its `index`-th: from the table where it is held, else from the free ones.
    auto page_of = [&](int s, int index, int held, int need) {
        if (index >= width) return -1;
        if (free_pages == nullptr || index < held) return table[static_cast<size_t>(s) * width + index];
        const int at = new_end[s] - (need - held) + index - held;
        return index < need && at < num_free ? free_pages[at] : -1;
    };

    const int all = gridDim.x * P8_TABLE_THREADS, me = blockIdx.x * P8_TABLE_THREADS + tid;
    for (int r = me; r < rows; r += all) {
        int lo = 0, hi = S;          // the first request whose rows end behind r
        while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (q_end[mid] > r) hi = mid;
            else lo = mid + 1;
        }
        int position = -1, slot = -1;
        if (lo < S) {
            int held, need;
            const int q = request(lo, held, need), c = ctx_len[lo];
            if (c >= q) {
                position = r - (q_end[lo] - q) + c - q;
                const int page = page_of(lo, position / block, held, need);
                if (page >= 0) slot = page * block + position % block;
            }
        }
        positions[r] = position;
        seq_of[r] = min(lo, S - 1);
        slots[r] = slot;
    }
    // Entries below `held` are read above by any workgroup and written by none.
    if (free_pages != nullptr) {
        for (int s = blockIdx.x; s < S; s += gridDim.x) {
            int held, need;
            request(s, held, need);
            for (int i = held + tid; i < width; i += P8_TABLE_THREADS) table[static_cast<size_t>(s) * width + i] = i < need ? page_of(s, i, held, need) : -1;
        }
    }
}

extern "C" int pl_step_tables(const void* q_len, const void* ctx_len, int S, void* table, int width, int block, const void* free_pages, int num_free, int rows,
                              void* q_start, void* positions, void* seq_of, void* slots, void* pages, void* stream) {
    PL_REQUIRE(S >= 1 && S <= P8_LARGEST_SEQS, "step tables: %d requests, the kernel takes 1 to %d", S, P8_LARGEST_SEQS);
    PL_REQUIRE(width >= 1 && block >= 1 && rows >= 0 && num_free >= 0, "step tables: width %d, pages of %d tokens, %d rows, %d free pages", width, block, rows, num_free);
    // a few rows or one request's entries a thread, up to a workgroup a compute unit
    const int work = max(pl_ceil_div(rows, P8_TABLE_THREADS), free_pages != nullptr ? S : 1);
    step_tables_kernel<<<max(1, min(work, pl_compute_units())), P8_TABLE_THREADS, 2 * S * sizeof(int), static_cast<hipStream_t>(stream)>>>(
        static_cast<const int*>(q_len), static_cast<const int*>(ctx_len), S, static_cast<int*>(table), width, block, static_cast<const int*>(free_pages), num_free, rows,
        static_cast<int*>(q_start), static_cast<int*>(positions), static_cast<int*>(seq_of), static_cast<int*>(slots), static_cast<int*>(pages));
    PL_CHECK_LAUNCH("step_tables");
    return 0;
}

// ---- the write ------------------------------------------------------------------------------------------------------------
// Rows of heads are taken eight values a lane, d / 8 lanes a row.  A run is what the step brings to one page: rows that follow each other with slots that follow
// each other.  One wave or workgroup takes a run of one key head, keys or values: the largest of its rows gives the page's new power, then the rows are
// rounded into the page.  Runs of more rows than it takes at a time are read (and normed, turned) twice, the second time from L2.  Queries are normed and turned by workgroups of their own in the
// same launch.  Prompts are bound by what they read and write (10,503 rows of 32 + 8 heads of 128: 237 MB in 70 us where inputs change from call to call, 3.4 TB/s; 60 us on the same ones), single tokens by the waits for slots, rows and powers one behind the other (64 of 16 + 8 heads: 5.4 us),
// and steps in between by a wave's chain of these for every run, all its rows a few at a time and twice (788 rows in 32 bits into 4 heads of 64: 9.1 us, their bytes 1.5).
struct P8Write {
    const void* qkv;
    void* q;
    int q_stride;                 // values between two rows of q
    const void *q_gain, *k_gain;
    int gain_dtype;
    float eps;
    const float *cos, *sin;
    int rot, angles;              // rotated values of a head; rows of the tables
    bool neighbours;
    const int *positions, *slots;
    int block, pool_rows;
    uint8_t *k_pool, *v_pool, *k_scale, *v_scale;
    int n, nq, nkv, d;
};

template <typename T>
__device__ __forceinline__ void p8_load8(const T* from, float (&to)[8]) {
    struct __attribute__((aligned(16))) Piece {
        T v[8];
    };
    const Piece p = *reinterpret_cast<const Piece*>(from);
#pragma unroll
    for (int e = 0; e < 8; ++e) to[e] = to_float(p.v[e]);
}
__device__ __forceinline__ void p8_gain8(const P8Write& a, bool key, int at, float (&to)[8]) {
    const void* gain = key ? a.k_gain : a.q_gain;
    if (a.gain_dtype == PL_DTYPE_F32) p8_load8(static_cast<const float*>(gain) + at, to);
    else p8_load8(static_cast<const bf16_t*>(gain) + at, to);
}

// Eight values (`chunk` of the row) of head `head` of row `row`, normed and turned where they are a query's or a key's.  All LPR lanes of a row call this together.  Everything that is read
// is asked for before the first sum, so a row costs one wait.
// PIECES: the rotation turns halves of whole pieces, so a piece's partners are another lane's piece and its angles a piece of the tables (or nothing is turned); any other rotation looks its
// partners up one by one, which takes two and a half times the registers and so has a kernel of its own.
// What a lane needs of a row beside its values: the same for all heads of queries, or of keys, of the row.
template <int LPR, bool PIECES>
struct P8Turn {
    float g[8], c[8], s[8];
    size_t angle;
    bool here, key, plain, turned, low;

    __device__ __forceinline__ P8Turn(const P8Write& a, int row, int head, int chunk, bool live) {
        const int half = a.rot / 2, first = chunk * 8;
        here = live && first < a.d;
        key = head >= a.nq;
        plain = head >= a.nq + a.nkv;
        turned = !plain && first < a.rot;
        low = first < half;
        angle = static_cast<size_t>(a.rot > 0 && !plain ? min(max(a.positions[row], 0), a.angles - 1) : 0) * half;
        if (!plain && here && a.q_gain != nullptr) p8_gain8(a, key, first, g);
        if (PIECES && turned && here) {
            p8_load8(a.cos + angle + (low ? first : first - half), c);
            p8_load8(a.sin + angle + (low ? first : first - half), s);
        }
    }

    // Eight values of the row that begins at `base`, normed and turned.  All LPR lanes of a row call this together.
    template <typename T>
    __device__ __forceinline__ void apply(const P8Write& a, const T* base, int chunk, float (&x)[8]) const {
        if (plain) return;
        const int half = a.rot / 2, first = chunk * 8;
        float rinv = 1.f;
        if (a.q_gain != nullptr) {
            float ss = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
            if constexpr (LPR == 16) {
                ss = hr_sum16(ss);
            } else {
#pragma unroll
                for (int off = LPR / 2; off > 0; off >>= 1) ss += __shfl_xor(ss, off, PL_WAVE);
            }
            rinv = 1.f / sqrtf(ss / static_cast<float>(a.d) + a.eps);
            if (here)
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = x[e] * rinv * g[e];
        }
        if (a.rot == 0) return;
        if constexpr (PIECES) {
            // (A head of 128 turned whole, the usual one: the partner is eight lanes on in the row of 16, which moves through the vector pipe and not through LDS.)
            if (LPR == 16 && half == 64) {
                if (!plain)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float p = hr_dpp<0x128>(x[e]);
                        x[e] = low ? x[e] * c[e] - p * s[e] : x[e] * c[e] + p * s[e];
                    }
                return;
            }
            const int lane = threadIdx.x % PL_WAVE, other = low ? lane + half / 8 : lane - half / 8;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float p = __shfl(x[e], other, PL_WAVE);
                if (turned && here) x[e] = low ? x[e] * c[e] - p * s[e] : x[e] * c[e] + p * s[e];
            }
        } else {
            if (!here || !turned) return;
            float old[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) old[e] = x[e];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int i = first + e;
                if (i >= a.rot) continue;
                if (a.neighbours) {
                    const float ci = a.cos[angle + i / 2], si = a.sin[angle + i / 2];
                    x[e] = e % 2 == 0 ? old[e] * ci - old[e ^ 1] * si : old[e] * ci + old[e ^ 1] * si;
                } else {
                    const bool lower = i < half;
                    const int at = lower ? i : i - half, other = lower ? i + half : i - half;
                    float p = to_float(base[other]);
                    if (a.q_gain != nullptr) p = p * rinv * load_as_float(key ? a.k_gain : a.q_gain, a.gain_dtype, other);
                    x[e] = lower ? old[e] * a.cos[angle + at] - p * a.sin[angle + at] : old[e] * a.cos[angle + at] + p * a.sin[angle + at];
                }
            }
        }
    }
};

template <typename T>
__device__ __forceinline__ const T* p8_row(const P8Write& a, int row, int head) {
    return static_cast<const T*>(a.qkv) + (static_cast<size_t>(row) * (a.nq + 2 * a.nkv) + head) * a.d;
}

// Eight values (`chunk` of the row) of head `head` of row `row`, normed and turned where they are a query's or a key's.
template <typename T, int LPR, bool PIECES>
__device__ __forceinline__ void p8_prepare(const P8Write& a, int row, int head, int chunk, float (&x)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = 0.f;
    const T* base = p8_row<T>(a, row, head);
    if (chunk * 8 < a.d) p8_load8(base + chunk * 8, x);
    const P8Turn<LPR, PIECES> turn(a, row, head, chunk, true);
    turn.apply(a, base, chunk, x);
}

__device__ __forceinline__ bool p8_finite(float v) { return (__float_as_uint(v) & 0x7f800000u) != 0x7f800000u; }

// The byte (exponent plus 127, one at least) of the least power of two whose 448-fold holds `top`, which is finite and not negative: with top = m 2^e, 1 <= m < 2, and 448 = 1.75 2^8.
__device__ __forceinline__ int p8_power(float top) {
    const uint32_t bits = __float_as_uint(top);
    return max(static_cast<int>(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0), 1);
}

// Eight values as e4m3, rounded to nearest, ties to even; what is not finite becomes NaN.
__device__ __forceinline__ uint2 p8_round8(const float (&x)[8], int power) {
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = p8_finite(x[e]) ? ldexpf(x[e], 127 - power) : __uint_as_float(0x7fc00000u);
    int lo = 0, hi = 0;
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], lo, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], lo, true);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[4], y[5], hi, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[6], y[7], hi, true);
    return make_uint2(static_cast<uint32_t>(lo), static_cast<uint32_t>(hi));
}

__device__ __forceinline__ void p8_values8(uint2 bytes, float (&x)[8]) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const int w[2] = {static_cast<int>(bytes.x), static_cast<int>(bytes.y)};
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(w[e], false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w[e], true);
        x[4 * e] = a[0];
        x[4 * e + 1] = a[1];
        x[4 * e + 2] = b[0];
        x[4 * e + 3] = b[1];
    }
}

template <typename T, int LPR, int WAVES, bool PIECES>
__device__ __forceinline__ void p8_run(const P8Write& a, int first, int slot, int head, bool keys, float* scratch) {
    constexpr int ROWS = WAVES * PL_WAVE / LPR;         // rows at a time
    const int tid = WAVES == 1 ? threadIdx.x % PL_WAVE : threadIdx.x;
    const int lane_row = tid / LPR, chunk = tid % LPR;
    const int page = slot / a.block, off = slot % a.block;
    const int source = keys ? a.nq + head : a.nq + a.nkv + head;
    uint8_t* pool = keys ? a.k_pool : a.v_pool;
    uint8_t* scale = (keys ? a.k_scale : a.v_scale) + static_cast<size_t>(page) * a.nkv + head;
    const size_t row_bytes = static_cast<size_t>(a.nkv) * a.d;
    uint8_t* rows = pool + static_cast<size_t>(page) * a.block * row_bytes + static_cast<size_t>(head) * a.d;
    // The first rows are read before it is known how many are the run's: that costs a wait of its own.
    const int most = min(a.block - off, a.n - first);
    const int before = off > 0 ? *scale : 0;
    float x[8], top = 0.f;
    p8_prepare<T, LPR, PIECES>(a, first + min(lane_row, most - 1), source, chunk, x);
    int count = most;
    for (int base = 0; base < most; base += PL_WAVE) {
        const int i = base + static_cast<int>(threadIdx.x % PL_WAVE);
        const uint64_t other = __ballot(i < most && a.slots[first + min(i, most - 1)] != slot + i);
        if (other != 0) {
            count = base + __ffsll(static_cast<unsigned long long>(other)) - 1;
            break;
        }
    }
    for (int r = 0; r < count; r += ROWS) {
        if (r > 0) p8_prepare<T, LPR, PIECES>(a, first + min(r + lane_row, count - 1), source, chunk, x);
        if (r + lane_row < count)
#pragma unroll
            for (int e = 0; e < 8; ++e) top = fmaxf(top, p8_finite(x[e]) ? fabsf(x[e]) : 0.f);
    }
    top = wave_max(top);
    if (WAVES > 1) {
        __syncthreads();
        if (threadIdx.x % PL_WAVE == 0) scratch[threadIdx.x / PL_WAVE] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WAVES; ++w) top = fmaxf(top, scratch[w]);
    }
    const int power = max(p8_power(top), before);
    // what the page holds of this request, in its new unit
    if (power > before && off > 0 && chunk * 8 < a.d) {
        for (int r = lane_row; r < off; r += ROWS) {
            uint2* at = reinterpret_cast<uint2*>(rows + r * row_bytes + chunk * 8);
            float old[8];
            p8_values8(*at, old);
            *at = p8_round8(old, 127 + power - before);
        }
    }
    for (int r = 0; r < count; r += ROWS) {
        if (count > ROWS) p8_prepare<T, LPR, PIECES>(a, first + min(r + lane_row, count - 1), source, chunk, x);
        if (r + lane_row < count && chunk * 8 < a.d) *reinterpret_cast<uint2*>(rows + (off + r + lane_row) * row_bytes + chunk * 8) = p8_round8(x, power);
    }
    if (tid == 0) *scale = static_cast<uint8_t>(power);
}

// Workgroups of four waves: first nkv * 2 units of WAVES waves a tile of `tile` rows for keys and values, then those of the queries.
template <typename T, int LPR, int WAVES, bool PIECES>
__global__ __launch_bounds__(P8_WAVES * PL_WAVE) void write_8bit_kernel(P8Write a, int tile) {
    __shared__ float scratch[P8_WAVES];
    constexpr int ROWS = P8_WAVES * PL_WAVE / LPR, UNITS = P8_WAVES / WAVES;
    const int tiles = a.slots != nullptr ? pl_ceil_div(a.n, tile) : 0, pairs = 2 * a.nkv;
    const long units = static_cast<long>(tiles) * pairs, of_pages = (units + UNITS - 1) / UNITS;
    if (blockIdx.x < of_pages) {
        const long unit = static_cast<long>(blockIdx.x) * UNITS + (WAVES == 1 ? threadIdx.x / PL_WAVE : 0);
        if (unit >= units) return;
        const int t = __builtin_amdgcn_readfirstlane(static_cast<int>(unit / pairs)), pair = __builtin_amdgcn_readfirstlane(static_cast<int>(unit % pairs));
        // the first rows of runs, found by every wave for itself
        const int r = t * tile + static_cast<int>(threadIdx.x % PL_WAVE);
        const bool mine = r < min((t + 1) * tile, a.n);
        const int slot = mine ? a.slots[r] : -1, before = mine && r > 0 ? a.slots[r - 1] : -2;
        uint64_t runs = __ballot(slot >= 0 && slot < a.pool_rows && (slot % a.block == 0 || before != slot - 1));
        for (; runs != 0; runs &= runs - 1) {
            const int which = __ffsll(static_cast<unsigned long long>(runs)) - 1;
            p8_run<T, LPR, WAVES, PIECES>(a, t * tile + which, __builtin_amdgcn_readfirstlane(__shfl(slot, which, PL_WAVE)), pair / 2, pair % 2 == 0, scratch);
        }
        return;
    }
    // The queries: P8_HEADS heads of a row a group of lanes, which share its angles and gains.
    const int i = static_cast<int>(blockIdx.x - of_pages) * ROWS + static_cast<int>(threadIdx.x / LPR);
    const int chunk = threadIdx.x % LPR, blocks = pl_ceil_div(a.nq, P8_HEADS);
    const bool live = i < a.n * blocks && chunk * 8 < a.d;
    const int row = i < a.n * blocks ? i / blocks : 0, head = i < a.n * blocks ? i % blocks * P8_HEADS : 0;
    float x[P8_HEADS][8];
#pragma unroll
    for (int h = 0; h < P8_HEADS; ++h) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[h][e] = 0.f;
        if (live && head + h < a.nq) p8_load8(p8_row<T>(a, row, head + h) + chunk * 8, x[h]);
    }
    const P8Turn<LPR, PIECES> turn(a, row, head, chunk, live);
    const bool written = live && a.positions[row] >= 0;
    struct __attribute__((aligned(16))) Piece {
        T v[8];
    } out;
#pragma unroll
    for (int h = 0; h < P8_HEADS; ++h) {
        turn.apply(a, p8_row<T>(a, row, head + min(h, a.nq - 1 - head)), chunk, x[h]);
        if (!written || head + h >= a.nq) continue;
#pragma unroll
        for (int e = 0; e < 8; ++e) out.v[e] = from_float<T>(x[h][e]);
        *reinterpret_cast<Piece*>(static_cast<T*>(a.q) + static_cast<size_t>(row) * a.q_stride + static_cast<size_t>(head + h) * a.d + chunk * 8) = out;
    }
}

// Lanes a row of d values, eight each.
static int p8_lanes(int d) { return d <= 32 ? 4 : d <= 64 ? 8 : d <= 128 ? 16 : 32; }

// How a step is written: the rows that a wave looks through for the first ones of runs, and the waves that take a run.
struct P8Shape {
    int tile, waves;
};
static P8Shape p8_shape(int n, int nkv, int block, int d) {
    // A wave takes a run, 64 / LPR rows at a time; in steps of many rows a workgroup does, four times as many.  It looks through `tile` rows for the first ones of runs: one each while all of a
    // step's may be first (decoding), else 32, since most of many rows are inside a page, and units that find nothing still cost their start: 10,503 rows of prompts into 8 heads took 182 us with a
    // workgroup a row and 77 with 32 rows when this was chosen (70 now), 600 single tokens 30 us with a workgroup each and 14 with a wave.  (Values of more rows held in registers, so that a run is not read again from L2 once its
    // power is known, cost the queries' workgroups of the same launch their places: 94 us with twice the rows, 117 with four times.)
    const int tile = static_cast<long>(n) * 2 * nkv <= P8_SINGLE_UNITS ? 1 : 32;
    return P8Shape{tile, tile > 1 && block > PL_WAVE / p8_lanes(d) ? P8_WAVES : 1};
}
extern "C" int pl_qk_norm_rope_kv_write_8bit_tile(int n, int nkv, int block, int d) { return p8_shape(n, nkv, block, d).tile; }
extern "C" int pl_qk_norm_rope_kv_write_8bit_waves(int n, int nkv, int block, int d) { return p8_shape(n, nkv, block, d).waves; }

template <typename T, int LPR>
static int launch_write(const P8Write& a, hipStream_t stream) {
    constexpr int ROWS = P8_WAVES * PL_WAVE / LPR;
    const P8Shape shape = p8_shape(a.n, a.nkv, a.block, a.d);
    const int tile = shape.tile;
    const bool whole = shape.waves > 1;
    const long units = a.slots != nullptr ? static_cast<long>(pl_ceil_div(a.n, tile)) * 2 * a.nkv : 0;
    const long groups = (whole ? units : (units + P8_WAVES - 1) / P8_WAVES) + (static_cast<long>(a.n) * pl_ceil_div(a.nq, P8_HEADS) + ROWS - 1) / ROWS;
    PL_REQUIRE(groups < (1l << 31) && static_cast<long>(a.n) * a.nq < (1l << 31) - ROWS, "8-bit write: %d rows of %d heads are too many for a launch", a.n, a.nq + 2 * a.nkv);
    const bool pieces = a.rot == 0 || (a.rot % 16 == 0 && !a.neighbours && (reinterpret_cast<uintptr_t>(a.cos) | reinterpret_cast<uintptr_t>(a.sin)) % 16 == 0);
    const auto kernel = whole ? (pieces ? write_8bit_kernel<T, LPR, P8_WAVES, true> : write_8bit_kernel<T, LPR, P8_WAVES, false>)
                              : (pieces ? write_8bit_kernel<T, LPR, 1, true> : write_8bit_kernel<T, LPR, 1, false>);
    kernel<<<static_cast<unsigned>(groups), P8_WAVES * PL_WAVE, 0, stream>>>(a, tile);
    PL_CHECK_LAUNCH("write_8bit");
    return 0;
}

template <typename T>
static int launch_write(const P8Write& a, hipStream_t stream) {
    switch (p8_lanes(a.d)) {
        case 4: return launch_write<T, 4>(a, stream);
        case 8: return launch_write<T, 8>(a, stream);
        case 16: return launch_write<T, 16>(a, stream);
        default: return launch_write<T, 32>(a, stream);
    }
}

extern "C" int pl_qk_norm_rope_kv_write_8bit(const void* qkv, void* q, int q_stride, const void* q_gain, const void* k_gain, int gain_dtype, float eps, const void* cos,
                                             const void* sin, int rot, int angles, int neighbours, const void* positions, const void* slots, int block, int pool_rows,
                                             void* k_pool, void* v_pool, void* k_scale, void* v_scale, int n, int nq, int nkv, int d, int dtype, void* stream) {
    PL_REQUIRE(d >= 16 && d <= 256 && d % 16 == 0, "8-bit write: head size %d, the kernel takes multiples of 16 up to 256", d);
    PL_REQUIRE(rot >= 0 && rot <= d && rot % 2 == 0 && (rot == 0 || angles >= 1), "8-bit write: a rotation over %d values of a head of %d, %d angles", rot, d, angles);
    PL_REQUIRE(n >= 0 && nq >= 0 && nkv >= 1 && block >= 1 && pool_rows >= block, "8-bit write: %d rows, %d and %d heads, pages of %d, %d rows of pages", n, nq, nkv, block, pool_rows);
    if (n == 0 || (slots == nullptr && nq == 0)) return 0;
    const P8Write a{qkv, q, q_stride, q_gain, k_gain, gain_dtype, eps, static_cast<const float*>(cos), static_cast<const float*>(sin), rot, angles, neighbours != 0,
                    static_cast<const int*>(positions), static_cast<const int*>(slots), block, pool_rows, static_cast<uint8_t*>(k_pool), static_cast<uint8_t*>(v_pool),
                    static_cast<uint8_t*>(k_scale), static_cast<uint8_t*>(v_scale), n, nq, nkv, d};
    return dtype == PL_DTYPE_F32 ? launch_write<float>(a, static_cast<hipStream_t>(stream)) : launch_write<bf16_t>(a, static_cast<hipStream_t>(stream));
}
