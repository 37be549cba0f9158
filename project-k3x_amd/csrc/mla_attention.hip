// mla_attention.hip -- attention over the cached latents, the up-projections
// absorbed into queries and outputs.
//
// All heads of a token read the same row of L + R values as the key and its
// first L as the value, so the rows (token, head) of a sequence are one operand:
// S^T = K Q^T and O^T = K[:, :L]^T P^T on the matrix cores, 32 cached tokens at a
// time, with the running maximum and sum of a softmax.  Both products take the
// tile of K from LDS, where it lies once for all rows of a workgroup.  S^T is
// computed with tokens as its rows because its result then already is, lane for
// lane, the operand P^T of the second product (a lane holds four neighbouring
// tokens of one row; the tokens of that product's depth are taken in the order
// that this leaves), and a row's maximum and sum lie in one lane of each half.
//
// The cached tokens of all sequences, in tiles of 32, are one line that is cut
// into equal ranges for the workgroups: a sequence that falls into several
// ranges is joined by a second launch.
//
// Bound: with many rows the reads of LDS, which each wave makes for both products, beside
// the matrix cores (busy for 28 to 38% of the cycles) and the weights between them; with
// few rows memory.  At a latent of 512 and a rotary part of 64: 64 sequences of 208000
// tokens, 128 heads, 16 bits 106 us (90 and the join's 18, whose pieces are 82 MB written
// and read); 8 windows of 5 tokens on 32 heads over 77000 tokens in E4M3 71 us; 4 sequences
// of 417000 tokens, 64 heads, in E2M1 99 us, 581 TFLOP/s; 64 sequences of 8192 tokens, 32
// heads, 16 bits 127 us, 4.8 TB/s; one of 1000 tokens on 16 heads 14, in two launches.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "k3x_mla.hpp"
#include "k3x_mla_mma.hpp"

using namespace k3x_dev;
using namespace k3x_ops;
using namespace k3x_mla;

namespace {

constexpr uint32_t kThreads = 256;
// Cached tokens of a range at least.  One sequence of 500 tokens on 16 heads: 11.7 us, with
// 128 13.5; on 128 heads 18.9 and 21.5.
constexpr uint32_t kLeast = 64;

// A group of row blocks of a sequence that begins in range w and ends in another.
struct Split {
    uint32_t pieces;  // ranges that it lies in; 0: none to join
    uint32_t w, begin, count, group;
    int32_t before;   // positions before the first of its tokens
};

struct AttentionArgs {
    Pages pages;
    const void* q;
    const uint8_t* pool;
    void* out;
    float* lse;
    uint32_t H, L, R;
    uint64_t qs, os;
    float rate;  // scale * log2(e)
    uint32_t G, RB;  // ranges, row blocks of a group
    uint32_t one;    // no sequence has more than one group
    Split* splits;   // [N], or where there are more sequences or groups than ranges [G], by range
    float2* sums;    // [G][RB][2][rows]: reference (log2) and sum of a piece
    float4* parts;   // [G][RB][2][rows * LP / 4]: its outputs, as the lanes hold them
    uint32_t* status;
};

// How four waves share a tile of TILE cached tokens.  WM row blocks by WD parts of the
// latent; RT blocks of HT rows a wave.  Of 32 tokens each wave forms the scores of its own
// rows.  Of 64 (JOINT) it forms those of one block of rows and half of the tokens, and
// all waves take the weights from LDS: each part of a tile is read from there fewer times.
// 64 sequences of 8192 tokens, 64 heads in E2M1: 139 us with 32 tokens, 109 with 64; 32
// heads 132 and 98, in 16 bits 150 and 127.  (Of 128 rows a wave's outputs and queries fill
// the registers with its own 32; of 16 two workgroups share a compute unit, and its LDS.)
template <int HT_, int WM_, int WD_, int RT_, int TILE_>
struct Shape {
    static constexpr int HT = HT_, WM = WM_, WD = WD_, RT = RT_, TILE = TILE_;
    static constexpr int rows = HT * WM * RT;
    static constexpr bool JOINT = TILE == 64;
};

// Tiles of a sequence; an empty one takes one, in which its rows are written as empty.
template <uint32_t TILE>
__device__ inline uint32_t tiles_in(const Tokens& s) { return max(1u, (s.len + TILE - 1) / TILE); }
// Groups of row blocks that it has.
__device__ inline uint32_t groups_in(const AttentionArgs& a, const Tokens& s, uint32_t rows) {
    return a.one ? 1 : (s.count * a.H + a.RB * rows - 1) / (a.RB * rows);
}
// What it takes in the line, each group its tiles; kLong: more than is run.  Up to 2^36 rows
// times positions stay below it: (rows + 63) (positions + 31) / 2048, of fewer than 2^31 rows
// and at most 2^29 positions.  64 sequences below it are counted in 32 bits, and all together
// have to stay below 2^31, so that ranges and their ends do too.
constexpr uint32_t kLong = 1u << 26;
template <uint32_t TILE>
__device__ inline uint32_t tiles_of(const AttentionArgs& a, uint32_t n, uint32_t rows, Tokens* s) {
    if (!tokens_of(a.pages, n, s) || !s->count) return 0;
    return (uint32_t)min((uint64_t)kLong, (uint64_t)tiles_in<TILE>(*s) * groups_in(a, *s, rows));
}

// FULL: L is LP (else the columns past L are zeros, and not brought or written) and
// a page holds whole eights of tokens.
template <uint32_t DT, uint32_t F, int LP, typename S, int BUFS, bool FULL>
__global__ __launch_bounds__(kThreads, S::rows == 16 ? 2 : 1) void mla_attention_kernel(AttentionArgs a) {
    constexpr int HT = S::HT, WD = S::WD, RT = S::RT, CG = LP / 64 + 1;
    constexpr bool JOINT = S::JOINT;
    constexpr uint32_t kTile = S::TILE;
    constexpr int XB = kTile / 32;              // eights of tokens a wave brings
    constexpr uint32_t kGroup = kTile * 128;    // bytes of 64 columns of a tile in LDS
    constexpr uint32_t kBuffer = CG * kGroup;
    // Behind the buffers, where waves share them: weights, a row's largest scores, flags.
    constexpr uint32_t kWeights = BUFS * kBuffer, kTops = kWeights + RT * 4096,
                       kFlags = kTops + RT * 256;
    constexpr int KS = HT == 32 ? 4 : 2;        // products over 64 columns
    constexpr int OT = LP / HT / WD;            // tiles of the latent, a wave
    // Operands on their way; eight where the registers hold them.
    constexpr int AHEAD = F != K3X_CACHE_16BIT && S::rows == 128 ? 4 : 8;
    typedef Mma<DT, HT> M;
    typedef typename M::Acc Acc;
    // One array: with several the compiler tells them apart, and waits for all direct
    // loads to LDS before any read of theirs.
    __shared__ __attribute__((aligned(256))) uint8_t smem[JOINT ? kFlags + 16 : kWeights];
    uint32_t* const scan = reinterpret_cast<uint32_t*>(smem);  // before the first tile
    uint32_t* const at_s = scan + 4;
    uint32_t* const stop_s = scan + 12;
    lds_byte* const lds = (lds_byte*)smem;
    const uint32_t tid = threadIdx.x, lane = tid & 63;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t status = *(volatile uint32_t*)a.status;  // looked at with the lengths
    if (blockIdx.x == 0) check_sequences(a.pages, a.status);

    // ---- the line and this workgroup's range of it --------------------------
    // Tiles before and in sequences base .. base + 255, a sequence a thread.
    Tokens mine;
    auto scan_tiles = [&](uint32_t base, uint32_t* own) {
        const uint32_t n = base + tid;
        uint32_t c = *own = n < a.pages.N ? tiles_of<kTile>(a, n, S::rows, &mine) : 0;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t o = __shfl_up(c, d);
            if (lane >= (uint32_t)d) c += o;
        }
        __syncthreads();
        if (lane == 63) scan[wave] = c;
        __syncthreads();
        uint32_t before = 0;
        for (uint32_t i = 0; i < wave; ++i) before += scan[i];
        return before + c;  // with the thread's own
    };
    const bool by_sequence = a.one && a.pages.N <= a.G;
    uint64_t all = 0;
    bool over_long = false;
    uint32_t own, upto = 0;
    for (uint32_t base = 0; base < a.pages.N; base += kThreads) {
        upto = scan_tiles(base, &own);
        over_long |= own >= kLong;
        all += (uint64_t)scan[0] + scan[1] + scan[2] + scan[3];
        if (by_sequence && blockIdx.x == 0 && !own && base + tid < a.pages.N)
            a.splits[base + tid].pieces = 0;  // in no range
    }
    // All waves or none: another workgroup may latch between their looks.  (Not by the
    // barrier that counts, which has an array of LDS of its own.)
    over_long |= all >> 31 != 0;
    if (over_long) latch(a.status, K3X_ERR_INVALID_STATE);
    const bool stop = __any(status || over_long);
    if (lane == 0) stop_s[wave] = stop;
    __syncthreads();
    if (stop_s[0] | stop_s[1] | stop_s[2] | stop_s[3]) return;
    const uint32_t total = (uint32_t)all;
    // More than its share where the join of so many pieces takes longer: of a sequence of t
    // tiles, c a range, both cost least together at about c = sqrt(t / (kTile / 2)); of N
    // sequences the pieces are joined side by side, and c is less by another sqrt(N).  One
    // sequence on 16 heads, of 16000 tokens: 25.3 us with its share alone and 19.7 so, of
    // 131072 54.4 and 43.2; two of 32000 32.9 and 31.6, four of 16384 28.2 and 28.8.
    const uint32_t chunk = max(max(kLeast / kTile, (total + a.G - 1) / a.G),
                               (uint32_t)(__builtin_sqrtf((float)total / (kTile / 2)) / a.pages.N));
    const uint32_t ranges = (total + chunk - 1) / chunk;  // in use, G at most
    // Consecutive ranges, and a range's row blocks, lie on one die: they share cached
    // tokens and queries.
    uint32_t w = blockIdx.x / a.RB, rb = blockIdx.x % a.RB;
    if (!by_sequence && rb == 0 && tid == 0 && w >= ranges) a.splits[w].pieces = 0;
    if (a.G % 8 == 0) {
        const uint32_t each = (ranges + 7) / 8, x = blockIdx.x / 8;
        if (x / a.RB >= each) return;
        w = blockIdx.x % 8 * each + x / a.RB;
        rb = x % a.RB;
    }
    if (w >= ranges) return;
    if (!by_sequence && rb == 0 && tid == 0) a.splits[w].pieces = 0;
    const uint32_t from = w * chunk, to = min(total, from + chunk);
    // The sequence that tile `from` is in, and the tiles before it.
    uint32_t carry = 0;
    for (uint32_t base = 0; base < a.pages.N; base += kThreads) {
        if (a.pages.N > kThreads) upto = scan_tiles(base, &own);
        if (own && from >= carry + upto - own && from < carry + upto) {
            at_s[0] = base + tid;
            at_s[1] = carry + upto - own;
            at_s[2] = mine.begin;
            at_s[3] = mine.count;
            at_s[4] = mine.len;
        }
        carry += scan[0] + scan[1] + scan[2] + scan[3];
        if (carry > from) break;
    }
    __syncthreads();
    auto uniform = [](uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane(x); };
    uint32_t n = uniform(at_s[0]), first = uniform(at_s[1]), group = 0;
    Tokens s{uniform(at_s[2]), uniform(at_s[3]), uniform(at_s[4])};
    __syncthreads();
    if (!a.one) {
        group = (from - first) / tiles_in<kTile>(s);
        first += group * tiles_in<kTile>(s);
    }

    // What is not brought to LDS stays zero there.
    if (!FULL) {
        for (uint32_t i = tid * 16; i < BUFS * kBuffer; i += kThreads * 16)
            *reinterpret_cast<u32x4*>(smem + i) = u32x4{};
        __syncthreads();
    }

    const uint32_t wm = wave / WD, wd = wave % WD;
    const uint32_t col = lane % HT, g = lane / HT;
    // The block of rows and the 32 tokens of a tile that the wave forms scores of.
    const uint32_t srow = JOINT ? wave / 2 % RT : wm, side = JOINT ? wave % 2 : 0;
    // Where the lane reads its operands in a tile: keys, and values of a 16-lane
    // row's four tokens.  Other columns of a 64-column group are an exclusive or away.
    const uint32_t kat0 = col * 128 + (g ^ swizzle(col)) * 16;
    const uint32_t i16 = lane & 15, vrow = 4 * g + i16 / 4;
    const uint32_t vat0 = vrow * 128 +
                          (((HT == 32 ? 2 * (lane >> 4 & 1) : 0) + (i16 & 3) / 2) ^ swizzle(vrow)) * 16 +
                          (i16 & 1) * 8;
    // What the lane brings of each tile: one of eight columns of 16 bytes (codes: 16
    // bytes) of a token.  Direct loads fill LDS lane by lane, eight tokens a wave;
    // through registers eight lanes write every other one of sixteen tokens, which do not
    // meet in a bank.
    constexpr bool DIRECT = F == K3X_CACHE_16BIT && FULL;
    const uint32_t btok = DIRECT ? 8 * wave + lane / 8
                                 : 16 * (wave / 2) + lane % 8 * 2 + lane / 8 % 2;
    const uint32_t bcol = DIRECT ? lane % 8 : lane / 16 + 4 * (wave % 2);
    const uint32_t bput = bcol ^ swizzle(btok);

    bool bad_page = false, bad_value = false;
    while (true) {
        const uint32_t tiles = tiles_in<kTile>(s);
        const uint32_t rows = s.count * a.H;
        const uint32_t t0 = max(from, first) - first, t1 = min(to - first, tiles);
        const bool whole = t0 == 0 && t1 == tiles;
        if (rb == 0 && tid == 0 && t0 == 0 && (by_sequence || t1 < tiles))
            a.splits[by_sequence ? n : w] =
                Split{t1 < tiles ? (first + tiles - 1) / chunk - w + 1 : 0, w, s.begin, s.count, group,
                      (int32_t)s.len - (int32_t)s.count};
        const uint32_t r0 = (group * a.RB + rb) * S::rows;
        if (r0 < rows) {
            // The row of this lane, and how many tokens it sees.
            const uint32_t r = min(r0 + srow * HT + opaque(col), rows - 1), ri = r / a.H;
            const int32_t sees = (int32_t)s.len - (int32_t)s.count + (int32_t)ri + 1;
            const int32_t sees_least = (int32_t)s.len - (int32_t)s.count + (int32_t)(r0 / a.H) + 1;
            const int32_t sees_most = (int32_t)s.len - (int32_t)s.count +
                                      (int32_t)(min(r0 + S::rows - 1, rows - 1) / a.H) + 1;
            const uint32_t seen = sees_most > 0 ? (uint32_t)sees_most : 0;
            const uint32_t end = min(t1, (seen + kTile - 1) / kTile);
            u32x4 qf[CG * KS];
            Acc o[RT * OT];
            {
                const float zero = __uint_as_float(opaque(0));
#pragma unroll
                for (int i = 0; i < RT * OT; ++i)
#pragma unroll
                    for (int j = 0; j < (int)(sizeof(Acc) / 4); ++j) o[i][j] = zero;
            }
            float m[RT], l = 0.0f;
#pragma unroll
            for (int i = 0; i < RT; ++i) m[i] = -3.4028235e38f;

            // ---- bringing tiles ---------------------------------------------
            // The wave's eight tokens of a tile's x-th 32, where a page holds whole eights.
            auto eight = [&](uint32_t t, int x) {
                return __builtin_amdgcn_readfirstlane(
                    min(t * kTile + 32 * x + 8 * wave, s.len - 1) & ~7u);
            };
            auto position = [&](uint32_t t, int x) {
                return min(t * kTile + 32 * x + btok, s.len - 1);
            };
            struct Ids {
                uint32_t of[XB];
            };
            auto page_of = [&](uint32_t t) {
                Ids id;
#pragma unroll
                for (int x = 0; x < XB; ++x) {
                    const uint32_t p = DIRECT ? eight(t, x) : position(t, x);
                    id.of[x] = a.pages.table[(size_t)n * a.pages.width + a.pages.page_of(p)];
                }
                return id;
            };
            auto row_of = [&](uint32_t p, uint32_t id) {
                bad_page |= id >= a.pages.pages;
                if (id >= a.pages.pages) id = 0;
                const uint32_t in = p - a.pages.page_of(p) * a.pages.page;
                return a.pool + ((size_t)id * a.pages.page + in) * a.pages.row.bytes;
            };
            constexpr int UNITS = F == K3X_CACHE_MXFP8   ? LP / 128
                                  : F == K3X_CACHE_MXFP4 ? LP / 256
                                  : DIRECT               ? 1
                                                         : LP / 64;
            u32x4 codes[XB][UNITS], scales[XB], turned[XB];
            // A tile's loads, straight to a buffer or to registers, in steps that can stand
            // between products: of each 32 tokens the first finds the rows, the others load.
            struct {
                __amdgpu_buffer_rsrc_t rows8;
                uint32_t from, turn;
                u32x4* dst;
                const uint8_t* row;
            } src;
            constexpr int kSteps = DIRECT ? CG + 1 : UNITS + 3, kBring = XB * kSteps;
            auto bring = [&](int at, uint32_t t, uint32_t b, const Ids& id) {
                const int x = at / kSteps, step = at % kSteps;
                if constexpr (DIRECT) {
                    // Eight tokens a wave, each load 128 bytes of every one.
                    if (step == 0) {
                        const uint32_t p = eight(t, x);
                        const uint8_t* row = row_of(p, __builtin_amdgcn_readfirstlane(id.of[x]));
                        src.rows8 = __builtin_amdgcn_make_buffer_rsrc(
                            const_cast<uint8_t*>(row), 0, 8 * a.pages.row.bytes, 0x00020000);
                        src.from = (position(t, x) - p) * a.pages.row.bytes + bput * 16;
                        // Columns without a rotary part meet zeros of the queries: any
                        // number will do there.
                        src.turn = bput < a.R / 8 ? LP * 2 : 0;
                        src.dst = reinterpret_cast<u32x4*>(smem + b * kBuffer + x * 4096 +
                                                           wave * 1024);
                    } else if (step < CG) {
                        load_lds16(src.rows8, src.dst + (step - 1) * (kGroup / 16), src.from,
                                   (step - 1) * 128);
                    } else {
                        load_lds16(src.rows8, src.dst + (CG - 1) * (kGroup / 16),
                                   src.from + src.turn, 0);
                    }
                } else {
                    if (step == 0) {
                        src.row = row_of(position(t, x), id.of[x]);
                    } else if (step <= UNITS) {
                        const uint32_t u = bcol + 8 * (step - 1);
                        codes[x][step - 1] = FULL || u * 16 < a.pages.row.codes
                                                 ? *reinterpret_cast<const u32x4*>(src.row + u * 16)
                                                 : u32x4{};
                    } else if (step == UNITS + 1) {
                        if constexpr (F != K3X_CACHE_16BIT)
                            scales[x] =
                                *reinterpret_cast<const u32x4*>(src.row + a.pages.row.scales);
                    } else {
                        turned[x] = *reinterpret_cast<const u32x4*>(
                            src.row + (bcol < a.R / 8 ? a.pages.row.codes + bcol * 16 : 0));
                    }
                }
            };
            auto bring_all = [&](uint32_t t, uint32_t b, const Ids& id) {
#pragma unroll
                for (int i = 0; i < kBring; ++i) bring(i, t, b, id);
            };
            // Codes in registers to the values that they stand for in buffer b, in steps.
            // 16 bytes of values a step, so that each passes beside one product.
            constexpr int PER = F == K3X_CACHE_MXFP4 ? 4 : F == K3X_CACHE_MXFP8 ? 2 : 1;
            constexpr int kPutSteps = UNITS * PER + 1, kPut = DIRECT ? 0 : XB * kPutSteps;
            auto put = [&](int at, uint32_t b) {
                if constexpr (!DIRECT) {
                    const int i = at / kPutSteps, step = at % kPutSteps;
                    uint8_t* dst = smem + b * kBuffer + i * 4096 + btok * 128;
                    const uint32_t z = swizzle(btok);
                    if (step == UNITS * PER) {
                        *reinterpret_cast<u32x4*>(dst + (CG - 1) * kGroup + (bcol ^ z) * 16) =
                            turned[i] & (bcol < a.R / 8 ? 0xffffffffu : 0u);
                        return;
                    }
                    const int k = step / PER, j = step % PER;
                    const uint32_t u = bcol + 8 * k;
                    if constexpr (F == K3X_CACHE_16BIT) {
                        if (u * 8 < a.L)
                            *reinterpret_cast<u32x4*>(dst + k * kGroup + (bcol ^ z) * 16) =
                                codes[i][k];
                    } else if constexpr (F == K3X_CACHE_MXFP8) {
                        const float sc = e8m0_to_f32(scales[i][k] >> (bcol / 2 * 8) & 0xff);
                        const uint32_t x = 2 * (u % 4) + j;
                        if (FULL || u * 16 < a.L)
                            *reinterpret_cast<bf16x8*>(dst + u / 4 * kGroup + (x ^ z) * 16) =
                                mxfp8_8(uint2{codes[i][k][2 * j], codes[i][k][2 * j + 1]}, sc);
                    } else {
                        const uint32_t dw = bcol / 4 ? scales[i][2 * k + 1] : scales[i][2 * k];
                        const float sc = e8m0_to_f32(dw >> (bcol % 4 * 8) & 0xff);
                        const uint32_t x = 4 * (u % 2) + j;
                        if (FULL || u * 32 < a.L)
                            *reinterpret_cast<bf16x8*>(dst + u / 2 * kGroup + (x ^ z) * 16) =
                                dequant8(codes[i][k][j], sc);
                    }
                }
            };

            auto load_queries = [&] {
                const uint32_t half = opaque(g);
                const uint8_t* q = static_cast<const uint8_t*>(a.q) +
                                   2 * ((uint64_t)(s.begin + ri) * a.qs +
                                        (uint64_t)(r - ri * a.H) * (a.L + a.R));
#pragma unroll
                for (int c = 0; c < CG; ++c)
#pragma unroll
                    for (int i = 0; i < KS; ++i) {
                        // Columns of the latent, then of the rotary part.
                        const uint32_t d = (c < CG - 1 ? c * 64 : 0) + (i * (8 / KS) + half) * 8;
                        const bool in = c < CG - 1 ? FULL || d < a.L : d < a.R;
                        const u32x4 x = *reinterpret_cast<const u32x4*>(
                            q + (in ? 2 * (c < CG - 1 ? d : a.L + d) : 0));
                        qf[c * KS + i] = x & (in ? 0xffffffffu : 0u);
                    }
            };

            // ---- one tile ---------------------------------------------------
            // Beside its products the loads of a later tile: direct ones to buffer nb; through
            // registers, tile t + 1 from them to the other buffer, then tile t + 2 to them.
            auto tile = [&](uint32_t t, uint32_t b, uint32_t nb, const Ids& id) {
                const lds_byte* kb = lds + b * kBuffer;
                const lds_byte* sb = kb + side * 4096;
                // Operands are read a few products ahead: LDS takes some 200 cycles for four
                // waves at once, a product 32.  (Left to itself the scheduler reads all of
                // them first, past the registers there are.)
                constexpr int XT = HT == 32 ? 1 : 2, HV = HT == 32 ? kTile / 16 : kTile / 32;
                constexpr int NK = CG * KS * XT, NW = OT * HV * RT;
                Acc sc[XT];
#pragma unroll
                for (int i = 0; i < XT; ++i) sc[i] = Acc{};
                // A later tile's loads beside product i of both: direct ones beside the scores',
                // those through registers, with what is done to codes, beside all.
                auto beside = [&](int i) {
                    constexpr int n = DIRECT ? NK : NK + NW;
#pragma unroll
                    for (int x = 0; x < kPut + kBring; ++x)
                        if (x * n / (kPut + kBring) == i) {
                            if (x < kPut) put(x, nb);
                            else bring(x - kPut, min(t + (DIRECT ? BUFS - 1 : 2), end - 1), nb, id);
                        }
                };
                u32x4 kf[AHEAD];
                const uint32_t kat = opaque(kat0);
                auto keys = [&](int i) {
                    const int c = i / (KS * XT), y = i / XT % KS, x = i % XT;
                    kf[i % AHEAD] = lds16(sb + c * kGroup + x * 2048 + (kat ^ y * (128 / KS)));
                };
                // (Without a rotary part its group is zeros.)
#pragma unroll
                for (int i = 0; i < AHEAD - 1; ++i) keys(i);
#pragma unroll
                for (int i = 0; i < NK; ++i) {
                    if (i + AHEAD - 1 < NK) keys(i + AHEAD - 1);
                    beside(i);
                    __builtin_amdgcn_sched_barrier(0);
                    sc[i % XT] = M::run(kf[i % AHEAD], qf[i / XT], sc[i % XT]);
                    __builtin_amdgcn_sched_barrier(0);
                }
                u32x4 vf[AHEAD];
                const uint32_t vat = opaque(vat0);
                auto values = [&](int i) {
                    const int y = i / HV, h = i % HV;
                    const uint32_t d = y + wd * OT;  // tile of HT columns of the latent
                    const lds_byte* vb = kb + d * HT / 64 * kGroup + h * 2048;
                    const uint32_t at = vat ^ y % (64 / HT) * (HT * 2);
                    // Tokens 16 h .. 16 h + 15 (or all 32), by fours of each half.
                    const uint2 v0 = lds_transposed(vb + at);
                    const uint2 v1 = HT == 32 ? lds_transposed(vb + 1024 + (at ^ 16))
                                              : lds_transposed(vb + 2048 + at);
                    vf[i % AHEAD] = u32x4{v0.x, v0.y, v1.x, v1.y};
                };
#pragma unroll
                for (int i = 0; i < AHEAD - 1; ++i) values(i);  // while weights are formed
                constexpr int NV = HT == 32 ? 16 : 8;
                float x[NV];
#pragma unroll
                for (int i = 0; i < NV; ++i) x[i] = HT == 32 ? sc[0][i] : sc[i / 4][i % 4];
                if ((int32_t)((t + 1) * kTile) > sees_least) {
                    // Past what the row sees.
#pragma unroll
                    for (int i = 0; i < NV; ++i) {
                        const int32_t tok = (int32_t)(t * kTile + side * 32) +
                                            (HT == 32 ? 8 * (i / 4) + 4 * (int)g + i % 4
                                                      : 16 * (i / 4) + 4 * (int)g + i % 4);
                        if (tok >= sees) x[i] = -__builtin_inff();
                    }
                }
                float top = x[0];
#pragma unroll
                for (int i = 1; i < NV; ++i) top = fmaxf(top, x[i]);
                top = across<HT>(top, [](float p, float r) { return fmaxf(p, r); }) * a.rate;
                constexpr bool HELD = RT * OT * sizeof(Acc) >= 512;
                float now = RT > 1 && srow ? m[RT - 1] : m[0];
                const bool over = __any(Weights<DT>::over(top, now));
                uint32_t p[NV / 2];
                float sum;
                auto weights = [&] {
                    sum = 0.0f;
#pragma unroll
                    for (int i = 0; i < NV; i += 2) {
                        const float u = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i], a.rate, -now));
                        const float v =
                            __builtin_amdgcn_exp2f(__builtin_fmaf(x[i + 1], a.rate, -now));
                        sum += u + v;
                        p[i / 2] = pack2<DT>(u, v);
                    }
                };
                u32x4 pf[RT * HV];  // weights as the operands of the second products
                if constexpr (JOINT) {
                    // The wave's weights to all waves, formed again if for any the maximum
                    // is passed.
                    auto share = [&] {
                        weights();
                        if (wave / 2 < RT)
#pragma unroll
                            for (int h = 0; h < 2; ++h)
                                *reinterpret_cast<u32x4*>(
                                    smem + kWeights + (srow * 4 + side * 2 + h) * 1024 +
                                    lane * 16) =
                                    u32x4{p[4 * h], p[4 * h + 1], p[4 * h + 2], p[4 * h + 3]};
                    };
                    share();
                    auto take = [&] {
#pragma unroll
                        for (int i = 0; i < RT * HV; ++i)
                            pf[i] = lds16(lds + kWeights + i * 1024 + lane * 16);
                    };
                    if (g == 0)
                        *reinterpret_cast<float*>(smem + kTops + (srow * 2 + side) * 128 +
                                                  col * 4) = top;
                    if (lane == 0) *reinterpret_cast<uint32_t*>(smem + kFlags + wave * 4) = over;
                    barrier();
                    const u32x4 flags = lds16(lds + kFlags);
                    take();
                    __builtin_amdgcn_sched_barrier(0);
                    if (__builtin_amdgcn_readfirstlane(flags[0] | flags[1] | flags[2] |
                                                       flags[3])) {
#pragma unroll
                        for (int i = 0; i < RT; ++i) {
                            const float* tops = reinterpret_cast<const float*>(smem + kTops);
                            const float up = Weights<DT>::reference(
                                fmaxf(tops[i * 64 + col], tops[i * 64 + 32 + col]), m[i]);
                            const float keep = __builtin_amdgcn_exp2f(m[i] - up);
                            m[i] = up;
                            if ((uint32_t)i == srow) l *= keep;
                            if (t != t0) {
                                if (i == 0) scale_tiles<HELD, 0, OT>(o, keep);
                                else scale_tiles<HELD, (RT - 1) * OT, OT>(o, keep);
                            }
                        }
                        now = RT > 1 && srow ? m[RT - 1] : m[0];
                        share();
                        barrier();
                        take();
                    }
                    l += sum;
                } else {
                    if (over) {
                        const float up = Weights<DT>::reference(top, m[0]);
                        const float keep = __builtin_amdgcn_exp2f(m[0] - up);
                        m[0] = now = up;
                        l *= keep;
                        if (t != t0) scale_tiles<HELD, 0, OT>(o, keep);
                    }
                    weights();
                    l += sum;
#pragma unroll
                    for (int h = 0; h < HV; ++h)
                        pf[h] = u32x4{p[4 * h], p[4 * h + 1], p[4 * h + 2], p[4 * h + 3]};
                }
#pragma unroll
                for (int i = 0; i < NW; ++i) {
                    const int v = i / RT, z = i % RT, y = v / HV, h = v % HV;
                    if (z == 0 && v + AHEAD - 1 < NW / RT) values(v + AHEAD - 1);
                    beside(NK + i);
                    __builtin_amdgcn_sched_barrier(0);
                    o[z * OT + y] = M::run(vf[v % AHEAD], pf[z * HV + h], o[z * OT + y]);
                    __builtin_amdgcn_sched_barrier(0);
                }
            };

            // ---- the piece's tiles --------------------------------------------
            if (t0 < end) {
                if constexpr (DIRECT) {
                    // BUFS - 1 tiles on their way.  When one is used, the loads of the
                    // later ones may be outstanding, and no others are behind its own.
                    Ids id = page_of(t0), next;
#pragma unroll
                    for (uint32_t i = 0; i < BUFS - 1; ++i) {
                        next = page_of(min(t0 + i + 1, end - 1));
                        bring_all(min(t0 + i, end - 1), i, id);
                        id = next;
                    }
                    load_queries();
                    uint32_t b = 0;
                    for (uint32_t t = t0; t < end; ++t) {
                        wait_loads<(BUFS - 2) * CG>();
                        barrier();
                        next = page_of(min(t + BUFS, end - 1));
                        tile(t, b, b >= 1 ? b - 1 : BUFS - 1, id);
                        id = next;
                        b = b + 1 == BUFS ? 0 : b + 1;
                    }
                    wait_loads<0>();
                    barrier();
                } else {
                    const Ids id = page_of(t0);
                    Ids next = page_of(min(t0 + 1, end - 1));
                    bring_all(t0, 0, id);
                    load_queries();
#pragma unroll
                    for (int i = 0; i < kPut; ++i) put(i, 0);
                    bring_all(min(t0 + 1, end - 1), 0, next);
                    next = page_of(min(t0 + 2, end - 1));
                    uint32_t b = 0;
                    for (uint32_t t = t0; t < end; ++t) {
                        barrier();
                        const Ids now = next;
                        next = page_of(min(t + 3, end - 1));
                        tile(t, b, b ^ 1, now);
                        b ^= 1;
                    }
                    barrier();
                }
            }

            // ---- out ----------------------------------------------------------
            l = across<HT>(l, [](float p, float r) { return p + r; });
            float ls[RT];
            ls[0] = l;
            if constexpr (JOINT) {
                // Of both halves of the tokens, for all waves.
                float* sums = reinterpret_cast<float*>(smem + kTops);
                barrier();
                if (g == 0) sums[(srow * 2 + side) * 32 + col] = l;
                barrier();
#pragma unroll
                for (int i = 0; i < RT; ++i) ls[i] = sums[i * 64 + col] + sums[i * 64 + 32 + col];
                barrier();
            }
            const size_t piece = ((size_t)w * a.RB + rb) * 2 + (t0 ? 0 : 1);
            constexpr int Q = HT == 32 ? 4 : 1;
            auto block = [&](auto which) {
                constexpr int z = decltype(which)::value;
                const uint32_t at = (wm * RT + z) * HT;  // of the workgroup's rows
                const float m1 = m[z], l1 = ls[z];
                const bool live = r0 + at + col < rows;
                const float inv = !whole ? 1.0f : l1 > 0.0f ? 1.0f / l1 : 0.0f;
                const uint32_t re = min(r0 + at + opaque(col), rows - 1);
                const uint64_t row = s.begin + re / a.H;
                const uint32_t head = re % a.H;
                uint16_t* out =
                    static_cast<uint16_t*>(a.out) + row * a.os + (uint64_t)head * a.L;
                float4* part = a.parts + piece * (S::rows * LP / 4) +
                               (wave * RT + z) * OT * Q * 64 + lane;
                float check = l1 * 0.0f;  // NaN once something is not finite
                auto each = [&](auto put4) {
#pragma unroll
                    for (int y = 0; y < OT; ++y) {
#pragma unroll
                        for (int i = 0; i < Q; ++i) {
                            const uint32_t d = (y + wd * OT) * HT + 8 * i + 4 * g;
                            const Acc& u = o[z * OT + y];
                            const float4 v{u[4 * i] * inv, u[4 * i + 1] * inv, u[4 * i + 2] * inv,
                                           u[4 * i + 3] * inv};
                            if (!FULL && d >= a.L) continue;
                            check = __builtin_fmaf(v.x, 0.0f, check);
                            check = __builtin_fmaf(v.y, 0.0f, check);
                            check = __builtin_fmaf(v.z, 0.0f, check);
                            check = __builtin_fmaf(v.w, 0.0f, check);
                            put4(y * Q + i, d, v);
                        }
                        __builtin_amdgcn_sched_barrier(0);
                    }
                };
                if (!whole)
                    each([&](int f, uint32_t, float4 v) { part[f * 64] = v; });
                else if (live)
                    each([&](int, uint32_t d, float4 v) {
                        *reinterpret_cast<uint2*>(out + d) = outputs4<DT>(v);
                    });
                bad_value |= live && !(check == 0.0f);
                if (whole)
                    bad_value |= live && no_softmax<DT>((int32_t)s.len - (int32_t)s.count +
                                                            (int32_t)(re / a.H) + 1, l1, m1);
                if (g == 0 && wd == 0) {
                    if (!whole)
                        a.sums[piece * S::rows + at + col] = float2{m1, l1};
                    else if (a.lse && live)
                        a.lse[row * a.H + head] =
                            l1 > 0.0f ? (m1 + __builtin_amdgcn_logf(l1)) * 0.69314718055994531f
                                      : -__builtin_inff();
                }
            };
            block(std::integral_constant<int, 0>{});
            if constexpr (RT > 1) block(std::integral_constant<int, 1>{});
        }
        first += tiles;
        if (first >= to) break;
        if (++group < groups_in(a, s, S::rows)) continue;
        group = 0;
        do ++n;
        while (n < a.pages.N && !tiles_of<kTile>(a, n, S::rows, &s));
        if (n == a.pages.N) break;
    }
    if (bad_page) latch(a.status, K3X_ERR_INVALID_STATE);
    if (bad_value) latch(a.status, K3X_ERR_INVALID_MXFP4);
}

// A call of no tokens: its offsets and lengths are looked at all the same.
__global__ __launch_bounds__(kThreads) void mla_check_kernel(Pages pages, uint32_t* status) {
    check_sequences(pages, status);
}

// Joins the pieces of a sequence that lies in several ranges, 64 float4 as a
// wave of the first launch held them: a wave each, or (FOUR, for many pieces) four
// waves, each every fourth piece.
template <uint32_t DT, int LP, typename S, bool FOUR>
__global__ __launch_bounds__(kThreads) void mla_join_kernel(AttentionArgs a) {
    constexpr int HT = S::HT, WD = S::WD, RT = S::RT;
    constexpr uint32_t kSlices = S::rows * LP / (FOUR ? 256 : 1024);
    constexpr uint32_t NF = LP / HT / WD * (HT == 32 ? 4 : 1);
    __shared__ float4 os[FOUR ? 4 : 1][64];
    __shared__ float2 ls[FOUR ? 4 : 1][64];
    const uint32_t slice = blockIdx.x % kSlices, x = blockIdx.x / kSlices;
    const uint32_t rb = x % a.RB, lane = threadIdx.x & 63, quarter = threadIdx.x / 64;
    const uint32_t status = *(volatile uint32_t*)a.status;
    const Split s = a.splits[x / a.RB];
    const uint32_t rows = s.count * a.H;
    const uint32_t r0 = (s.group * a.RB + rb) * S::rows;
    if (status || !s.pieces || r0 >= rows) return;
    const uint32_t f = FOUR ? slice : slice * 4 + quarter, wave = f / NF, i = f % NF;
    const uint32_t wd = wave / RT % WD;  // (wave: with its block of rows)
    const uint32_t at = (wave / RT / WD * RT + wave % RT) * HT + lane % HT, r = r0 + at;
    const uint32_t d = HT == 32 ? wd * (LP / WD) + i / 4 * 32 + i % 4 * 8 + lane / 32 * 4
                                : wd * (LP / WD) + i * 16 + lane / 16 * 4;
    const bool live = r < rows && d < a.L;
    auto piece = [&](uint32_t p) { return ((size_t)(s.w + p) * a.RB + rb) * 2 + (p ? 0 : 1); };
    float m = -3.4028235e38f, l = 0.0f;
    float4 o{};
    constexpr uint32_t kStep = FOUR ? 4 : 1, kAhead = 4;
    for (uint32_t p0 = FOUR ? quarter : 0; p0 < s.pieces; p0 += kStep * kAhead) {
        float2 ml[kAhead];
        float4 v[kAhead];
#pragma unroll
        for (uint32_t j = 0; j < kAhead; ++j) {
            const size_t q = piece(min(p0 + j * kStep, s.pieces - 1));
            ml[j] = a.sums[q * S::rows + at];
            v[j] = live ? a.parts[q * (S::rows * LP / 4) + f * 64 + lane] : float4{};
        }
        float top = m;
#pragma unroll
        for (uint32_t j = 0; j < kAhead; ++j) top = fmaxf(top, ml[j].x);
        const float keep = __builtin_amdgcn_exp2f(m - top);
        m = top;
        l *= keep;
        o = float4{o.x * keep, o.y * keep, o.z * keep, o.w * keep};
#pragma unroll
        for (uint32_t j = 0; j < kAhead; ++j) {
            // A piece that the row does not see has no sum, and may hold no outputs.
            if (p0 + j * kStep >= s.pieces || !(ml[j].y > 0.0f)) continue;
            const float k = __builtin_amdgcn_exp2f(ml[j].x - m);
            l = __builtin_fmaf(ml[j].y, k, l);
            o.x = __builtin_fmaf(v[j].x, k, o.x);
            o.y = __builtin_fmaf(v[j].y, k, o.y);
            o.z = __builtin_fmaf(v[j].z, k, o.z);
            o.w = __builtin_fmaf(v[j].w, k, o.w);
        }
    }
    if constexpr (FOUR) {
        os[quarter][lane] = o;
        ls[quarter][lane] = float2{m, l};
        __syncthreads();
        if (quarter) return;
        for (int j = 1; j < 4; ++j) m = fmaxf(m, ls[j][lane].x);
        l = 0.0f;
        o = float4{};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float k = __builtin_amdgcn_exp2f(ls[j][lane].x - m);
            const float4 v = os[j][lane];
            l = __builtin_fmaf(ls[j][lane].y, k, l);
            o.x = __builtin_fmaf(v.x, k, o.x);
            o.y = __builtin_fmaf(v.y, k, o.y);
            o.z = __builtin_fmaf(v.z, k, o.z);
            o.w = __builtin_fmaf(v.w, k, o.w);
        }
    }
    if (!live) return;
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    const uint64_t t = s.begin + r / a.H;
    uint16_t* out = static_cast<uint16_t*>(a.out) + t * a.os + (uint64_t)(r % a.H) * a.L + d;
    o = float4{o.x * inv, o.y * inv, o.z * inv, o.w * inv};
    // Pieces that are numbers may have a sum that is none.
    const float check = o.x * 0.0f + o.y * 0.0f + o.z * 0.0f + o.w * 0.0f;
    if (!(check == 0.0f) || no_softmax<DT>(s.before + (int32_t)(r / a.H) + 1, l, m))
        latch(a.status, K3X_ERR_INVALID_MXFP4);
    *reinterpret_cast<uint2*>(out) = outputs4<DT>(o);
    if (a.lse && d == 0)
        a.lse[t * a.H + r % a.H] = l > 0.0f ? (m + __builtin_amdgcn_logf(l)) * 0.69314718055994531f
                                            : -__builtin_inff();
}

// How a call is laid out: rows of a workgroup, ranges, row blocks.
struct Plan {
    uint32_t rows, G, RB, LP;
    bool full, one;
};
Plan plan_of(const k3x_hip_mla_params* p) {
    Plan x;
    const uint64_t most = (uint64_t)(p->longest ? p->longest : p->tokens) * p->heads;
    x.LP = p->latent <= 256 ? 256 : 512;
    // As few rows as hold a sequence's: 16 heads, 64 sequences of 8192 tokens in 16 and 4 bits
    // 120 and 81 us, with 32 rows 126 and 92.  More than 64 in blocks of 64, or of 128 once those
    // of all sequences are 64: half as many reads of the cache and of LDS, but twice the
    // outputs of a range for the join.  128 heads, 16 bits, in blocks of 128 and of 64: 8
    // sequences of 16384 69.6 and 58.4 us, 32 of 2048 57.3 and 43.1, of 8192 113 and 107; 64
    // of 1000 54.5 and 45.5, of 4096 108 and 110, of 8192 184 and 198, in 8 bits 184 and 220.
    x.rows = most <= 16 ? 16 : most <= 32 ? 32 : most <= 64 ? 64 : 128;
    if (x.rows == 128 && (most + 127) / 128 * p->sequences < 64) x.rows = 64;
    x.full = p->latent == x.LP && (p->cache_format != K3X_CACHE_16BIT || p->page_size % 8 == 0);
    if (!x.full && x.rows > 16) x.rows = 64;  // the others: two shapes
    // The row blocks of a sequence run side by side and share its cached tokens; of more than
    // eight a group of as many as sequences have on average, so that a long window does not
    // leave single tokens beside it to one workgroup: a window of 512 tokens and 63 tokens over
    // 4096 each, 128 heads in 16 bits, 358 us, with all blocks of a sequence in one group 13274;
    // the window alone 179, and 492.
    const uint64_t blocks = std::max<uint64_t>(1, (most + x.rows - 1) / x.rows);
    const uint64_t average = (uint64_t)p->tokens * p->heads / p->sequences / x.rows + 1;
    x.one = blocks <= 8;
    x.RB = (uint32_t)(x.one ? blocks : std::min<uint64_t>(8, average));
    // Two workgroups a compute unit where registers and LDS allow.
    const uint32_t places = x.rows == 16 ? 512 : 256;
    x.G = std::max(1u, places / x.RB);
    if (x.G >= 8) x.G -= x.G % 8;
    return x;
}
size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

template <uint32_t DT, uint32_t F, int LP, typename S, bool FULL>
int launch(k3x_hip_ctx* ctx, const AttentionArgs& a) {
    // Tiles in LDS: what it holds, for two workgroups of 16 rows.
    constexpr int BUFS = F == K3X_CACHE_16BIT && FULL && S::rows == 128 ? 3 : 2;
    hipLaunchKernelGGL((mla_attention_kernel<DT, F, LP, S, BUFS, FULL>), dim3(a.G * a.RB),
                       dim3(kThreads), 0, ctx->stream, a);
    const uint32_t splits = (a.one ? std::min(a.G, a.pages.N) : a.G) * a.RB;
    // Eight ranges a sequence and more: pieces by four waves.  One sequence in 250 ranges, 16
    // heads: 26 us, with one wave 59; 64 in 4 each, 128 heads: 195, with one wave 181.
    if (a.G / a.pages.N >= 8)
        hipLaunchKernelGGL((mla_join_kernel<DT, LP, S, true>), dim3(splits * (S::rows * LP / 256)),
                           dim3(kThreads), 0, ctx->stream, a);
    else
        hipLaunchKernelGGL((mla_join_kernel<DT, LP, S, false>),
                           dim3(splits * (S::rows * LP / 1024)), dim3(kThreads), 0, ctx->stream, a);
    return launched(ctx, 2);
}

template <uint32_t DT, uint32_t F, int LP>
int launch_shape(k3x_hip_ctx* ctx, const AttentionArgs& a, const Plan& x) {
    if (!x.full)
        return x.rows == 16 ? launch<DT, F, LP, Shape<16, 1, 4, 1, 32>, false>(ctx, a)
                            : launch<DT, F, LP, Shape<32, 2, 2, 1, 32>, false>(ctx, a);
    switch (x.rows) {
        case 16: return launch<DT, F, LP, Shape<16, 1, 4, 1, 32>, true>(ctx, a);
        case 32: return launch<DT, F, LP, Shape<32, 1, 4, 1, 64>, true>(ctx, a);
        case 64: return launch<DT, F, LP, Shape<32, 1, 4, 2, 64>, true>(ctx, a);
        default: return launch<DT, F, LP, Shape<32, 4, 1, 1, 32>, true>(ctx, a);
    }
}
template <uint32_t DT, uint32_t F>
int launch_width(k3x_hip_ctx* ctx, const AttentionArgs& a, const Plan& x) {
    return x.LP == 256 ? launch_shape<DT, F, 256>(ctx, a, x) : launch_shape<DT, F, 512>(ctx, a, x);
}

bool attention_ok(const k3x_hip_mla_params* p) {
    if (!mla_ok(p)) return false;
    const Plan x = plan_of(p);
    return (uint64_t)(p->longest ? p->longest : p->tokens) * p->heads < (1ull << 31) && x.G;
}

}  // namespace

extern "C" {

size_t k3x_hip_mla_attention_workspace(const k3x_hip_mla_params* p) {
    if (!p || !attention_ok(p)) return 0;
    const Plan x = plan_of(p);
    const size_t pieces = (size_t)x.G * x.RB * 2;
    return up256(x.G * sizeof(Split)) + up256(pieces * x.rows * sizeof(float2)) +
           pieces * x.rows * x.LP * sizeof(float);
}

int k3x_hip_mla_attention(k3x_hip_ctx* ctx, const k3x_hip_mla_params* p, const void* q,
                          const void* pool, const uint32_t* table, const uint32_t* offsets,
                          const uint32_t* lens, void* out, float* lse, void* workspace,
                          size_t workspace_bytes) {
    if (!ctx || !p || !attention_ok(p) || (p->tokens && (!q || !out)) || !pool || !table ||
        !lens || p->q_stride % 8 || p->out_stride % 8)
        return K3X_ERR_INVALID_EXTENT;
    if (!aligned(q, 16) || !aligned(out, 16) || !aligned(pool, 256) || !aligned(table, 4) ||
        !aligned(offsets, 4) || !aligned(lens, 4) || !aligned(lse, 4))
        return K3X_ERR_INVALID_EXTENT;
    if (!workspace || !aligned(workspace, 256) ||
        workspace_bytes < k3x_hip_mla_attention_workspace(p))
        return K3X_ERR_INVALID_EXTENT;
    if (hipSetDevice(ctx->device) != hipSuccess) return K3X_ERR_BACKEND_UNAVAILABLE;
    const Plan x = plan_of(p);
    AttentionArgs a{};
    a.pages = pages_of(p, table, offsets, lens);
    a.q = q;
    a.pool = static_cast<const uint8_t*>(pool);
    a.out = out;
    a.lse = lse;
    a.H = p->heads;
    a.L = p->latent;
    a.R = p->rotary;
    a.qs = p->q_stride ? p->q_stride : (uint64_t)p->heads * (p->latent + p->rotary);
    a.os = p->out_stride ? p->out_stride : (uint64_t)p->heads * p->latent;
    a.rate = p->scale * 1.4426950408889634f;
    a.G = x.G;
    a.RB = x.RB;
    a.one = x.one;
    uint8_t* w = static_cast<uint8_t*>(workspace);
    const size_t pieces = (size_t)x.G * x.RB * 2;
    a.splits = reinterpret_cast<Split*>(w);
    w += up256(x.G * sizeof(Split));
    a.sums = reinterpret_cast<float2*>(w);
    w += up256(pieces * x.rows * sizeof(float2));
    a.parts = reinterpret_cast<float4*>(w);
    a.status = ctx->status;
    if (!p->tokens) {
        hipLaunchKernelGGL(mla_check_kernel, dim3(1), dim3(kThreads), 0, ctx->stream, a.pages,
                           a.status);
        return launched(ctx, 1);
    }
    if (p->dtype == K3X_DTYPE_F16) return launch_width<K3X_DTYPE_F16, K3X_CACHE_16BIT>(ctx, a, x);
    switch (p->cache_format) {
        case K3X_CACHE_16BIT: return launch_width<K3X_DTYPE_BF16, K3X_CACHE_16BIT>(ctx, a, x);
        case K3X_CACHE_MXFP8: return launch_width<K3X_DTYPE_BF16, K3X_CACHE_MXFP8>(ctx, a, x);
        default: return launch_width<K3X_DTYPE_BF16, K3X_CACHE_MXFP4>(ctx, a, x);
    }
}

}  // extern "C"
