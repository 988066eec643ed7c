// paged_attention.cu - attention of new tokens over the paged key / value cache: s_j = scale * q.k_j over the keys a token sees,
// out = sum_j e^{s_j} v_j / sum_j e^{s_j}, in one pass over the keys with a running maximum and sum.
//
// Bound by HBM where there is enough to read: a key and its value come once for the G heads of their group and carry 4 G D operations, G / 2
// a byte of bf16, G a byte of e4m3.  That keeps the tensor pipe a tenth to a fifth busy with warp-wide MMAs of 8 or 16 columns, whose operands
// can be any lines of memory (64 ragged requests 14 %, e4m3 26 %); what runs short before it is instructions, and in small calls latency.
//
// A warp's tile is 16 keys of one kv head.  Keys are the MMAs' rows and heads their columns, 8 a column tile (NT of them), so that a
// group of 8 heads wastes nothing: scores S [16 keys][8 heads] = K Q^T, out O^T [D][8 heads] += V^T P^T.  Operands are read as their
// fragments, 16 bytes a lane:
//   K, rows: lane (g, j) = (lane / 4, lane % 4) has keys g and g + 8, of each block of 4 x 16 bytes the j-th 16 bytes.  A k-step of 16
//     then takes the values in an order of its own, and Q is loaded in the same order.
//   V^T, rows: lane (g, j) has keys 2j, 2j + 1, 2j + 8, 2j + 9, of each block of 8 x 16 bytes the g-th 16 bytes; a byte permutation of two
//     keys' words gives the pairs along the keys that the fragment wants, for two neighbouring rows of D.
//   P^T: the scores' fragment has keys along its rows; one 8 x 8 transposition a key octet (movmatrix) turns it.
// The weights enter the second product as two terms, p = hi + lo, each rounded to the operands' type: 16 bits or more of p in place of
// bf16's 8, for half as many MMAs again, which the loads leave room for.  e4m3 values become fp16 exactly; q then is fp16
// too, each head's row scaled by a power of two to the range of 1 (what falls below fp16's range is 2^-24 of the row's largest value).
// Maximum, sum and out stay in fp32, and so does every addition over the keys: the tensor core cuts off, it does not round, where it adds
// to an accumulator, always towards zero, so a tile's product starts from zero and is added by an fp32 instruction.  A tile's maximum
// is taken across lanes only when some lane is above the running one.
//
// Keys in flight: every warp has a ring of half tiles in shared memory (K, V, K, V ...), filled by its own asynchronous copies of 16 bytes a
// lane, three to eight halves deep; no barrier stands inside the loop.  With three blocks of four warps an SM that is 100 to 150 KB under
// way, twice what HBM's latency asks for.  (Tiles straight into registers: 64 ragged requests 80 us, rings and the rule below 62.)
//
// Work is split by keys, not by requests: all tokens' keys in chunks form one line, of which each block takes an equal run, whatever
// the lengths.  A unit is a (token, kv head, head group); its fixed work (Q, page ids, the parts' joining) counts as four chunks of the
// line (64 ragged requests: as none 95 us, as two 66, as four 62, as eight 63).  A block that has all of a unit's chunks writes its rows,
// else it leaves maximum, sum and out in the workspace, and the block that comes last joins the parts in their order, so that a call's
// bits do not depend on which that was; many parts are joined in two steps (131072 keys, 148 parts: 103 us in one, 56 in two).  The line's
// running sums are made by every block itself up to 512 tokens, by a launch before beyond.
//
// Measured on a B200, device time in a graph, three caches in turn: 64 requests of 17 to 8191 keys, 32 / 8 heads of 128, bf16, 353, 420 and
// 425 MB: 65, 74 and 76 us, 5.4 to 5.6 TB/s; 256 of 500 to 8000, 64 / 8, e4m3, 1.39, 1.44 and 1.50 GB: 255, 257 to 264 and 267 us, 5.4 to
// 5.6 TB/s (54 % of the issue slots); one of 131072, 16 / 2 heads of 256, bf16, 268 MB: 56 us, 4.8 TB/s (400000 keys: 135 us, 6.1 TB/s); one
// of 1000, 32 / 4 of 128: 10.2 us, of which 5.5 are an unsplit call's.
#include "paged.cuh"
#include "pdl.cuh"

#include <atomic>
#include <cfloat>

#include <cuda_fp16.h>
#include <cuda_fp8.h>

namespace bsx {
namespace {

constexpr int kAttnThreads = 128;
constexpr int kWarps = kAttnThreads / 32;
// up to so many tokens every block makes the line's running sums itself, beyond a launch before does (us, itself and by the launch: 64 requests
// of 64 keys 10.4, 12.5; 512 of 64 41, 45; 512 of 700 241, 244)
constexpr int kScanTokens = 512;
constexpr int kMaxSms = 148;
// Parts of a unit that one block joins at a time.  A join holds of each part a column of four values a thread (2 KB) and a weight for every
// head of the unit, first of so many parts, then of as many joined ones as the device's blocks make: see Shape
constexpr int join_size(int unit_heads) { return unit_heads <= 16 ? 15 : unit_heads <= 32 ? 18 : 20; }
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct AttnParams {
    const uint16_t* q;
    const void *k, *v;
    const float *k_scale, *v_scale, *sinks;
    const int32_t *table, *pos, *row;
    void* out;
    float* lse;
    int32_t* status;
    uint32_t* counter;       // three a block, 0 between calls
    float* parts;            // two slots a block
    long long* line;         // running sums of more than kScanTokens tokens
    int64_t q_stride, table_stride;
    uint32_t k_page, v_page, n_pages;   // bytes from page to page
    float scale, softcap;
    int32_t hq, hk, group, T, n_rows, max_pages, page_shift, window, out_kind;
    int32_t sets, group_sets; // the heads that one warp has are a set: of a token, of a kv head
    int32_t head_shift;      // 2^it warps of a block have other sets, the rest of the warps other keys
    int32_t units;           // of a token: sets / head_warps, rounded up
};

// what token t sees: keys [begin, end) of a table row
struct Seen {
    int row, begin, end;
};
__device__ __forceinline__ int begin_of(const AttnParams& p, int end) { return p.window > 0 && end > p.window ? end - p.window : 0; }
__device__ __forceinline__ Seen seen_by(const AttnParams& p, int t, int& why) {
    Seen s;
    s.row = p.row ? p.row[t] : t;
    int last = p.pos[t];
    const int most = (int) (((int64_t) p.max_pages << p.page_shift) - 1);
    if (s.row >= p.n_rows) s.row = -1, why |= BSX_PAGED_BAD_ROW;
    if (s.row >= 0 && last > most) last = most, why |= BSX_PAGED_BAD_ROW;
    s.end = s.row < 0 ? 0 : max(last + 1, 0);
    s.begin = begin_of(p, s.end);
    return s;
}
constexpr int kSetup = 4;          // a unit's fixed cost, in chunks
// chunks of keys; they begin at a multiple of 16: a tile lies in one page, or in two of 8
__device__ __forceinline__ int chunks_of(const Seen& s, int chunk) { return s.end > s.begin ? (s.end - (s.begin & ~15) + chunk - 1) / chunk : 0; }

__device__ __forceinline__ int length_of(int chunks) { return chunks ? chunks + kSetup : 0; }   // on the line

// a / b of non-negative numbers, in 32 bits where they fit, as they nearly always do
__device__ __forceinline__ long long quotient(long long a, long long b) { return (a | b) >> 32 ? a / b : (long long) ((uint32_t) a / (uint32_t) b); }
// Runs the line is cut into, of at most `blocks`; most: the longest unit, 0 where not known.  Short units are not split, longer ones only into
// as many parts as are joined at one time (bf16, one request of 4 kv heads of 128: 256 keys 9.7 us in parts of a chunk, 8.4 whole;
// 2048 keys 12.7 in 32 parts, 11.8 in 11)
__device__ __forceinline__ long long runs_of(long long blocks, long long total, int most) {
    constexpr int kFewest = join_size(8);
    const int chunks = most - kSetup, at_least = most == 0 ? 1 : chunks <= 4 ? most : chunks <= 4 * kFewest ? (chunks + kFewest - 1) / kFewest : 1;
    return at_least == 1 || total >= blocks * at_least ? blocks : max(quotient(total, at_least), 1ll);
}

__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(d) : "r"(a));
    return d;
}
// c = a b, or c + a b
template <bool F16, bool ADD>
__device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    const float z0 = ADD ? c[0] : 0.f, z1 = ADD ? c[1] : 0.f, z2 = ADD ? c[2] : 0.f, z3 = ADD ? c[3] : 0.f;
    if (F16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};\n"
                     : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(z0), "f"(z1), "f"(z2), "f"(z3));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};\n"
                     : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(z0), "f"(z1), "f"(z2), "f"(z3));
}
__device__ __forceinline__ void halves_of_e4m3(uint32_t four, uint32_t& lo, uint32_t& hi) {   // four e4m3 values as fp16 pairs
    asm("{\n.reg .b16 l, h;\nmov.b32 {l, h}, %2;\ncvt.rn.f16x2.e4m3x2 %0, l;\ncvt.rn.f16x2.e4m3x2 %1, h;\n}\n" : "=r"(lo), "=r"(hi) : "r"(four));
}
// (a, b) as the operands' type, a in the low half; and what that rounding left over
template <bool F16>
__device__ __forceinline__ uint32_t pack2(float a, float b, float& ra, float& rb) {
    if (F16) {
        const __half2 h = __floats2half2_rn(a, b);
        const float2 f = __half22float2(h);
        ra = a - f.x, rb = b - f.y;
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    const uint32_t w = *reinterpret_cast<const uint32_t*>(&h);
    ra = a - __uint_as_float(w << 16), rb = b - __uint_as_float(w & 0xffff0000u);
    return w;
}
// 16 bytes to shared memory, past L1 and the registers; zeros without a read where !ok
__device__ __forceinline__ void copy16(uint32_t to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool ok) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(to), "l"(from), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_end() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory"); }   // all but the last N groups
__device__ __forceinline__ void read_shared(uint4& v, uint32_t at) {
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
}
__device__ __forceinline__ void read_shared(uint2& v, uint32_t at) {
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];\n" : "=r"(v.x), "=r"(v.y) : "r"(at));
}
// 1 - 2 / (e^2x + 1), or where that cancels the series x - x^3 / 3 + 2 x^5 / 15 - 17 x^7 / 315 + 62 x^9 / 2835: off by under 2e-7 everywhere
__device__ __forceinline__ float tanh_fast(float x) {
    const float a = fabsf(x), y = x * x;
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(e) : "f"(a * (2.f * kLog2e)));
    const float large = copysignf(1.f - __fdividef(2.f, e + 1.f), x);
    const float small = x * fmaf(y, fmaf(y, fmaf(y, fmaf(y, 62.f / 2835.f, -17.f / 315.f), 2.f / 15.f), -1.f / 3.f), 1.f);
    return a < 0.35f ? small : large;
}
__device__ __forceinline__ uint32_t count_up(uint32_t* counter, uint32_t last) {   // the count before; after `last` it is 0 again
    uint32_t old;
    asm volatile("atom.acq_rel.gpu.global.inc.u32 %0, [%1], %2;\n" : "=r"(old) : "l"(counter), "r"(last) : "memory");
    return old;
}
__device__ __forceinline__ float exp2_fast(float x) {   // 0 where the result falls below the normal range
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}

// blocks an SM: three where 168 registers a thread suffice (256 requests, e4m3, heads of 128: 262 us, two blocks 286; bf16 the same within 1 %)
constexpr int blocks_an_sm(int d, int nt) { return nt == 1 && d <= 128 || d == 64 ? 3 : 2; }

template <int D, int NT, bool E4M3>
struct Shape {
    static constexpr int kHeads = 8 * NT;                    // of a warp
    static constexpr int kBlocks = blocks_an_sm(D, NT);
    static constexpr int kRow = D + 8;                       // of out in shared memory, in values
    static constexpr int kRowBytes = E4M3 ? D : 2 * D;
    static constexpr int kHalf = 16 * kRowBytes;             // a tile's keys, or its values
    static constexpr int kRing = kHalf >= 8192 ? 3 : kHalf >= 6144 ? 4 : kHalf >= 4096 ? (kBlocks == 3 ? 4 : 5) : kHalf > 2048 ? 6 : 8;
    // the warps' rings; once these are read, the warps' parts, each in its own ring, and the other blocks' parts that one joins
    static constexpr int smem = kWarps * kRing * kHalf > 65536 ? kWarps * kRing * kHalf : 65536;
    static_assert(kHeads * kRow * 4 <= kRing * kHalf, "");
    static constexpr bool joins(int unit_heads) {
        const int size = join_size(unit_heads), joined = (kMaxSms * kBlocks + size - 1) / size, room = smem / (kAttnThreads * 16 + unit_heads * 8);
        return size <= room && joined <= room;
    }
    static_assert(joins(kHeads) && joins(2 * kHeads) && joins(4 * kHeads), "a block joins all parts of a unit in two steps");
};

template <int D, int NT, bool E4M3>
__global__ void __launch_bounds__(kAttnThreads, (Shape<D, NT, E4M3>::kBlocks)) paged_attention_kernel(const AttnParams p) {
    using S = Shape<D, NT, E4M3>;
    constexpr int kHeads = S::kHeads, kElem = E4M3 ? 1 : 2, kRowBytes = S::kRowBytes, kHalf = S::kHalf, kRing = S::kRing;
    constexpr int kKeyLoads = D * kElem / 64;                // 16-byte loads a key row of K, a lane
    // weights are held 2^kUp times as large, against the running maximum less kUp: fp16's range then reaches from the largest down to 2e-9 of it
    // without loss.  A small weight counts where the large one's value is 0
    constexpr float kUp = E4M3 ? 15.f : 0.f;
    constexpr bool kWide = !E4M3 || D % 128 == 0;            // V in 16-byte loads, else in 8-byte ones
    using VLoad = typename std::conditional<kWide, uint4, uint2>::type;
    constexpr int kValLoads = D * kElem / (kWide ? 128 : 64);
    extern __shared__ __align__(128) float out_s[];           // rings; later [warp][head][kRow], each in its warp's ring
    __shared__ float top_s[kWarps][kHeads], sum_s[kWarps][kHeads];
    __shared__ long long line_s[kScanTokens + 1];
    __shared__ int2 seen_s[kScanTokens];                      // row, end
    __shared__ long long warp_s[kWarps];
    __shared__ int most_s[kWarps];                            // a token's greatest length on the line
    struct Vote {
        int ok, tokens, in4, in2, keys4, keys2;
    };
    __shared__ Vote vote_s[kWarps];
    __shared__ uint32_t last_s;
    // what only a unit's end needs, out of the registers while its keys go by
    struct Part {
        long long total, blocks;
        int of, unit, length, unit_shift;
        bool whole, begins_here;
    };
    __shared__ Part part_s;

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, j = lane & 3;
    pdl_wait();
    // warps: of tokens, then of sets of heads, then of keys
    int together = 1;                                        // consecutive tokens that share a block
    const int hw = 1 << p.head_shift;
    int why = 0;
    constexpr int kPart = kRing * kHalf / 4;                 // floats from one warp's part to the next one's
    const uint32_t ring = (uint32_t) __cvta_generic_to_shared(out_s) + warp * (kRing * kHalf);
    // Copies: instruction i of a half takes its bytes 512 i + 16 lane, the lines' 16-byte pieces permuted among themselves so that the reads
    // below meet every bank once: piece c of row r lies at c ^ 4 (r & 1) in K, at c ^ 2 (r / 2 & 3) in V.
    constexpr bool kSwizzle = kRowBytes % 128 == 0;
    auto place = [&](int i, bool v) {
        const int b = 512 * i + 16 * lane, r = b / kRowBytes;
        return (uint32_t) (b ^ (kSwizzle ? (v ? (r >> 1 & 3) << 5 : (r & 1) << 6) : 0));
    };
    // reads: K row g, pieces 4 i + j; V row 2 j, pieces 8 i + g (of 16 bytes, or of 8)
    const uint32_t k_even = g * kRowBytes + j * 16 + (kSwizzle ? (g & 1) * 64 : 0), k_odd = g * kRowBytes + j * 16 + (kSwizzle ? 64 - (g & 1) * 64 : 64);
    const uint32_t v_at = 2 * j * kRowBytes + (kWide ? (kSwizzle ? g ^ 2 * j : g) * 16 : ((kSwizzle ? (g >> 1) ^ 2 * j : g >> 1) * 16 + (g & 1) * 8));

    const long long* line = p.line;
    int most = 0;
    if (p.T <= kScanTokens) {
        constexpr int kEach = kScanTokens / kAttnThreads;
        Seen own[kEach];
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int t = tid * kEach + i;
            own[i].row = -1, own[i].begin = own[i].end = 0;
            if (t < p.T) {
                own[i] = seen_by(p, t, why);
                seen_s[t] = make_int2(own[i].row, own[i].end);
            }
        }
        // Windows of tokens of one request: where all fours of consecutive tokens, or all twos, are of one table row each and full but for a
        // quarter, a block may take them together, a token a warp: the keys then come from HBM once, not once a token.  It pays where L2 does
        // not hold the keys anyway and there are units enough that few are split, since a unit's parts then are as many times larger
        // (us, apart and together, bf16: 64 x 4 tokens of 2048 keys, 32 / 8 heads, 330, 187; 64 x 2 of 4096, 8 / 2, 93, 60; 16 x 4 of 4096,
        // 32 / 4, 58, 61; 16 x 4 of 1024 25, 29; 4 x 4 of 100000, 5 / 1, 150, 149)
        if (p.T > 1 && hw < kWarps) {
            static_assert(kEach == 4, "");
            bool fours = true, twos = true;
            int tokens = 0, in4 = 0, in2 = 0, keys4 = 0, keys2 = 0, row4 = -1;   // keys by 64, at most 2^28
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                const bool a = own[i].end > 0, b = own[i + 1].end > 0;
                twos = twos && !(a && b && own[i].row != own[i + 1].row);
                tokens += a + b, in2 += a || b;
                if (a) fours = fours && (row4 < 0 || row4 == own[i].row), row4 = own[i].row;
                if (b) fours = fours && (row4 < 0 || row4 == own[i + 1].row), row4 = own[i + 1].row;
                const int keys = min(max(own[i].end - own[i].begin, own[i + 1].end - own[i + 1].begin), 1 << 28) / 64;
                keys2 += keys, keys4 = max(keys4, keys);
            }
            in4 = row4 >= 0;
            fours = __all_sync(kFull, fours), twos = __all_sync(kFull, twos);
            tokens = __reduce_add_sync(kFull, tokens), in4 = __reduce_add_sync(kFull, in4), in2 = __reduce_add_sync(kFull, in2);
            keys4 = __reduce_add_sync(kFull, keys4), keys2 = __reduce_add_sync(kFull, keys2);
            if (lane == 0) vote_s[warp] = Vote{fours | twos << 1, tokens, in4, in2, keys4, keys2};
            __syncthreads();
            int ok = 3;
            long long bytes4 = 0, bytes2 = 0;
            tokens = in4 = in2 = 0;
            for (int w = 0; w < kWarps; ++w) {
                const Vote v = vote_s[w];
                ok &= v.ok, tokens += v.tokens, in4 += v.in4, in2 += v.in2, bytes4 += v.keys4, bytes2 += v.keys2;
            }
            const long long of64 = 128ll * kRowBytes * p.hk, many = 128ll << 20;
            if (hw == 1 && (ok & 1) && tokens >= 3 * in4 && bytes4 * of64 >= many && (long long) in4 * p.units >= 100) together = 4;
            else if ((ok & 2) && tokens == 2 * in2 && bytes2 * of64 >= many && (long long) in2 * p.units >= 100) together = 2;
        }
        long long mine = 0, n[kEach] = {0, 0, 0, 0};
        const int lines = kEach / together, chunk = kWarps / (hw * together) * 16;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const long long m = length_of(chunks_of(own[i], chunk));
            if (together == 1) n[i] = m;
            else if (together == 2) n[i / 2] = max(n[i / 2], m);
            else n[0] = max(n[0], m);
        }
#pragma unroll
        for (int i = 0; i < kEach; ++i) mine += n[i];
        long long incl = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const long long o = __shfl_up_sync(kFull, incl, d);
            if (lane >= d) incl += o;
        }
#pragma unroll
        for (int i = 0; i < kEach; ++i) most = max(most, (int) n[i]);
        most = __reduce_max_sync(kFull, most);
        if (lane == 0) most_s[warp] = most;
        if (lane == 31) warp_s[warp] = incl;
        __syncthreads();
        for (int w = 0; w < kWarps; ++w) most = max(most, most_s[w]);
        long long run = incl - mine;
        for (int w = 0; w < warp; ++w) run += warp_s[w];
        if (tid == 0) line_s[0] = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            if (i >= lines) continue;
            run += n[i];
            line_s[tid * lines + i + 1] = run;
        }
        __syncthreads();
        line = line_s;
        if (blockIdx.x) why = 0;
    }
    const int together_shift = together >> 1, unit_shift = p.head_shift + together_shift;   // 1, 2, 4: 0, 1, 2
    const int kw = kWarps >> unit_shift, head_group = warp >> (2 - unit_shift), key_warp = warp & (kw - 1);
    const int chunk = kw * 16, groups = (p.T + together - 1) >> together_shift;
    // rows of tokens that see nothing
    for (int t = blockIdx.x; t < p.T; t += gridDim.x) {
        const int of = t >> together_shift;
        if (line[of + 1] != line[of]) continue;
        for (int i = tid; i < p.hq * D; i += kAttnThreads) {
            const int64_t at = (int64_t) t * p.hq * D + i;
            if (p.out_kind == BSX_OUT_BF16) static_cast<uint16_t*>(p.out)[at] = 0;
            else static_cast<float*>(p.out)[at] = 0.f;
        }
        if (p.lse)
            for (int h = tid; h < p.hq; h += kAttnThreads) p.lse[(int64_t) t * p.hq + h] = p.sinks ? p.sinks[h] : -INFINITY;
    }

    const long long total = line[groups] * p.units;
    const long long blocks = runs_of(min((long long) gridDim.x, total), total, most);
    const long long first = blockIdx.x < blocks ? quotient(total * blockIdx.x, blocks) : 0, end = blockIdx.x < blocks ? quotient(total * (blockIdx.x + 1), blocks) : 0;
    int t = 0;
    if (first < end) {   // the tokens of place `first`
        int lo = 0, hi = groups;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (line[mid + 1] * p.units > first) hi = mid;
            else lo = mid + 1;
        }
        t = lo;
    }
    long long left = end - first;
    int length = 0, unit = 0, off = 0;   // of token t's units; the unit the run is in, and the place in it: kSetup places, then the chunks'
    const float cap = p.softcap * kLog2e, cap_inv = 1.f / p.softcap;   // used where softcap > 0
    if (left > 0) {
        length = (int) (line[t + 1] - line[t]);
        const long long of_token = first - line[t] * p.units;
        unit = (int) quotient(of_token, length);
        off = (int) (of_token - (long long) unit * length);
    }
    while (left > 0) {
        const int take = (int) min(left, (long long) (length - off)), c0 = max(off - kSetup, 0), c1 = off + take - kSetup;
        const int of = t, of_unit = unit, of_length = length;
        const bool off_first = off < kSetup;   // the unit's chunks begin after the run does
        left -= take;
        off = 0;
        if (++unit == p.units && left > 0) {
            unit = 0;
            do {
                ++t;
                length = (int) (line[t + 1] - line[t]);
            } while (length == 0);
        }
        if (c0 >= c1) continue;
        if (tid == 0) part_s = Part{total, blocks, of, of_unit, of_length, unit_shift, c0 == 0 && c1 == of_length - kSetup, off_first};
        // the warp's token and set of heads; past the last of them it has nothing to do
        const int token = (of << together_shift) + (head_group >> p.head_shift), set = (of_unit << p.head_shift) + (head_group & (hw - 1));
        Seen seen{-1, 0, 0};
        if (p.T > kScanTokens) {
            seen = seen_by(p, token, why);
        } else if (token < p.T) {
            const int2 x = seen_s[token];
            seen.row = x.x, seen.end = x.y, seen.begin = begin_of(p, x.y);
        }
        const bool works = set < p.sets && seen.end > 0;
        const int kh = !works ? 0 : p.group_sets == 1 ? set : set / p.group_sets, h0 = (set - kh * p.group_sets) * kHeads;   // first head within the group
        const int base = (seen.begin & ~15) + key_warp * 16;

        // Q, as B fragments
        uint32_t q[NT][D / 8];
        float factor[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int h = h0 + nt * 8 + g;
            const uint16_t* src = p.q + token * p.q_stride + (int64_t) (kh * p.group + h) * D;
            if (!E4M3) {
#pragma unroll
                for (int b = 0; b < D / 32; ++b) {
                    uint4 w = make_uint4(0, 0, 0, 0);
                    if (works && h < p.group) w = *reinterpret_cast<const uint4*>(src + b * 32 + j * 8);
                    q[nt][4 * b] = w.x, q[nt][4 * b + 1] = w.y, q[nt][4 * b + 2] = w.z, q[nt][4 * b + 3] = w.w;
                }
                factor[nt][0] = factor[nt][1] = p.softcap > 0.f ? p.scale : p.scale * kLog2e;
            } else {
                uint4 w[D / 64][2];
                float big = 0.f;
#pragma unroll
                for (int b = 0; b < D / 64; ++b)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        w[b][i] = make_uint4(0, 0, 0, 0);
                        if (works && h < p.group) w[b][i] = *reinterpret_cast<const uint4*>(src + b * 64 + j * 16 + i * 8);
                        const uint32_t u[4] = {w[b][i].x, w[b][i].y, w[b][i].z, w[b][i].w};
#pragma unroll
                        for (int x = 0; x < 4; ++x)
                            big = fmaxf(big, fmaxf(fabsf(__uint_as_float(u[x] << 16)), fabsf(__uint_as_float(u[x] & 0xffff0000u))));
                    }
                big = fmaxf(big, __shfl_xor_sync(kFull, big, 1));
                big = fmaxf(big, __shfl_xor_sync(kFull, big, 2));
                // big = m 2^e, 1 <= m < 2: the row times 2^-e (an infinite row stays as it is)
                const int e = big > 0.f && big < INFINITY ? min(max((int) (__float_as_uint(big) >> 23) - 127, -125), 125) : 0;
                const float down = __uint_as_float((uint32_t) (127 - e) << 23), up = __uint_as_float((uint32_t) (127 + e) << 23);
#pragma unroll
                for (int b = 0; b < D / 64; ++b)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint32_t u[4] = {w[b][i].x, w[b][i].y, w[b][i].z, w[b][i].w};
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const __half2 f = __floats2half2_rn(__uint_as_float(u[x] << 16) * down, __uint_as_float(u[x] & 0xffff0000u) * down);
                            q[nt][8 * b + 4 * i + x] = *reinterpret_cast<const uint32_t*>(&f);
                        }
                    }
                const float f = up * p.scale * p.k_scale[kh] * (p.softcap > 0.f ? 1.f : kLog2e);
                factor[nt][0] = __shfl_sync(kFull, f, 8 * j);
                factor[nt][1] = __shfl_sync(kFull, f, 8 * j + 4);
            }
        }

        float o[NT][D / 16][4], top[NT][2], sum[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            top[nt][0] = top[nt][1] = -FLT_MAX;
            sum[nt][0] = sum[nt][1] = 0.f;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
        }
        const int32_t* table = p.table + seen.row * p.table_stride;
        const int mask = (1 << p.page_shift) - 1;
        const char* k_lane = static_cast<const char*>(p.k) + ((int64_t) kh << p.page_shift) * kRowBytes + lane * 16;
        const char* v_lane = static_cast<const char*>(p.v) + ((int64_t) kh << p.page_shift) * kRowBytes + lane * 16;
        // a tile's two octets of keys: their pages (one unless pages hold 8); past every page where no key of the range lies
        auto page_at = [&](int key) { return key < seen.end && key + 8 > seen.begin ? (uint32_t) table[key >> p.page_shift] : ~0u; };
        auto pages_at = [&](int key, uint32_t& a, uint32_t& b) {
            a = page_at(key);
            b = p.page_shift == 3 || (key < seen.begin && key + 8 <= seen.begin) ? page_at(key + 8) : a;
        };
        // the octets of tile `key` that can be used (bits 0, 1), and bit 2 where all 16 keys count
        auto state_of = [&](int key, uint32_t a, uint32_t b) {
            if (a < p.n_pages && b < p.n_pages && key >= seen.begin && key + 16 <= seen.end) return 7;
            if ((a >= p.n_pages && key < seen.end && key + 8 > seen.begin) || (b >= p.n_pages && key + 8 < seen.end && key + 16 > seen.begin))
                why |= BSX_PAGED_BAD_PAGE;
            return (a < p.n_pages ? 1 : 0) | (b < p.n_pages ? 2 : 0);
        };
        // tile `key`'s keys or values to ring slot `slot`
        auto fetch = [&](const char* from, uint32_t page_bytes, bool v, int key, uint32_t a, uint32_t b, int state, int slot) {
            const uint32_t to = ring + slot * kHalf;
            const char* oct0 = from + (uint64_t) a * page_bytes + (uint32_t) (key & mask) * kRowBytes;
            const char* oct1 = oct0;
            if (p.page_shift == 3) oct1 = from + (uint64_t) b * page_bytes - kHalf / 2;
            if (state & 4) {
#pragma unroll
                for (int i = 0; i < kHalf / 512; ++i) copy16(to + place(i, v), (i < kHalf / 1024 ? oct0 : oct1) + 512 * i);
            } else {
                // octet 0 may lie before the range, with a page that is not looked at
                if (a != b) oct1 = from + (uint64_t) b * page_bytes + (uint32_t) (key + 8 & mask) * kRowBytes - kHalf / 2;
#pragma unroll
                for (int i = 0; i < kHalf / 512; ++i) {
                    const bool low = i < kHalf / 1024;
                    const int at = key + (512 * i + 16 * lane) / kRowBytes;
                    const bool ok = (state & (low ? 1 : 2)) && at < seen.end && at >= seen.begin;
                    copy16(to + place(i, v), ok ? (low ? oct0 : oct1) + 512 * i : from, ok);
                }
            }
        };
        // The ring takes halves in the order K, V, K, V ...: half x is consumed while x + 1 .. x + kRing - 1 are under way.  `far` is the tile
        // whose half is fetched next, its state that of both of its halves
        const int key_first = base + c0 * chunk, key_end = works ? min(base + c1 * chunk, seen.end) : key_first;
        int far = key_first, far_state = 0, put = 0, get = 0;
        uint32_t far_a = 0, far_b = 0, next_a = 0, next_b = 0;
        uint32_t states = 0;   // of the tiles fetched and not yet consumed, four bits each, the oldest lowest
        int under_way = 0;
        pages_at(far, next_a, next_b);
        auto fetch_k = [&]() {
            if (far < key_end) {
                far_a = next_a, far_b = next_b;
                far_state = state_of(far, far_a, far_b);
                if (far + chunk < key_end) pages_at(far + chunk, next_a, next_b);
                states |= (uint32_t) far_state << (4 * under_way);
                ++under_way;
                fetch(k_lane, p.k_page, false, far, far_a, far_b, far_state, put);
                put = put + 1 == kRing ? 0 : put + 1;
            }
            copies_end();
        };
        auto fetch_v = [&]() {
            if (far < key_end) {
                fetch(v_lane, p.v_page, true, far, far_a, far_b, far_state, put);
                put = put + 1 == kRing ? 0 : put + 1;
                far += chunk;
            }
            copies_end();
        };
#pragma unroll
        for (int i = 0; i < kRing - 1; ++i) {
            if (i & 1) fetch_v();
            else fetch_k();
        }
        for (int key0 = key_first; key0 < key_end; key0 += chunk) {
            copies_wait<kRing - 2>();
            __syncwarp();
            // the half before this one has been read: its slot is free
            if (kRing & 1) fetch_k();
            else fetch_v();
            const int state = states & 7;
            states >>= 4;
            --under_way;
            float s[NT][4];
            {
                const uint32_t from = ring + get * kHalf;
#pragma unroll
                for (int i = 0; i < kKeyLoads; ++i) {
                    uint4 ka, kb;
                    const uint32_t at = from + (i & 1 ? k_odd : k_even) + (i & ~1) * 64;
                    read_shared(ka, at);
                    read_shared(kb, at + 8 * kRowBytes);
                    const uint32_t a[4] = {ka.x, ka.y, ka.z, ka.w}, b[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float part[4];
                        if (!E4M3) {
                            mma16<false, false>(part, a[0], b[0], a[1], b[1], q[nt][4 * i], q[nt][4 * i + 1]);
                            mma16<false, true>(part, a[2], b[2], a[3], b[3], q[nt][4 * i + 2], q[nt][4 * i + 3]);
                        } else {
#pragma unroll
                            for (int y = 0; y < 4; ++y) {
                                uint32_t a0, a1, a2, a3;
                                halves_of_e4m3(a[y], a0, a2);
                                halves_of_e4m3(b[y], a1, a3);
                                if (y == 0) mma16<true, false>(part, a0, a1, a2, a3, q[nt][8 * i], q[nt][8 * i + 1]);
                                else mma16<true, true>(part, a0, a1, a2, a3, q[nt][8 * i + 2 * y], q[nt][8 * i + 2 * y + 1]);
                            }
                        }
#pragma unroll
                        for (int y = 0; y < 4; ++y) s[nt][y] = i ? s[nt][y] + part[y] : part[y];
                    }
                }
                get = get + 1 == kRing ? 0 : get + 1;
            }
            uint32_t hi[NT][2], lo[NT][2];
            float down[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int i = 0; i < 4; ++i) s[nt][i] *= factor[nt][i & 1];
                if (p.softcap > 0.f) {   // here the factor is without log2(e)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[nt][i] = cap * tanh_fast(s[nt][i] * cap_inv);
                }
                if (!(state & 4)) {
                    const int key = key0 + g;
                    const bool in0 = (state & 1) && key < seen.end && key >= seen.begin, in1 = (state & 2) && key + 8 < seen.end && key + 8 >= seen.begin;
                    s[nt][0] = in0 ? s[nt][0] : -INFINITY, s[nt][1] = in0 ? s[nt][1] : -INFINITY;
                    s[nt][2] = in1 ? s[nt][2] : -INFINITY, s[nt][3] = in1 ? s[nt][3] : -INFINITY;
                }
                down[nt][0] = down[nt][1] = 1.f;
                float m0 = fmaxf(s[nt][0], s[nt][2]), m1 = fmaxf(s[nt][1], s[nt][3]);
                if (__any_sync(kFull, m0 > top[nt][0] + kUp || m1 > top[nt][1] + kUp)) {
#pragma unroll
                    for (int m = 4; m < 32; m <<= 1) {
                        m0 = fmaxf(m0, __shfl_xor_sync(kFull, m0, m));
                        m1 = fmaxf(m1, __shfl_xor_sync(kFull, m1, m));
                    }
                    m0 = fmaxf(m0 - kUp, top[nt][0]), m1 = fmaxf(m1 - kUp, top[nt][1]);
                    down[nt][0] = exp2_fast(top[nt][0] - m0), down[nt][1] = exp2_fast(top[nt][1] - m1);
                    top[nt][0] = m0, top[nt][1] = m1;
                    sum[nt][0] *= down[nt][0], sum[nt][1] *= down[nt][1];
                }
                float w[4], r[4], none;
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = exp2_fast(s[nt][i] - top[nt][i & 1]);
                sum[nt][0] += w[0] + w[2], sum[nt][1] += w[1] + w[3];
                hi[nt][0] = movmatrix_trans(pack2<E4M3>(w[0], w[1], r[0], r[1]));
                hi[nt][1] = movmatrix_trans(pack2<E4M3>(w[2], w[3], r[2], r[3]));
                lo[nt][0] = movmatrix_trans(pack2<E4M3>(r[0], r[1], none, none));
                lo[nt][1] = movmatrix_trans(pack2<E4M3>(r[2], r[3], none, none));
            }
            copies_wait<kRing - 2>();
            __syncwarp();
            if (kRing & 1) fetch_v();
            else fetch_k();
            const uint32_t from = ring + get * kHalf + v_at;
            get = get + 1 == kRing ? 0 : get + 1;
            auto add = [&](int i, int nt, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
                float part[4];
                mma16<E4M3, false>(part, a0, a1, a2, a3, lo[nt][0], lo[nt][1]);
                mma16<E4M3, true>(part, a0, a1, a2, a3, hi[nt][0], hi[nt][1]);
#pragma unroll
                for (int x = 0; x < 4; ++x) o[nt][i][x] = fmaf(o[nt][i][x], down[nt][x & 1], part[x]);
            };
#pragma unroll
            for (int i = 0; i < kValLoads; ++i) {
                constexpr int kWords = kWide ? 4 : 2;
                VLoad vf[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) read_shared(vf[r], from + (8 * (r >> 1) + (r & 1)) * kRowBytes + i * (kWide ? 128 : 64));
                const uint32_t(&v0)[kWords] = reinterpret_cast<const uint32_t(&)[kWords]>(vf[0]);
                const uint32_t(&v1)[kWords] = reinterpret_cast<const uint32_t(&)[kWords]>(vf[1]);
                const uint32_t(&v2)[kWords] = reinterpret_cast<const uint32_t(&)[kWords]>(vf[2]);
                const uint32_t(&v3)[kWords] = reinterpret_cast<const uint32_t(&)[kWords]>(vf[3]);
#pragma unroll
                for (int x = 0; x < kWords; ++x) {
                    if (!E4M3) {
                        const uint32_t a0 = __byte_perm(v0[x], v1[x], 0x5410), a1 = __byte_perm(v0[x], v1[x], 0x7632);
                        const uint32_t a2 = __byte_perm(v2[x], v3[x], 0x5410), a3 = __byte_perm(v2[x], v3[x], 0x7632);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            add(i * kWords + x, nt, a0, a1, a2, a3);
                        }
                    } else {
#pragma unroll
                        for (int y = 0; y < 2; ++y) {
                            const uint32_t a = __byte_perm(v0[x], v1[x], y ? 0x7362 : 0x5140), b = __byte_perm(v2[x], v3[x], y ? 0x7362 : 0x5140);
                            uint32_t a0, a1, a2, a3;
                            halves_of_e4m3(a, a0, a1);
                            halves_of_e4m3(b, a2, a3);
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                add((i * kWords + x) * 2 + y, nt, a0, a1, a2, a3);
                            }
                        }
                    }
                }
            }
        }

        // the warps' parts meet in shared memory.  Row 2x, 2x + 1 of a load's rows lie side by side: four values of a head a store
        constexpr int kPer = kWide ? 16 / kElem : 8;   // values of D that a lane has of a V load
        __syncwarp();                                  // the ring has been read
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int m = 4; m < 32; m <<= 1) sum[nt][e] += __shfl_xor_sync(kFull, sum[nt][e], m);
                const int h = nt * 8 + 2 * j + e;
                if (g == 0) top_s[warp][h] = top[nt][e], sum_s[warp][h] = sum[nt][e];
                float* dst = out_s + warp * kPart + h * S::kRow;
#pragma unroll
                for (int i = 0; i < D / 16; i += 2) {
                    const int d = i * 2 / kPer * (8 * kPer) + g * kPer + i * 2 % kPer;
                    *reinterpret_cast<float4*>(dst + d) = make_float4(o[nt][i][e], o[nt][i][2 + e], o[nt][i + 1][e], o[nt][i + 1][2 + e]);
                }
            }
        __syncthreads();
        // A head's threads lie in one warp: 128 over the unit's heads, four values each at a time
        constexpr int kShareShift = NT == 1 ? 4 : 3;
        const Part part = part_s;
        const int unit_shift = part.unit_shift, unit_heads = kHeads << unit_shift, together_shift = unit_shift - p.head_shift, kw = kWarps >> unit_shift;
        const int share_shift = kShareShift - unit_shift, share = 1 << share_shift, h = tid >> share_shift, d0 = (tid & (share - 1)) * 4;
        const int h_warp = h / kHeads, h_token = (part.of << together_shift) + (h_warp >> p.head_shift), h_set = (part.unit << p.head_shift) + (h_warp & (hw - 1));
        const int h_kh = p.group_sets == 1 ? h_set : h_set / p.group_sets;
        const int in_group = (h_set - h_kh * p.group_sets) * kHeads + h % kHeads, head = h_kh * p.group + in_group;
        const bool mine = h_token < p.T && h_set < p.sets && in_group < p.group, whole = part.whole;
        // the factor of a head's values whose weights sum to l at maximum m; its logarithm written
        auto close = [&](float m, float l) {
            float f = E4M3 ? p.v_scale[h_kh] : 1.f;
            if (p.sinks) {
                const float sink = p.sinks[head] * kLog2e, both = fmaxf(m, sink);
                f *= exp2f(m - both);
                l = l * exp2f(m - both) + (sink == both ? 1.f : exp2f(sink - both));   // an infinite sink less itself is no number
                m = both;
            }
            if (d0 == 0 && p.lse) p.lse[(int64_t) h_token * p.hq + head] = l != 0.f ? (m + log2f(l)) * kLn2 : -INFINITY;
            return l != 0.f ? f / l : 0.f;
        };
        const int64_t out_at = ((int64_t) h_token * p.hq + head) * D;
        auto write = [&](int d, float4 v) {
            if (p.out_kind == BSX_OUT_BF16) {
                const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
                *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + out_at + d) =
                    make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
            } else {
                *reinterpret_cast<float4*>(static_cast<float*>(p.out) + out_at + d) = v;
            }
        };
        // Parts of a unit in the workspace, two slots a block, the second for a unit whose chunks begin inside its run.  A slot: out, then
        // maxima and sums, then those of joined parts
        const size_t slot = (size_t) unit_heads * (D + 4);
        const int own_ml = unit_heads * D, joined_ml = unit_heads * (D + 2);
        float* const left_at = p.parts + (2 * (size_t) blockIdx.x + (part.begins_here ? 1 : 0)) * slot;
        if (mine) {
            const int w0 = h / kHeads * kw, hh = h % kHeads;
            float f[kWarps], m = -FLT_MAX, l = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w)
                if (w < kw) m = fmaxf(m, top_s[w0 + w][hh]);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                f[w] = 0.f;
                if (w < kw) f[w] = exp2_fast(top_s[w0 + w][hh] - m), l = fmaf(f[w], sum_s[w0 + w][hh], l);
            }
            if (whole) {
                const float c = close(m, l);
#pragma unroll
                for (int w = 0; w < kWarps; ++w) f[w] *= c;
            } else if (d0 == 0) {
                __stcg(reinterpret_cast<float2*>(left_at + own_ml + 2 * h), make_float2(m, l));
            }
            for (int d = d0; d < D; d += 4 * share) {
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    if (w >= kw) continue;
                    const float4 x = *reinterpret_cast<const float4*>(out_s + (w0 + w) * kPart + hh * S::kRow + d);
                    v.x = fmaf(f[w], x.x, v.x), v.y = fmaf(f[w], x.y, v.y), v.z = fmaf(f[w], x.z, v.z), v.w = fmaf(f[w], x.w, v.w);
                }
                if (whole) write(d, v);
                else __stcg(reinterpret_cast<float4*>(left_at + h * D + d), v);
            }
        }
        if (!whole) {
            // the blocks that share the unit, in the order of their keys.  Up to join_size of them are joined by the last of these; the joined
            // parts of more, in the first one's slot, by the last of those
            const long long unit_first = line[part.of] * p.units + (long long) part.unit * part.length;
            const long long b0 = quotient((unit_first + kSetup + 1) * part.blocks - 1, part.total), b1 = quotient((unit_first + part.length) * part.blocks - 1, part.total);
            const int lead = quotient(part.total * b0, part.blocks) < unit_first + kSetup ? 1 : 0;   // only the first can have it in its second slot
            const int sharers = (int) (b1 - b0) + 1, size = join_size(unit_heads), group = (int) (blockIdx.x - b0) / size, joined = (sharers + size - 1) / size;
            auto slot_of = [&](int i) { return 2 * (b0 + i) + (i ? 0 : lead); };
            // parts i0, i0 + step, ... joined into `to`, or finished where there is none
            auto join = [&](int i0, int step, int count, int at_ml, float* to) {
                if (!mine) return;
                float2* const weight = reinterpret_cast<float2*>(out_s) + h * count;
                const float* const parts = p.parts + slot_of(i0) * slot;
                const size_t next = 2 * (size_t) step * slot;   // all but the first lie in their block's first slot
                const float* const rest = p.parts + 2 * (b0 + i0) * slot;
                auto part = [&](int y) { return y ? rest + y * next : parts; };
                float m = -FLT_MAX, l = 0.f;
                // a thread's values of the parts, columns 4 share apart, as many columns at a time as the rings' memory holds
                const int columns = (D / 4) >> share_shift, room = (S::smem - unit_heads * count * 8) / (kAttnThreads * 16 * count);   // at least 1, see Shape
                const int at_once = room < columns ? room : columns;
                const uint32_t data = (uint32_t) __cvta_generic_to_shared(out_s) + unit_heads * count * 8 + tid * 16;
                auto ask = [&](int x0) {
                    for (int x = 0; x < at_once && x0 + x < columns; ++x)
#pragma unroll 5
                        for (int y = 0; y < count; ++y)
                            copy16(data + (x * count + y) * (kAttnThreads * 16), part(y) + h * D + d0 + (x0 + x) * 4 * share);
                    copies_end();
                };
                ask(0);
                for (int y = d0 / 4; y < count; y += share) {
                    weight[y] = __ldcg(reinterpret_cast<const float2*>(part(y) + at_ml + 2 * h));
                    m = fmaxf(m, weight[y].x);
                }
                const uint32_t lanes = (share == 32 ? kFull : ((1u << share) - 1)) << (lane & ~(share - 1));
                for (int x = share / 2; x; x >>= 1) m = fmaxf(m, __shfl_xor_sync(lanes, m, x));
                for (int y = d0 / 4; y < count; y += share) {
                    const float f = exp2_fast(weight[y].x - m);
                    l = fmaf(f, weight[y].y, l);
                    weight[y].x = f;
                }
                for (int x = share / 2; x; x >>= 1) l += __shfl_xor_sync(lanes, l, x);
                __syncwarp(lanes);
                float c = 1.f;
                if (!to) c = close(m, l);
                else if (d0 == 0) __stcg(reinterpret_cast<float2*>(to + joined_ml + 2 * h), make_float2(m, l));   // others may still read the part's own
                for (int x0 = 0; x0 < columns; x0 += at_once) {
                    if (x0) ask(x0);
                    copies_wait<0>();
                    for (int x = 0; x < at_once && x0 + x < columns; ++x) {
                        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 5
                        for (int y = 0; y < count; ++y) {
                            uint4 u;
                            read_shared(u, data + (x * count + y) * (kAttnThreads * 16));
                            const float f = weight[y].x;
                            v.x = fmaf(f, __uint_as_float(u.x), v.x), v.y = fmaf(f, __uint_as_float(u.y), v.y);
                            v.z = fmaf(f, __uint_as_float(u.z), v.z), v.w = fmaf(f, __uint_as_float(u.w), v.w);
                        }
                        v.x *= c, v.y *= c, v.z *= c, v.w *= c;
                        const int d = d0 + (x0 + x) * 4 * share;
                        if (!to) write(d, v);
                        else __stcg(reinterpret_cast<float4*>(to + h * D + d), v);
                    }
                }
            };
            // whether this block is the last of `count`; the counter is back at 0 with it.  The block's stores are ordered before the count, and
            // what follows after the others' stores, by the barriers and the count's own release and acquire
            auto last_of = [&](uint32_t* counter, int count) {
                __syncthreads();
                if (tid == 0) last_s = count_up(counter, (uint32_t) count - 1) == (uint32_t) count - 1;
                __syncthreads();
                return last_s != 0;
            };
            const bool again = joined > 1;
            const int count = min(size, sharers - group * size);
            if (last_of(p.counter + slot_of(group * size), count)) {
                join(group * size, 1, count, own_ml, again ? p.parts + slot_of(group * size) * slot : nullptr);
                if (again && last_of(p.counter + 2 * gridDim.x + b0, joined)) join(0, size, joined, joined_ml, nullptr);
            }
        }
        __syncthreads();   // the parts have been read: the rings are free
    }
    if (why && p.status) atomicOr(p.status, why);
}

// the running sums of the tokens' chunks, for calls of many tokens
__global__ void __launch_bounds__(1024) attention_line_kernel(const AttnParams p, int chunk) {
    __shared__ long long warp_s[32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    long long before = 0;
    int why = 0;
    if (tid == 0) p.line[0] = 0;
    for (int t0 = 0; t0 < p.T; t0 += 1024) {
        const int t = t0 + tid;
        long long v = t < p.T ? length_of(chunks_of(seen_by(p, t, why), chunk)) : 0;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const long long o = __shfl_up_sync(kFull, v, d);
            if (lane >= d) v += o;
        }
        __syncthreads();
        if (lane == 31) warp_s[warp] = v;
        __syncthreads();
        long long all = 0;
        for (int w = 0; w < 32; ++w) {
            if (w < warp) v += warp_s[w];
            all += warp_s[w];
        }
        if (t < p.T) p.line[t + 1] = before + v;
        before += all;
    }
    if (why && p.status) atomicOr(p.status, why);
}

size_t up256(size_t n) { return (n + 255) & ~(size_t) 255; }

// how a call's heads are laid on warps
struct Plan {
    int nt, sets, group_sets, head_warps, blocks, slot;   // blocks: an SM; slot: floats
};
Plan plan_of(const bsx_kv_cache* c, int n_q_heads, int64_t T) {
    const int group = n_q_heads / c->n_kv_heads, D = c->head_dim;
    Plan r{};
    r.nt = group > 8 && D <= 128 ? 2 : 1;   // 16 heads of 192 or 256 values do not fit a warp's registers
    const int per = 8 * r.nt;
    r.blocks = blocks_an_sm(D, r.nt);
    r.group_sets = (group + per - 1) / per;
    r.sets = c->n_kv_heads * r.group_sets;
    // A kv head's sets stay together, they read the same keys.  Where there are eight sets a block and more, a block's warps have other sets
    // instead of other keys: a unit's fixed work is then one warp's for its own keys, not four warps' for a quarter each
    // (us, four warps on the keys or on the sets: 1024 requests of 64 keys, 64 / 8 heads, e4m3 91, 60; 32 / 8, bf16 84, 69; 512 of 128, e4m3
    // 60, 49; 1000 of 700, e4m3 299, 264, bf16 451, 462; with fewer the ends of the runs cost more: 64 ragged requests, bf16 62, 75).
    // The host knows T, the call's places, not how many of them hold a token: in a long window that is nearly empty the rule has the other
    // side's cost (one token of 1000 keys, 32 / 8, bf16, in 256 places 12, in 512 25)
    r.head_warps = r.group_sets == 1 ? 1 : r.group_sets == 2 ? 2 : 4;
    if (T * r.sets >= 8ll * kMaxSms * r.blocks)
        while (r.head_warps < kWarps && r.head_warps < r.sets) r.head_warps *= 2;
    r.slot = per * kWarps * (D + 4);   // tokens that share a block share its slots too
    return r;
}
// the same for every call, so that calls of different shapes find each other's counters at 0
constexpr size_t kCounterBytes = 5376;
static_assert(kCounterBytes >= (size_t) 3 * kMaxSms * 3 * 4 && kCounterBytes % 256 == 0, "");
size_t parts_bytes(const Plan& r) { return up256((size_t) 2 * kMaxSms * r.blocks * r.slot * 4); }

template <int D, int NT, bool E4M3>
int32_t launch_attention(const AttnParams& p, int64_t most_chunks, cudaStream_t st) {
    using S = Shape<D, NT, E4M3>;
    static std::atomic<bool> configured[64];   // per device; threads of different devices call concurrently
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return (int32_t) cudaErrorInvalidDevice;
    if (!configured[dev].load(std::memory_order_acquire)) {
        const cudaError_t e = cudaFuncSetAttribute(paged_attention_kernel<D, NT, E4M3>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::smem);
        if (e != cudaSuccess) return (int32_t) e;
        configured[dev].store(true, std::memory_order_release);
    }
    if (p.T > kScanTokens) attention_line_kernel<<<1, 1024, 0, st>>>(p, (kWarps >> p.head_shift) * 16);
    const int64_t sms = sm_count() < kMaxSms ? sm_count() : kMaxSms;
    const int64_t runs = sms * S::kBlocks;
    const int64_t grid = most_chunks < runs ? (most_chunks > 0 ? most_chunks : 1) : runs;
    launch_early(paged_attention_kernel<D, NT, E4M3>, dim3((unsigned) grid), dim3(kAttnThreads), S::smem, st, p);
    return launch_status();
}

}  // namespace
}  // namespace bsx

using namespace bsx;

extern "C" size_t bsx_paged_attention_workspace_bytes(const bsx_kv_cache* cache, int32_t n_q_heads, int32_t T) {
    if (cache_status(cache) || n_q_heads <= 0 || n_q_heads % cache->n_kv_heads || T < 0) return 0;
    const Plan r = plan_of(cache, n_q_heads, T);
    return kCounterBytes + parts_bytes(r) + (T > kScanTokens ? up256(((size_t) T + 1) * 8) : 0);
}

extern "C" int32_t bsx_paged_attention(const bsx_kv_cache* cache, const void* q, int64_t q_stride, int32_t n_q_heads, int32_t T,
                                       const int32_t* block_table, int64_t table_stride, int32_t n_rows, int32_t max_pages, const int32_t* pos,
                                       const int32_t* row, float scale, int32_t window, float softcap, const float* sinks, void* out, int32_t out_kind,
                                       float* lse, void* workspace, int32_t* status, void* stream) {
    if (!stream) return BSX_E_STREAM;
    const int32_t bad = cache_status(cache);
    if (bad) return bad;
    if (out_kind != BSX_OUT_F32 && out_kind != BSX_OUT_BF16) return BSX_E_TYPE;
    if (n_q_heads <= 0 || n_q_heads % cache->n_kv_heads || T < 0 || n_rows < 0 || max_pages < 0 || table_stride < max_pages || q_stride % 8 ||
        window < 0 || !(softcap >= 0.f && softcap < INFINITY))
        return BSX_E_GEOMETRY;
    if (n_q_heads > 1024 || T > BSX_PAGED_MAX_TOKENS || (int64_t) max_pages * cache->page_size > BSX_PAGED_MAX_KEYS) return BSX_E_LIMIT;
    const int64_t elem = cache->kind == BSX_KV_BF16 ? 2 : 1, k_bytes = cache->k_page_stride * elem, v_bytes = cache->v_page_stride * elem;
    if (cache->k_page_stride > 0x7fffffff || cache->v_page_stride > 0x7fffffff) return BSX_E_LIMIT;
    if (T == 0) return BSX_OK;
    if (!aligned(q, 16) || !aligned(out, 16) || !aligned(workspace, 256) || !pos || (n_rows && max_pages && !block_table) || (lse && !aligned(lse, 4)) ||
        (sinks && !aligned(sinks, 4)))
        return BSX_E_POINTER;
    const Plan r = plan_of(cache, n_q_heads, T);
    AttnParams p{};
    p.q = static_cast<const uint16_t*>(q), p.k = cache->k, p.v = cache->v;
    p.k_scale = cache->k_scale, p.v_scale = cache->v_scale, p.sinks = sinks;
    p.table = block_table, p.pos = pos, p.row = row, p.out = out, p.lse = lse, p.status = status;
    p.q_stride = q_stride, p.table_stride = table_stride, p.k_page = (uint32_t) k_bytes, p.v_page = (uint32_t) v_bytes;
    p.n_pages = (uint32_t) cache->n_pages, p.scale = scale, p.softcap = softcap;
    p.hq = n_q_heads, p.hk = cache->n_kv_heads, p.group = n_q_heads / cache->n_kv_heads, p.T = T, p.n_rows = n_rows, p.max_pages = max_pages;
    p.page_shift = log2_of(cache->page_size), p.window = window, p.out_kind = out_kind;
    p.head_shift = r.head_warps >> 1, p.sets = r.sets, p.group_sets = r.group_sets;
    p.units = (r.sets + r.head_warps - 1) / r.head_warps;
    char* w = static_cast<char*>(workspace);
    p.counter = reinterpret_cast<uint32_t*>(w);
    p.parts = reinterpret_cast<float*>(w + kCounterBytes);
    p.line = reinterpret_cast<long long*>(w + kCounterBytes + parts_bytes(r));
    // no more blocks than there can be places on the line
    const int chunk = kWarps / r.head_warps * 16;
    int64_t keys = (int64_t) max_pages * cache->page_size;
    if (window > 0 && window + 15ll < keys) keys = window + 15ll;
    const int64_t most = keys ? (int64_t) T * p.units * ((keys + chunk - 1) / chunk + kSetup) : 0;
    if (most >= 1ll << 52) return BSX_E_LIMIT;   // times the blocks it still fits 64 bits
    const bool e4m3 = cache->kind == BSX_KV_E4M3;
    cudaStream_t st = (cudaStream_t) stream;
    switch (cache->head_dim) {
        case 64:
            if (r.nt == 2) return e4m3 ? launch_attention<64, 2, true>(p, most, st) : launch_attention<64, 2, false>(p, most, st);
            return e4m3 ? launch_attention<64, 1, true>(p, most, st) : launch_attention<64, 1, false>(p, most, st);
        case 128:
            if (r.nt == 2) return e4m3 ? launch_attention<128, 2, true>(p, most, st) : launch_attention<128, 2, false>(p, most, st);
            return e4m3 ? launch_attention<128, 1, true>(p, most, st) : launch_attention<128, 1, false>(p, most, st);
        case 192: return e4m3 ? launch_attention<192, 1, true>(p, most, st) : launch_attention<192, 1, false>(p, most, st);
        default: return e4m3 ? launch_attention<256, 1, true>(p, most, st) : launch_attention<256, 1, false>(p, most, st);
    }
}
