// Decode attention over the 8-bit paged cache (kv_quant.cuh): one query token per request in bfloat16, the query heads of a kv
// head as one or two column tiles of tensor-core products, all requests' pages dealt out evenly to one wave of blocks, what several blocks
// made of one head's sums added up by a second kernel.
//
//   s_k = scale q.K_k with K_k = c_k 2^e_k,  o = sum_k p_k V_k / sum_k p_k,  p_k = 2^(s_k log2 e - m),  V_k = d_k 2^f_k
//
// Codes become halves (exactly) in registers and go straight into m16n8k16 products with f32 sums; nothing is scaled before a
// product. The exponent of K multiplies the score; the exponent of V joins the softmax's: with t_k = s_k log2 e + f_k and a reference m 7 below the
// running maximum of t_k, the weight w_k = 2^(t_k - m) is what V's codes are multiplied by, at most 2^15 and therefore a half with 11 bits
// where they count (down to 2^-21 of the largest; the smallest of a half is 2^-31 of it), and the denominator adds w_k 2^-f_k in 32 bits (2^-93 to 2^107 a key). Where exponents
// of V lie so far apart that w_k may be 0 although p_k counts, the denominator's 2^(t_k - f_k - m) is an exponential of its own. A row of zeros counts as one of the lowest
// exponent. Else one exponential a score, as without a quantised cache. q goes to halves times a
// power of two of its row's (its largest magnitude then lies in 2^8 .. 2^9, so that a score times the largest power of two of K, 2^100, stays within 32 bits): what a half
// cannot hold of it is below 2^-33 of that.
//
//   Products: S^T = K.Q^T and O^T = V^T.P^T, keys and V's columns as the 16 rows of a tile, heads as its 8 columns (NT tiles: one up to eight heads a kv head, two
//   beyond): with the heads as rows, half of every product, softmax and register would belong to rows that are not there where a kv head has eight heads or fewer.
//   S^T: a product step's 16 columns of K are four codes of each lane of a group of four, so a lane's 16-byte piece of a key row feeds four steps.
//   O^T: lane (g, q) of a warp takes columns g head_dim/8 .. of keys 2q, 2q + 1, 8 + 2q, 9 + 2q; pairs of keys are joined byte by byte, and tile t holds columns 2t and
//   2t + 1 of every lane's columns. P goes from the scores' places to the operand's by a transposing move of 8 x 8 halves.
//
//   Work: the pages that request e sees, once for each of its units (a kv head, and of its query heads up to 8 NT), one behind the other over requests and units. Block b
//   takes pages b S .. (b + 1) S of that row, S = all / blocks: requests of any lengths fill the blocks alike. A stretch of one unit is computed by the block's four warps
//   (warp w takes pages w, w + 4, ... of it; a page's record of a kv head is one untiled bulk copy into the warp's own ring) and merged
//   in shared memory. A unit that lies in one block is final there, else its parts go to scratch. Short requests: a block a unit, all of them final
//   (per_unit 1). In between, where one wave of blocks holds two to eight blocks a unit that are not much longer than dealt out: a cluster of them (per_unit), whose blocks read each other's parts
//   from shared memory: no scratch, no second kernel (eight requests of 1,024 tokens, 32 heads on 8 of 128, 10.0 -> 8.4 us).
//   (Parts added up by the block that finishes last, with fences and counts, took 8 us more than blocks that are final; the second kernel takes 2 to 3.)
//
// Token t (= entry t) sits at position kvlen - 1 and sees positions max(0, kvlen - window) .. kvlen - 1 (window < 0: runs of -window; 0: all). No
// key to see: zeros. A block-table entry below 0 is never followed, its keys count as masked. A masked key's score is replaced and its codes of V cleared, so
// what a page holds behind a request's end does not matter.
#include <cfloat>

#include "kv_quant.cuh"

#ifndef HEAD_DIM
#error "compile with -DHEAD_DIM=64, 128 or 256"
#endif
static_assert(HEAD_DIM == 64 || HEAD_DIM == 128 || HEAD_DIM == 256, "the 8-bit decode kernel takes head_dim 64, 128 or 256");

constexpr int DQ_HD = HEAD_DIM;
constexpr int DQ_REC = kvq_record(HEAD_DIM);
constexpr int DQ_STAGES = 2;                      // records of a warp's ring: three gain nothing (105, 111 us when tried, 64 requests of up to 8,192 tokens, 32 heads on 8 of 128)
constexpr int DQ_CH = HEAD_DIM / 16;               // pieces of 16 columns of a head
constexpr int DQ_KG = HEAD_DIM / 64;              // groups of four product steps of Q.K^T
constexpr int DQ_MT = HEAD_DIM / 16;              // tiles of 16 columns of V
constexpr int DQ_VB = HEAD_DIM / 8 < 16 ? HEAD_DIM / 8 : 16;      // columns a lane takes of a key row at a time
constexpr int DQ_NVB = HEAD_DIM / 8 / DQ_VB;      // ... and how often
constexpr int DQ_WARPS = 4;
// Pages of a block at least. Four and eight, us: eight requests of 2,048 tokens, 32 heads on 2 of 128, 11.3 / 10.4 (fewer parts to add up); one of 512 8.0 / 8.2, of 8,192 9.9 / 9.2.
constexpr int DQ_LEAST = 8;
constexpr int DQ_OS = HEAD_DIM + 4;
constexpr int DQ_CLUSTER = 8;                    // blocks of a cluster at most
// Shared memory of a block: the warps' rings, over them the merge; behind, the rings' barriers and the stretch's queries.
__host__ __device__ constexpr int dq_bars(int rows) {
    const int merge = DQ_WARPS * rows * (DQ_OS + 2) * 4 + rows * 8, pipe = DQ_WARPS * DQ_STAGES * DQ_REC;
    return ((pipe > merge ? pipe : merge) + 15) / 16 * 16;
}
__host__ __device__ constexpr int dq_q(int rows) { return dq_bars(rows) + (DQ_WARPS * DQ_STAGES * 8 + 15) / 16 * 16; }          // q's halves and the heads' factors
__host__ __device__ constexpr int dq_smem(int rows) { return dq_q(rows) + rows * DQ_HD * 2 + rows * 4; }
// Blocks an SM that the registers are to allow. (Heads of 128, three / four, us: 64 requests of up to 8,192 tokens, 32 heads on 8, e4m3, 107.6 / 105.9; 32 of 4,096, 32 on 2, e4m3, 21.5 / 20.2; one of
// 131,072 in e4m3 20.9 / 22.5, in whole numbers, whose codes take more registers to convert, 22.7 / 24.7. With four, the form for e4m3 with two column tiles spills 32 bytes a thread, heads of 256 up to 20;
// five spill more: 29 to 30 us for the last two.)
constexpr int dq_per_sm(int kind, int nt) { return HEAD_DIM == 64 ? (nt == 1 ? 5 : 4) : HEAD_DIM == 128 ? (nt == 2 && kind == KVQ_INT8 ? 3 : 4) : (nt == 1 ? 3 : 2); }
constexpr unsigned DQ_SPIN = 1u << 24;
constexpr float DQ_RAISE = 8.f;                   // the reference follows the maximum only when a page's is more than this above it (log2 units)
constexpr float DQ_UP = 7.f;                      // ... and lies this far below it: weights up to 2^15 (a half holds 65,504), so that small ones keep their bits down to 2^-21, and some down to 2^-31, of the largest
// Bytes of V's exponents that are in order: 2^-80 .. 2^-1 (rows up to 224 in e4m3, 63 as whole numbers). Among these a weight that is flushed to 0, below 2^-126, has a score 2^53 below the best
// one: no share of the denominator.
// Rows beyond (32 requests of 4,096, 32 heads on 2 of 128, e4m3, us: 18.6 in order, 24.1 where V is in the thousands; 64 of 4,500, 32 on 8, 99.7 / 104) and of zeros (25.2 / 109 with one on
// each page) take the long way.
constexpr unsigned DQ_V_LOW = 47, DQ_V_SPAN = 80;

__device__ __forceinline__ void dq_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void dq_mma_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {       // sums from zero
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
// Four codes of a word as two pairs of halves. e4m3: bytes 0 and 1, then 2 and 3, by the conversion instruction (shifts and masks instead, which run on another
// unit, were slower for K, for V and for both: 112, 112 and 123 us where this takes 108, 64 requests of up to 8,192 tokens, 32 heads on 8 of 128). Whole numbers: bytes 0 and 2, then 1 and 3; 1024 + 128 +
// code as a half is its bits and a constant's, one subtraction leaves the code.
template <int KIND>
__device__ __forceinline__ void dq_halves(uint32_t w, uint32_t& a, uint32_t& b) {
    if constexpr (KIND == KVQ_E4M3) {
        a = kvq_low<KIND>(w), b = kvq_high<KIND>(w);
    } else {
        asm("sub.rn.f16x2 %0, %1, %2;\n" : "=r"(a) : "r"((w & 0x00ff00ffu) ^ 0x64806480u), "r"(0x64806480u));
        asm("sub.rn.f16x2 %0, %1, %2;\n" : "=r"(b) : "r"((w >> 8 & 0x00ff00ffu) ^ 0x64806480u), "r"(0x64806480u));
    }
}
__device__ __forceinline__ bool dq_wait(uint32_t bar, uint32_t parity) {
    for (unsigned spin = 0; spin < DQ_SPIN; ++spin) {
        uint32_t done;
        asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n"
                     : "=r"(done) : "r"(bar), "r"(parity) : "memory");
        if (done) return true;
    }
    return false;
}
__device__ __forceinline__ float dq_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float dq_ex2_small(float x) {              // ... down to 2^-149
    const float root = dq_ex2(0.5f * x);
    return root * root;
}
// The root of the factor that brings sums from the reference m to M >= m (m = -infinity: there are none). A denominator may be near 2^108 where the factor is below 2^-126: it is
// multiplied by the root twice.
__device__ __forceinline__ float dq_root(float m, float M) { return m == -INFINITY ? 0.f : dq_ex2(0.5f * (m - M)); }
__device__ __forceinline__ uint32_t dq_pack_half(float lo, float hi) {
    uint32_t h;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;\n" : "=r"(h) : "f"(hi), "f"(lo));
    return h;
}
__device__ __forceinline__ uint32_t dq_transpose(uint32_t x) {       // of 8 x 8 halves: lane (g, q) has row g, columns 2q and 2q + 1
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t dq_pack_bf16(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
}

// Pages that a token at the end of kvlen tokens sees, and the first of them.
__device__ __forceinline__ int dq_pages(int kvlen, int window, int* first) {
    *first = il_mask_lo(kvlen - 1, window) / KVQ_PAGE;
    return kvlen > 0 ? (kvlen - 1) / KVQ_PAGE - *first + 1 : 0;
}
// How the pages of all requests are dealt out: pages of all units, pages of a block, and the request that page block * share belongs to, with how many pages lie in front of
// that request's. Every warp makes it for itself.
struct DqDeal {
    int all, share, e, before;
};
__device__ __forceinline__ DqDeal dq_deal(const int* entry_kvlen, int n_decode, int window, int units, int n_blocks, int block, int lane) {
    DqDeal d;
    int first, n0 = 0;
    d.all = 0;
    for (int e0 = 0; e0 < n_decode; e0 += 32) {
        const int n = e0 + lane < n_decode ? dq_pages(entry_kvlen[e0 + lane], window, &first) : 0;
        d.all += __reduce_add_sync(0xffffffffu, n);
        if (e0 == 0) n0 = n;
    }
    d.all *= units;
    d.share = max(DQ_LEAST, (int)(((unsigned)d.all + n_blocks - 1) / (unsigned)n_blocks));
    d.e = 0, d.before = 0;
    const long long from = (long long)block * d.share;
    if (from >= d.all) return d;
    int seen = 0;
    for (int e0 = 0; e0 < n_decode; e0 += 32) {
        const int n = e0 == 0 ? n0 : e0 + lane < n_decode ? dq_pages(entry_kvlen[e0 + lane], window, &first) : 0;
        int sum = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int s = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += s;
        }
        const unsigned past = __ballot_sync(0xffffffffu, seen + sum * units > (int)from);
        if (past) {
            const int l0 = __ffs(past) - 1;
            d.e = e0 + l0, d.before = seen + __shfl_sync(0xffffffffu, sum - n, l0) * units;
            break;
        }
        seen += __shfl_sync(0xffffffffu, sum, 31) * units;
    }
    return d;
}
// Of block `rank` of the cluster.
__device__ __forceinline__ float2 dq_peer2(uint32_t addr, int rank) {
    float2 v;
    asm volatile("{\n.reg .b32 at;\nmapa.shared::cluster.u32 at, %2, %3;\nld.shared::cluster.v2.f32 {%0,%1}, [at];\n}\n" : "=f"(v.x), "=f"(v.y) : "r"(addr), "r"(rank) : "memory");
    return v;
}
__device__ __forceinline__ float4 dq_peer4(uint32_t addr, int rank) {
    float4 v;
    asm volatile("{\n.reg .b32 at;\nmapa.shared::cluster.u32 at, %4, %5;\nld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [at];\n}\n"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr), "r"(rank) : "memory");
    return v;
}
// Where a unit's parts lie: its first block's second place, the others' first (a block holds at most the end of one unit and the start of another).
__device__ __forceinline__ int dq_place(int b0, int i) { return i == 0 ? 2 * b0 + 1 : 2 * (b0 + i); }

// A row's sums, four columns of it: final to `out`, else as a part.
__device__ __forceinline__ void dq_write(const float4& acc, float M, float L, __nv_bfloat16* out, float* o_part, float* ml_part, int r, int d) {
    if (out) {
        const float inv = L == 0.f ? 0.f : 1.f / L;           // (no key seen: zeros)
        *reinterpret_cast<uint2*>(out + (size_t)r * DQ_HD + d) = make_uint2(dq_pack_bf16(acc.x * inv, acc.y * inv), dq_pack_bf16(acc.z * inv, acc.w * inv));
    } else {
        *reinterpret_cast<float4*>(o_part + r * DQ_HD + d) = acc;
        if (d == 0) *reinterpret_cast<float2*>(ml_part + 2 * r) = make_float2(M, L);
    }
}
// (q and the newest token's slot of the cache, without `early` also lengths and tables, and in the second kernel the parts, may be written by the kernel before and are then read after a wait:
// they are not declared __restrict__, whose loads may be moved above it.)
template <int KIND, int NT>
__global__ void __launch_bounds__(DQ_WARPS * 32, dq_per_sm(KIND, NT)) attn_decode_quant_kernel(
    const __nv_bfloat16* q, long long q_stride, const unsigned char* cache, const int* block_table, int bt_stride,
    const int* entry_kvlen, int n_decode, int nh, int nkv, int G, int row_tiles, float scale_log2, int window, int per_unit, float* o_part, float* ml_part,
    __nv_bfloat16* out, int* status, int early) {
    if (!early) il_pdl_wait();
    extern __shared__ __align__(128) unsigned char smem[];
    constexpr int ROWS = 8 * NT, BARS = dq_bars(ROWS);
    const int units = nkv * row_tiles, n_blocks = gridDim.x;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, lg = lane >> 2, lq = lane & 3;

    // early: the caller vouches that lengths, block tables and the pages of earlier tokens do not come from the kernel in front (which writes q and
    // the newest token's slot, in the last page). What depends only on them is then done before waiting for it.
    int from, to, e, before;
    if (per_unit) {                               // one unit, or this block's share of it
        int first;
        const int u = blockIdx.x / per_unit, rank = blockIdx.x - u * per_unit;
        e = u / units, before = 0;
        const int n = dq_pages(entry_kvlen[e], window, &first);
        from = (u - e * units) * n + n * rank / per_unit, to = (u - e * units) * n + n * (rank + 1) / per_unit;
    } else {
        const DqDeal d = dq_deal(entry_kvlen, n_decode, window, units, n_blocks, blockIdx.x, lane);
        e = d.e, before = d.before;
        from = min((long long)blockIdx.x * d.share, (long long)d.all), to = min((long long)from + d.share, (long long)d.all);
    }

    if (per_unit > 1 && from >= to && threadIdx.x < ROWS) reinterpret_cast<float2*>(smem)[DQ_WARPS * ROWS + threadIdx.x] = make_float2(-INFINITY, 0.f);      // (no pages: no part)
    const uint32_t pipe = (uint32_t)__cvta_generic_to_shared(smem) + warp * DQ_STAGES * DQ_REC;
    const uint32_t bars = (uint32_t)__cvta_generic_to_shared(smem) + BARS + warp * DQ_STAGES * 8;
    uint2* q_sm = reinterpret_cast<uint2*>(smem + dq_q(ROWS));             // [product step][lane][NT]
    float* q_scale = reinterpret_cast<float*>(smem + dq_q(ROWS) + ROWS * DQ_HD * 2);
    const size_t page_bytes = (size_t)nkv * DQ_REC;
    if (lane == 0) {
        for (int s = 0; s < DQ_STAGES; ++s) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;\n" ::"r"(bars + s * 8));
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    __syncwarp();
    int done = 0;                                 // records this warp has been through: the ring's place and parity
    bool waited = !early, dead = false;
    for (int at = from, unit = 0; at < to;) {
        // ---- one stretch: pages p0 .. p1 of unit (e, head, rt), which starts at page `start` of the row
        int first_page, kvlen = entry_kvlen[e], n_pages = dq_pages(kvlen, window, &first_page);
        while (at >= before + n_pages * units) {
            before += n_pages * units;
            kvlen = entry_kvlen[++e], n_pages = dq_pages(kvlen, window, &first_page);
        }
        unit = at == from ? (at - before) / n_pages : at == before ? 0 : unit + 1;
        const int head = row_tiles == 1 ? unit : unit / row_tiles, rt = unit - head * row_tiles;
        const int start = before + unit * n_pages, end = min(start + n_pages, to);
        const int p0 = first_page + at - start, p1 = first_page + end - start, last_page = first_page + n_pages - 1;
        at = end;
        const int lo = il_mask_lo(kvlen - 1, window), head0 = head * G + rt * ROWS, rows_valid = min(ROWS, G - rt * ROWS);
        const int* bt = block_table + (size_t)e * bt_stride;
        const unsigned char* recs = cache + (size_t)head * DQ_REC;
        const int n_my = dead ? 0 : max(0, (p1 - p0 - warp + DQ_WARPS - 1) / DQ_WARPS);
        // Page ids of this warp's iterations, 32 at a time: lane l holds the id of iteration base + l.
        int ids_base = 0, my_ids = lane < n_my ? bt[p0 + warp + lane * DQ_WARPS] : 0;
        unsigned bad = 0;                         // bit (iteration % 32): the page is not there, its keys are masked
        const auto issue = [&](int it) {
            if (it >= n_my) return;
            if (it >= ids_base + 32) {
                ids_base += 32;
                my_ids = ids_base + lane < n_my ? bt[p0 + warp + (ids_base + lane) * DQ_WARPS] : 0;
            }
            const int page = __shfl_sync(0xffffffffu, my_ids, it - ids_base);
            bad = page < 0 ? bad | 1u << (it & 31) : bad & ~(1u << (it & 31));
            if (lane == 0) {
                const int place = (done + it) % DQ_STAGES;
                const uint32_t dst = pipe + place * DQ_REC, bar = bars + place * 8;
                asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");  // the place was read (or written by the merge) by ordinary instructions
                asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(bar), "r"(DQ_REC) : "memory");
                asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n"
                             ::"r"(dst), "l"(recs + (size_t)max(page, 0) * page_bytes), "r"(DQ_REC), "r"(bar) : "memory");
            }
        };
        int issued = 0;
        if (!waited) {
            for (; issued < DQ_STAGES && p0 + warp + issued * DQ_WARPS < last_page; ++issued) issue(issued);
            il_pdl_wait();
            waited = true;
        }
        for (; issued < DQ_STAGES; ++issued) issue(issued);

        // Q as the products' right operand, in shared memory in the order in which a product step's lanes read it: head 8 j + lg, of each group of 64 columns the 16 from 16 lq on. A thread
        // makes 16 columns of a head, the lanes of a head agree on its power of two.
#pragma unroll
        for (int i0 = 0; i0 < ROWS * DQ_CH; i0 += DQ_WARPS * 32) {
            const int item = i0 + threadIdx.x, r = item / DQ_CH, c = item % DQ_CH;
            if (ROWS * DQ_CH < DQ_WARPS * 32 && item >= ROWS * DQ_CH) break;       // (whole warps)
            uint32_t x[8], most = 0u;
            {
                const uint4* at = reinterpret_cast<const uint4*>(q + (size_t)e * q_stride + (size_t)(head0 + r) * DQ_HD + 16 * c);
                const uint4 u = r < rows_valid ? at[0] : make_uint4(0u, 0u, 0u, 0u), w = r < rows_valid ? at[1] : make_uint4(0u, 0u, 0u, 0u);
                x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w, x[4] = w.x, x[5] = w.y, x[6] = w.z, x[7] = w.w;
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) most = max(most, max(x[k] & 0x7fffu, x[k] >> 16 & 0x7fffu));
#pragma unroll
            for (int k = 1; k < DQ_CH; k <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, k));
            const int ex = max((int)(most >> 7) - 127, -100);
            const float up = __int_as_float((127 + 8 - ex) << 23);
            if (c == 0) q_scale[r] = scale_log2 * __int_as_float((127 - 8 + ex) << 23);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const __nv_bfloat162 a = *reinterpret_cast<const __nv_bfloat162*>(&x[2 * k]), b = *reinterpret_cast<const __nv_bfloat162*>(&x[2 * k + 1]);
                const float x0 = __low2float(a) * up, x1 = __high2float(a) * up, x2 = __low2float(b) * up, x3 = __high2float(b) * up;
                // (in the order in which K's codes come)
                q_sm[((4 * (c / 4) + k) * 32 + (r % 8) * 4 + c % 4) * NT + r / 8] =
                    KIND == KVQ_E4M3 ? make_uint2(dq_pack_half(x0, x1), dq_pack_half(x2, x3)) : make_uint2(dq_pack_half(x0, x2), dq_pack_half(x1, x3));
            }
        }
        __syncthreads();
        il_f2 s_scale[NT];                        // what the scores of heads 8 j + 2 lq, + 1 are multiplied by (q's power of two taken back)
#pragma unroll
        for (int j = 0; j < NT; ++j) s_scale[j] = il_f2_make(q_scale[8 * j + 2 * lq], q_scale[8 * j + 2 * lq + 1]);

        float o[DQ_MT][NT][4];                    // columns 2 t, 2 t + 1 of lane lg's (elements 0, 1 and 2, 3), heads 8 j + 2 lq, + 1
#pragma unroll
        for (int t = 0; t < DQ_MT; ++t)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[t][j][i] = 0.f;
        float m[NT][2];
        il_f2 l[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) m[j][0] = m[j][1] = -FLT_MAX, l[j] = il_f2_dup(0.f);
        unsigned v_low = DQ_V_LOW;                // (256: none is in order any more)
        for (int it = 0; it < n_my; ++it) {
            if (!dq_wait(bars + (done + it) % DQ_STAGES * 8, (done + it) / DQ_STAGES & 1)) {
                if (lane == 0) atomicExch(status, 91);
                for (int k = it + 1; k < min(it + DQ_STAGES, n_my); ++k) dq_wait(bars + (done + k) % DQ_STAGES * 8, (done + k) / DQ_STAGES & 1);
                dead = true;
                break;
            }
            unsigned char* rec = smem + (size_t)(warp * DQ_STAGES + (done + it) % DQ_STAGES) * DQ_REC;
            // ---- scores of the page's 16 keys: elements 0, 1 are key lg and heads 8 j + 2 lq, + 1; elements 2, 3 key 8 + lg
            float s[NT][4], s1[NT][4];            // (two chains of products where there is one column tile: one alone is all latency)
#pragma unroll
            for (int kg = 0; kg < DQ_KG; ++kg) {
                uint32_t c[2][4];
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const int key = 8 * n + lg, piece = (key * (DQ_HD / 16) + 4 * kg + lq) ^ kvq_turn(DQ_HD, false, key);
                    const uint4 w = *reinterpret_cast<const uint4*>(rec + piece * 16);
                    c[n][0] = w.x, c[n][1] = w.y, c[n][2] = w.z, c[n][3] = w.w;
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t a[4];
                    dq_halves<KIND>(c[0][i], a[0], a[2]);
                    dq_halves<KIND>(c[1][i], a[1], a[3]);
                    uint2 qf[NT];
                    if constexpr (NT == 2) {
                        const uint4 w = *reinterpret_cast<const uint4*>(q_sm + ((4 * kg + i) * 32 + lane) * 2);
                        qf[0] = make_uint2(w.x, w.y), qf[1] = make_uint2(w.z, w.w);
                    } else {
                        qf[0] = q_sm[(4 * kg + i) * 32 + lane];
                    }
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        float(&sum)[4] = NT == 1 && (i & 1) ? s1[j] : s[j];
                        if (kg == 0 && i < (NT == 1 ? 2 : 1)) dq_mma_first(sum, a, qf[j].x, qf[j].y);
                        else dq_mma(sum, a, qf[j].x, qf[j].y);
                    }
                }
            }
            if constexpr (NT == 1)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[0][i] += s1[0][i];
            // ---- exponents of this lane's two keys, softmax in base 2, two heads an instruction. K's power and V's inverse power are made one unit of 2^-23 too large,
            // so that the byte of a row that is NaN, 255, gives a NaN and not an infinity.
            const int page0 = (p0 + warp + it * DQ_WARPS) * KVQ_PAGE;
            const bool gone = (bad >> (it & 31)) & 1, edge = gone || page0 < lo || page0 + KVQ_PAGE > kvlen;
            float tv[NT][4], inv_v[2];
            bool odd[2];                          // an exponent of V out of order
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const uint32_t ke = rec[2 * KVQ_PAGE * DQ_HD + 8 * n + lg], ve = rec[2 * KVQ_PAGE * DQ_HD + KVQ_PAGE + 8 * n + lg];
                const float kp = __uint_as_float(ke << 23 | 1u), add = __uint_as_float(0x4b000000u | ve) - 8388735.f;     // (2^23 + byte as a float has the byte in its lowest bits)
                inv_v[n] = __uint_as_float(0x7f000001u - (ve << 23)), odd[n] = ve - v_low >= DQ_V_SPAN;
#pragma unroll
                for (int j = 0; j < NT; ++j)
                    il_f2_get(il_f2_fma(il_f2_mul(il_f2_make(s[j][2 * n], s[j][2 * n + 1]), il_f2_dup(kp)), s_scale[j], il_f2_dup(add)), tv[j][2 * n], tv[j][2 * n + 1]);
            }
            if (edge) {
                if (KIND == KVQ_E4M3)             // (which has codes that are NaN: rows of V that do not count are cleared where they lie)
                    for (int i = lane; i < KVQ_PAGE * DQ_CH; i += 32) {
                        const int k = i / DQ_CH, key = page0 + k;
                        if (gone || key < lo || key >= kvlen) *reinterpret_cast<uint4*>(rec + KVQ_PAGE * DQ_HD + (i ^ kvq_turn(DQ_HD, true, k)) * 16) = make_uint4(0u, 0u, 0u, 0u);
                    }
                __syncwarp();
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const int key = page0 + 8 * n + lg;
                    if (gone || key < lo || key >= kvlen) {
                        inv_v[n] = 0.f, odd[n] = false;
#pragma unroll
                        for (int j = 0; j < NT; ++j) tv[j][2 * n] = tv[j][2 * n + 1] = -INFINITY;
                    }
                }
            }
            // how far above the reference (which starts at the lowest float, so that no difference is one of infinities)
            float dv[NT][4], top = -INFINITY;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const il_f2 neg_m = il_f2_make(-m[j][0], -m[j][1]);
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    il_f2_get(il_f2_add(il_f2_make(tv[j][2 * n], tv[j][2 * n + 1]), neg_m), dv[j][2 * n], dv[j][2 * n + 1]);
                    top = fmaxf(fmaxf(top, dv[j][2 * n]), dv[j][2 * n + 1]);
                }
            }
            if (__any_sync(0xffffffffu, top > DQ_UP + DQ_RAISE || odd[0] || odd[1])) {           // also the first keys of a head
                const bool far = __any_sync(0xffffffffu, odd[0] || odd[1]);
                if (__builtin_expect(far, 0)) {
                    // A row of zeros has the exponent 2^0, far above its neighbours', and must not set the reference that their weights are rounded against: it gets the lowest.
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        const int key = 8 * n + lg;
                        uint32_t some = inv_v[n] != __uint_as_float(0x7f000001u - (127u << 23));
                        if (!some)
                            for (int c = lq; c < DQ_CH; c += 4) {
                                const uint4 w = *reinterpret_cast<const uint4*>(rec + KVQ_PAGE * DQ_HD + ((key * DQ_CH + c) ^ kvq_turn(DQ_HD, true, key)) * 16);
                                some |= (w.x | w.y | w.z | w.w) & 0x7f7f7f7fu;        // (zeros of either sign)
                            }
                        some |= __shfl_xor_sync(0xffffffffu, some, 1);
                        some |= __shfl_xor_sync(0xffffffffu, some, 2);
                        if (some) continue;
                        inv_v[n] = __uint_as_float(0x7f000001u - ((unsigned)(KVQ_LEAST + 127) << 23));
#pragma unroll
                        for (int j = 0; j < NT; ++j) tv[j][2 * n] += (float)KVQ_LEAST, tv[j][2 * n + 1] += (float)KVQ_LEAST;
                    }
                }
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    float root[2], corr[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float mx = fmaxf(tv[j][i], tv[j][2 + i]);
#pragma unroll
                        for (int x = 4; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
                        const float mn = mx > m[j][i] + (far ? DQ_UP : DQ_UP + DQ_RAISE) ? mx - DQ_UP : m[j][i];     // (far: a key's share of the denominator stays below 2^107)
                        root[i] = dq_root(m[j][i], mn), corr[i] = root[i] * root[i];      // 0 when nothing was summed yet
                        m[j][i] = mn, dv[j][i] = tv[j][i] - mn, dv[j][2 + i] = tv[j][2 + i] - mn;
                    }
                    l[j] = il_f2_mul(il_f2_mul(l[j], il_f2_make(root[0], root[1])), il_f2_make(root[0], root[1]));
#pragma unroll
                    for (int t = 0; t < DQ_MT; ++t) o[t][j][0] *= corr[0], o[t][j][1] *= corr[1], o[t][j][2] *= corr[0], o[t][j][3] *= corr[1];
                }
                if (__builtin_expect(far, 0)) {   // a key's share of the denominator by an exponential of its own: its weight may be flushed to 0 where its score counts all the same
                    bool above = false;
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        const int v = (int)(0x7f000001u - __float_as_uint(inv_v[n]) >> 23);       // the exponent's byte again; of a masked key 254
                        above = above || (v >= (int)(DQ_V_LOW + DQ_V_SPAN) && v <= KVQ_MOST + 127);
                        if (v == KVQ_NAN) continue;           // (stays NaN)
#pragma unroll
                        for (int j = 0; j < NT; ++j)
                            l[j] = il_f2_add(l[j], il_f2_make(dq_ex2_small(dv[j][2 * n] - (float)(v - 127)), dq_ex2_small(dv[j][2 * n + 1] - (float)(v - 127))));
                        inv_v[n] = 0.f;
                    }
                    if (__any_sync(0xffffffffu, above)) v_low = 256u;     // what is in order so far may be far below this one: every page of the stretch from here on
                }
            }
            uint32_t pf[NT][2];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const float w0 = dq_ex2(dv[j][2 * n]), w1 = dq_ex2(dv[j][2 * n + 1]);
                    l[j] = il_f2_fma(il_f2_make(w0, w1), il_f2_dup(inv_v[n]), l[j]);          // (this lane's keys; a head's lanes are added at the end)
                    pf[j][n] = dq_transpose(dq_pack_half(w0, w1));
                }
            }
            // ---- P.V: four keys of this lane's columns, DQ_VB of them at a time
#pragma unroll
            for (int vb = 0; vb < DQ_NVB; ++vb) {
                uint32_t x[4][DQ_VB / 4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int key = 2 * lq + (k & 1) + 8 * (k >> 1), col = vb * 8 * DQ_VB + lg * DQ_VB;
                    const int piece = (key * (DQ_HD / 16) + col / 16) ^ kvq_turn(DQ_HD, true, key);
                    const unsigned char* at = rec + KVQ_PAGE * DQ_HD + piece * 16 + col % 16;
                    if constexpr (DQ_VB == 16) {
                        const uint4 w = *reinterpret_cast<const uint4*>(at);
                        x[k][0] = w.x, x[k][1] = w.y, x[k][2] = w.z, x[k][3] = w.w;
                    } else {
                        const uint2 w = *reinterpret_cast<const uint2*>(at);
                        x[k][0] = w.x, x[k][1] = w.y;
                    }
                }
#pragma unroll
                for (int i = 0; i < DQ_VB / 4; ++i)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {             // columns 4 i + 2 c, + 1: two keys of a column side by side
                        uint32_t a[4];
#pragma unroll
                        for (int n = 0; n < 2; ++n) {
                            const uint32_t w = __byte_perm(x[2 * n][i], x[2 * n + 1][i], KIND == KVQ_E4M3 ? (c ? 0x7362 : 0x5140) : (c ? 0x7632 : 0x5410));
                            dq_halves<KIND>(w, a[2 * n], a[2 * n + 1]);
                        }
#pragma unroll
                        for (int j = 0; j < NT; ++j) dq_mma(o[vb * (DQ_VB / 2) + 2 * i + c][j], a, pf[j][0], pf[j][1]);
                    }
            }
            __syncwarp();
            issue(it + DQ_STAGES);                // refill the place this record came from
        }
        done += n_my;
        if (at >= to) il_pdl_tail();              // (behind the last stretch's products: what follows may become resident)
        float lsum[NT][2];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            il_f2_get(l[j], lsum[j][0], lsum[j][1]);
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) lsum[j][i] += __shfl_xor_sync(0xffffffffu, lsum[j][i], x);
        }
        __syncthreads();                          // the rings' memory is reused for the merge

        // The four warps' sums, brought to the heads' common maximum, then added in warp order.
        float* sm_ml = reinterpret_cast<float*>(smem);                     // [warp][row][m, l]
        float* sm_o = sm_ml + (DQ_WARPS + 1) * ROWS * 2;                   // behind the rows' own m and l: [warp][row][DQ_OS]
        if (lg == 0) {
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    sm_ml[(warp * ROWS + 8 * j + 2 * lq + i) * 2] = m[j][i];
                    sm_ml[(warp * ROWS + 8 * j + 2 * lq + i) * 2 + 1] = lsum[j][i];
                }
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = 8 * j + 2 * lq + i;
                float M = -INFINITY;
#pragma unroll
                for (int w = 0; w < DQ_WARPS; ++w) M = fmaxf(M, sm_ml[(w * ROWS + r) * 2]);
                const float f = m[j][i] == -INFINITY ? 0.f : dq_ex2(m[j][i] - M);
                float* row = sm_o + (size_t)(warp * ROWS + r) * DQ_OS;
#pragma unroll
                for (int vb = 0; vb < DQ_NVB; ++vb)
#pragma unroll
                    for (int t = 0; t < DQ_VB / 2; t += 2) {
                        const int tt = vb * (DQ_VB / 2) + t;
                        *reinterpret_cast<float4*>(row + vb * 8 * DQ_VB + lg * DQ_VB + 2 * t) = make_float4(f * o[tt][j][i], f * o[tt][j][2 + i], f * o[tt + 1][j][i], f * o[tt + 1][j][2 + i]);
                    }
            }
        if (threadIdx.x < ROWS) {
            const int r = threadIdx.x;
            float M = -INFINITY, L = 0.f;
#pragma unroll
            for (int w = 0; w < DQ_WARPS; ++w) M = fmaxf(M, sm_ml[(w * ROWS + r) * 2]);
#pragma unroll
            for (int w = 0; w < DQ_WARPS; ++w) {
                const float mw = sm_ml[(w * ROWS + r) * 2];
                const float root = dq_root(mw, M);
                L += sm_ml[(w * ROWS + r) * 2 + 1] * root * root;
            }
            *reinterpret_cast<float2*>(sm_ml + (DQ_WARPS * ROWS + r) * 2) = make_float2(M, L);
        }
        __syncthreads();
        // final where the whole unit lies in this block, else a part: in scratch, or for the cluster here, in the first warp's place
        const bool final = start >= from && start + n_pages <= to;
        const size_t place = 2 * blockIdx.x + (start >= from ? 1 : 0);
        __nv_bfloat16* out_rows = out + ((size_t)e * nh + head0) * DQ_HD;
#pragma unroll
        for (int i = 0; i < ROWS * (DQ_HD / 4); i += DQ_WARPS * 32) {
            const int idx = i + threadIdx.x, r = idx / (DQ_HD / 4), d = (idx - r * (DQ_HD / 4)) * 4;
            if (r >= rows_valid) break;
            const float2 ML = *reinterpret_cast<const float2*>(sm_ml + (DQ_WARPS * ROWS + r) * 2);
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < DQ_WARPS; ++w) {
                const float4 v = *reinterpret_cast<const float4*>(sm_o + (size_t)(w * ROWS + r) * DQ_OS + d);
                acc.x += v.x, acc.y += v.y, acc.z += v.z, acc.w += v.w;
            }
            if (per_unit > 1) *reinterpret_cast<float4*>(sm_o + (size_t)r * DQ_OS + d) = acc;
            else dq_write(acc, ML.x, ML.y, final ? out_rows : nullptr, o_part + place * ROWS * DQ_HD, ml_part + place * (2 * ROWS), r, d);
        }
        __syncthreads();                              // the next stretch's copies come where the merge was
    }
    if (!waited) il_pdl_wait();
    if (per_unit > 1) {                           // the cluster's parts added up in block order, each block a share of the columns
        const uint32_t sm_ml = (uint32_t)__cvta_generic_to_shared(smem) + DQ_WARPS * ROWS * 8, sm_o = sm_ml + ROWS * 8;
        const int u = blockIdx.x / per_unit, rank = blockIdx.x - u * per_unit, i = u / units, head = (u - i * units) / row_tiles, rt = u - i * units - head * row_tiles;
        const int head0 = head * G + rt * ROWS, rows_valid = min(ROWS, G - rt * ROWS);
        il_cluster_sync();
        for (int idx = rank * DQ_WARPS * 32 + threadIdx.x; idx < rows_valid * (DQ_HD / 4); idx += per_unit * DQ_WARPS * 32) {
            const int r = idx / (DQ_HD / 4), d = (idx - r * (DQ_HD / 4)) * 4;
            float2 ml[DQ_CLUSTER];
            float4 v[DQ_CLUSTER], acc = make_float4(0.f, 0.f, 0.f, 0.f);
            float M = -INFINITY, L = 0.f;
#pragma unroll
            for (int p = 0; p < DQ_CLUSTER; ++p)
                if (p < per_unit) ml[p] = dq_peer2(sm_ml + r * 8, p), v[p] = dq_peer4(sm_o + (r * DQ_OS + d) * 4, p), M = fmaxf(M, ml[p].x);
#pragma unroll
            for (int p = 0; p < DQ_CLUSTER; ++p)
                if (p < per_unit && ml[p].x != -INFINITY) {           // (no part: what lies there is not one)
                    const float root = dq_root(ml[p].x, M), f = root * root;
                    L += ml[p].y * root * root, acc.x += f * v[p].x, acc.y += f * v[p].y, acc.z += f * v[p].z, acc.w += f * v[p].w;
                }
            dq_write(acc, M, L, out + ((size_t)i * nh + head0) * DQ_HD, nullptr, nullptr, r, d);
        }
        il_cluster_sync();                        // (nobody leaves while its part is read)
    }
    // requests without a key: zeros
    for (int z = blockIdx.x; z < n_decode; z += n_blocks)
        if (entry_kvlen[z] <= 0)
            for (int i = threadIdx.x; i < nh * (DQ_HD / 8); i += DQ_WARPS * 32) *reinterpret_cast<uint4*>(out + (size_t)z * nh * DQ_HD + i * 8) = make_uint4(0u, 0u, 0u, 0u);
}

// The parts of a row (a head of a request) added up, WPR warps a row: warp w takes parts w, w + WPR, ..., DQM_ROUND loads under way at a time, a lane four columns, with a
// running maximum over its rounds (a maximum over all parts first would be one more trip to memory); the warps' sums are then added in warp order. Lengths are read before the
// wait: they were there when the kernel in front, which waits before it ends, began.
constexpr int DQM_ROUND = HEAD_DIM > 128 ? 8 : 16;
template <int WPR>
__global__ void __launch_bounds__(WPR > 4 ? WPR * 32 : 128) attn_decode_quant_merge_kernel(const float* o_part, const float* ml_part, const int* __restrict__ entry_kvlen, int n_decode,
                                                                                          int nh, int G, int rows, int row_tiles, int units, int window, int n_blocks, __nv_bfloat16* out) {
    constexpr int PER = WPR > 4 ? 1 : 4 / WPR;    // rows of a block
    constexpr int LPR = DQ_HD / 4 < 32 ? DQ_HD / 4 : 32, PPW = 32 / LPR;      // lanes that a part's row takes; the others take the next part of the warp
    constexpr int NC = DQ_HD > 128 ? 2 : 1;
    __shared__ float comb[WPR > 1 ? WPR * DQ_HD : 1];
    __shared__ float2 sums[WPR > 1 ? WPR : 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = warp % WPR, row = blockIdx.x * PER + warp / WPR;
    const bool there = row < n_decode * nh;
    const int e = there ? row / nh : 0, h = row - e * nh;
    const int head = h / G, rt = (h - head * G) / rows, r = h - head * G - rt * rows;
    const DqDeal d = dq_deal(entry_kvlen, n_decode, window, units, n_blocks, 0, lane);
    int before = 0, first;
    for (int i = lane; i < e; i += 32) before += dq_pages(entry_kvlen[i], window, &first);
    before = __reduce_add_sync(0xffffffffu, before) * units;
    const int n = there ? dq_pages(entry_kvlen[e], window, &first) : 0, start = before + (head * row_tiles + rt) * n;
    const int b0 = start / d.share, n_parts = n > 0 ? (start + n - 1) / d.share - b0 + 1 : 0;
    il_pdl_wait();
    if (n_parts <= 1) return;                     // final already (all warps of a row alike; with more than one warp a row, the block)
    float acc[NC][4], M = -INFINITY, L = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) acc[c][0] = acc[c][1] = acc[c][2] = acc[c][3] = 0.f;
    const int d0 = lane % LPR * 4;
    for (int i0 = sub * PPW + lane / LPR; i0 < n_parts; i0 += DQM_ROUND * WPR * PPW) {
        float4 v[NC][DQM_ROUND];
        float2 ml[DQM_ROUND];
#pragma unroll
        for (int k = 0; k < DQM_ROUND; ++k) {     // (behind the last part: a part that is there, counted with factor 0; loads behind a branch would wait for one another)
            const int i = i0 + k * WPR * PPW;
            const size_t at = (size_t)dq_place(b0, i < n_parts ? i : i0) * rows + r;
#pragma unroll
            for (int c = 0; c < NC; ++c) v[c][k] = *reinterpret_cast<const float4*>(o_part + at * DQ_HD + 128 * c + d0);
            ml[k] = *reinterpret_cast<const float2*>(ml_part + at * 2);
            if (i >= n_parts) ml[k] = make_float2(-INFINITY, 0.f);
        }
        float mx = M;
#pragma unroll
        for (int k = 0; k < DQM_ROUND; ++k) mx = fmaxf(mx, ml[k].x);
        const float back = dq_root(M, mx), corr = back * back;
        M = mx, L = L * back * back;
#pragma unroll
        for (int c = 0; c < NC; ++c) acc[c][0] *= corr, acc[c][1] *= corr, acc[c][2] *= corr, acc[c][3] *= corr;
#pragma unroll
        for (int k = 0; k < DQM_ROUND; ++k) {
            const float root = dq_root(ml[k].x, M), f = root * root;
            L += ml[k].y * root * root;           // (a NaN of a part that is there stays one)
#pragma unroll
            for (int c = 0; c < NC; ++c) acc[c][0] += f * v[c][k].x, acc[c][1] += f * v[c][k].y, acc[c][2] += f * v[c][k].z, acc[c][3] += f * v[c][k].w;
        }
    }
#pragma unroll
    for (int x = LPR; x < 32; x <<= 1) {          // lanes that had other parts of the same columns
        const float Mo = __shfl_xor_sync(0xffffffffu, M, x), mx = fmaxf(M, Mo), root = dq_root(M, mx), f = root * root;
        L = L * root * root, L += __shfl_xor_sync(0xffffffffu, L, x);
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[0][c] *= f, acc[0][c] += __shfl_xor_sync(0xffffffffu, acc[0][c], x);
        M = mx;
    }
    if constexpr (WPR > 1) {
        if (lane < LPR)
#pragma unroll
            for (int c = 0; c < NC; ++c) *reinterpret_cast<float4*>(comb + sub * DQ_HD + 128 * c + d0) = make_float4(acc[c][0], acc[c][1], acc[c][2], acc[c][3]);
        if (lane == 0) sums[sub] = make_float2(M, L);
        __syncthreads();
        if (sub) return;
        float f[WPR];
        M = -INFINITY, L = 0.f;
#pragma unroll
        for (int w = 0; w < WPR; ++w) M = fmaxf(M, sums[w].x);
#pragma unroll
        for (int w = 0; w < WPR; ++w) {
            const float root = dq_root(sums[w].x, M);
            f[w] = root * root, L += sums[w].y * root * root;
        }
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            acc[c][0] = acc[c][1] = acc[c][2] = acc[c][3] = 0.f;
#pragma unroll
            for (int w = 0; w < WPR; ++w) {
                const float4 v = *reinterpret_cast<const float4*>(comb + w * DQ_HD + 128 * c + d0);
                acc[c][0] += f[w] * v.x, acc[c][1] += f[w] * v.y, acc[c][2] += f[w] * v.z, acc[c][3] += f[w] * v.w;
            }
        }
    }
    if (lane >= LPR) return;
#pragma unroll
    for (int c = 0; c < NC; ++c) dq_write(make_float4(acc[c][0], acc[c][1], acc[c][2], acc[c][3]), M, L, out + (size_t)row * DQ_HD, nullptr, nullptr, 0, 128 * c + d0);
}

// Calls go(kernel, shared memory) for the kernel of these.
template <typename Go>
static auto dq_pick(int kind, int group, Go go) {
    if (group <= 8) return kind == KVQ_E4M3 ? go(attn_decode_quant_kernel<KVQ_E4M3, 1>, dq_smem(8)) : go(attn_decode_quant_kernel<KVQ_INT8, 1>, dq_smem(8));
    return kind == KVQ_E4M3 ? go(attn_decode_quant_kernel<KVQ_E4M3, 2>, dq_smem(16)) : go(attn_decode_quant_kernel<KVQ_INT8, 2>, dq_smem(16));
}
static int dq_prepare(int dev) {
    static bool done[64];
    if (dev < 0 || dev >= 64 || done[dev]) return IL_OK;
    cudaError_t e = cudaSuccess;
    for (int i = 0; i < 4 && e == cudaSuccess; ++i)
        e = dq_pick(i & 1, i & 2 ? 16 : 1, [](auto kernel, int smem) { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); });
    if (e != cudaSuccess) return 1000 + (int)e;
    done[dev] = true;
    return IL_OK;
}

// Blocks that this device runs at once, with `group` query heads a kv head; 0 if the query fails.
IL_EXPORT int il_attn_decode_quant_resident_blocks(int kind, int group) {
    int dev = 0, sms = 0, n = 0;
    const bool ok = cudaGetDevice(&dev) == cudaSuccess && dq_prepare(dev) == IL_OK && cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess &&
                    dq_pick(kind, group, [&](auto kernel, int smem) { return cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, DQ_WARPS * 32, smem); }) == cudaSuccess;
    if (!ok) cudaGetLastError();
    return ok ? n * sms : 0;
}

// n_blocks: blocks that the pages are dealt out to; 0: a block a unit; -2 .. -8: a cluster of so many blocks a unit. Scratch for n_blocks > 0: o_part float32 [2 * n_blocks * 16 * head_dim], ml_part [2 * n_blocks * 32].
// (Arguments as one struct: see kv_quant.cu.)
struct DqArgs {
    const void* q;
    long long q_stride;
    void* out;
    const void* cache;
    const int *block_table, *entry_kvlen;
    float *o_part, *ml_part;
    int* status;
    cudaStream_t stream;
    int kind, bt_stride, n_decode, nh, nkv, hd, window, n_blocks, early;
    float scale;
};
static_assert(sizeof(DqArgs) == 120, "what ops.py packs, padding included");
IL_EXPORT int il_attn_decode_quant(const DqArgs* args) {
    const DqArgs& a = *args;
    const int kind = a.kind, n_decode = a.n_decode, nh = a.nh, nkv = a.nkv, hd = a.hd, n_blocks = a.n_blocks;
    if (n_decode <= 0) return IL_OK;
    if (hd != HEAD_DIM) return IL_UNSUPPORTED;
    if (nh <= 0 || nkv <= 0 || nh % nkv != 0 || n_blocks < -DQ_CLUSTER || (kind != KVQ_E4M3 && kind != KVQ_INT8) || !a.status) return IL_BAD_ARG;
    const int group = nh / nkv, rows = group <= 8 ? 8 : 16, row_tiles = (group + rows - 1) / rows, units = nkv * row_tiles;
    if ((long long)n_decode * units * (a.bt_stride > DQ_CLUSTER ? a.bt_stride : DQ_CLUSTER) > 0x7fffffffLL || n_blocks > 0x3fffffff) return IL_UNSUPPORTED;   // (pages of all units are counted in 32 bits)
    if (n_blocks > 0 && (!a.o_part || !a.ml_part)) return IL_BAD_ARG;
    if ((((uintptr_t)a.cache | (uintptr_t)a.q | (uintptr_t)a.out) & 15) || (a.q_stride & 7) || a.q_stride < (long long)nh * hd) return IL_BAD_ARG;
    int dev = 0;
    cudaGetDevice(&dev);
    const int rc = dq_prepare(dev);
    if (rc != IL_OK) return rc;
    const int per_unit = n_blocks > 0 ? 0 : n_blocks == 0 ? 1 : -n_blocks;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization, attr[0].val.programmaticStreamSerializationAllowed = il_pdl_enabled();
    attr[1].id = cudaLaunchAttributeClusterDimension, attr[1].val.clusterDim.x = per_unit, attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.gridDim = dim3(per_unit ? n_decode * units * per_unit : n_blocks), cfg.blockDim = dim3(DQ_WARPS * 32), cfg.stream = a.stream, cfg.attrs = attr, cfg.numAttrs = per_unit > 1 ? 2 : 1;
    cudaError_t e = dq_pick(kind, group, [&](auto kernel, int smem) {
        cfg.dynamicSmemBytes = (size_t)smem;
        return cudaLaunchKernelEx(&cfg, kernel, (const __nv_bfloat16*)a.q, (long long)a.q_stride, (const unsigned char*)a.cache, a.block_table, (int)a.bt_stride, a.entry_kvlen, (int)n_decode, (int)nh,
                                  (int)nkv, (int)group, (int)row_tiles, a.scale * 1.4426950408889634f, (int)a.window, (int)per_unit, a.o_part, a.ml_part, (__nv_bfloat16*)a.out, a.status, (int)a.early);
    });
    if (e == cudaSuccess && !per_unit) {
        // warps a row by the parts that a unit has if the requests are alike
        const int parts = n_blocks / (n_decode * units), n_rows = n_decode * nh;
        const auto merge = [&](auto kernel, int blocks, int threads) {
            return il_launch(kernel, dim3(blocks), dim3(threads), (size_t)0, a.stream, (const float*)a.o_part, (const float*)a.ml_part, a.entry_kvlen, n_decode, nh, group, rows, row_tiles, units, a.window, n_blocks,
                             (__nv_bfloat16*)a.out);
        };
        e = parts > 64 ? merge(attn_decode_quant_merge_kernel<16>, n_rows, 512) : parts > 8 ? merge(attn_decode_quant_merge_kernel<4>, n_rows, 128)
                                                                                : merge(attn_decode_quant_merge_kernel<1>, (n_rows + 3) / 4, 128);
    }
    if (e != cudaSuccess) return 1000 + (int)e;
    IL_LAUNCH_CHECK();
    return IL_OK;
}
