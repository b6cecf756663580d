// Prompt attention over pages of 16 keys in bfloat16 on the 5th-generation tensor cores, two tiles of 128 rows a block (head_dim 64 or 128): each token of a portion
// attends causally (and inside its window) to what its request has in the cache, earlier steps' keys and this step's own.
//
//   A block owns two row tiles, A and B: each TPT consecutive tokens of one entry times the G query heads of one kv head (row r -> token r / G, head r % G), B's tokens
//   behind A's. Both walk the same key tiles of 128 keys (eight pages), so a key tile is fetched once for 256 rows.
//     S = Q.K^T   tcgen05.mma, M 128, N 128, both operands in shared memory (K-major, 128-byte swizzle); S lies in tensor memory, 128 columns for each row tile.
//     softmax     four warps a row tile, one thread a row: its 128 scores come into registers at once, their maximum; then weights, base 2 with the scale folded in, two scores an
//                 instruction, f32 sums. The reference m is raised only when a tile's maximum is more than 2^8 above it; the row of O is then rescaled in tensor memory. P goes
//                 back as bfloat16 over the scores: the left operand of the next product comes from tensor memory.
//     O += P.V    tcgen05.mma, M 128, N head_dim, A = P from tensor memory, B = the V pages as they lie in the cache (MN-major); O in tensor memory, divided by the sums in the end.
//   One thread issues all products: P.V of A, then S of A's next tile, then the same for B. While one row tile's softmax runs, the tensor cores have the other's products; products are
//   worked off in the order they are issued, so S may follow the P.V that reads P from its place, and a tile's scores are complete only when O holds everything before.
//   Roles by warp: 0 producer (TMA, one copy a page through a view of the cache whose box lands as tensor-core tiles), 1 tensor-memory allocation, 2 products, 3 waits for keys and values, 4 - 7 and 8 - 11
//   softmax and output of A and of B. All 512 columns of tensor memory and (head_dim 128) 192 KB of shared memory: one block an SM.
//   What bounds it: a row tile's chain, some 3,250 clocks a key tile - its products 890, their way to the softmax and back 500, loads and maximum 450, exponentials 1,300 (1,024 of them
//   the special-function unit's) -, two of which the block runs against each other; the tensor cores are busy seven tenths of it. One row tile a block, key tiles of 64 and two
//   blocks an SM (attn_prefill_tc5) / this, us with the pages' reading: 8,192 tokens, 32 heads on 8 of 128, 563 / 483; 4,096 of 32 on 2 164 / 145 to 159; 8,192 of 16 on 2 of 64 265 / 209; 1,024 behind
//   8,000, 32 on 8, 170 / 144. Slower, from 501 us of the first, were: a thread of its own for each row tile's products (they then interleave in the tensor cores: 728 for 501), P handed over in halves
//   (492, but 152 for 145), one pair of exponentials of eight by a polynomial on the multiply-add units (549), scores read twice instead of kept in registers (512).
//
//   Every mbarrier wait is bounded; one that runs out sets *status and all roles leave their loops.
//   grid tiles x kv heads. Tiles of 2 TPT tokens are numbered over the entries [first_entry, n_entries) in order; a block finds its entry by walking entry_qstart.
#include "tcgen05.cuh"

#ifndef HEAD_DIM
#error "compile with -DHEAD_DIM=64 or 128"
#endif
static_assert(HEAD_DIM == 64 || HEAD_DIM == 128, "the paired prompt kernel takes head_dim 64 or 128");

constexpr int PP_HD = HEAD_DIM;
constexpr int PP_HALVES = HEAD_DIM / 64;          // 128-byte column blocks of a row
constexpr int PP_ROWS = 128;                      // rows of a tile; a block has two tiles
constexpr int PP_KEYS = 128;
constexpr int PP_PAGE = 16;
constexpr int PP_TILE_PAGES = PP_KEYS / PP_PAGE;
constexpr int PP_STAGES = 2;                      // of K and of V each
constexpr int PP_Q_HALF = PP_ROWS * 128;          // bytes of one column block of a row tile of Q
constexpr int PP_Q_BYTES = PP_HALVES * PP_Q_HALF;
constexpr int PP_ATOM = PP_HALVES * 1024;         // K and V tiles: 1 KB atoms (8 keys x 64 columns); the next 8 keys this far on, the next column block 1 KB
constexpr int PP_PAGE_BYTES = 2 * PP_ATOM;
constexpr int PP_K_BYTES = PP_TILE_PAGES * PP_PAGE_BYTES;
constexpr int PP_THREADS = 384;
constexpr int PP_COL_S = 0, PP_COL_O = 2 * PP_KEYS;           // S of A, S of B, O of A, O of B
constexpr int PP_N_BARS = 1 + 4 * PP_STAGES + 7;
constexpr int PP_SMEM = 2 * PP_Q_BYTES + 2 * PP_STAGES * PP_K_BYTES + PP_N_BARS * 8 + 16;
static_assert(PP_SMEM <= 227 * 1024, "shared memory of a block");
constexpr unsigned PP_SPIN = 1u << 22;
constexpr float PP_RAISE = 8.f;                   // the running maximum follows a tile's only beyond this (log2 units)

__device__ __forceinline__ void pp_tma_page(uint32_t dst, const CUtensorMap* map, int block16, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %3, %3, %3, %4}], [%2];\n"
                 ::"r"(dst), "l"(map), "r"(bar), "r"(0), "r"(block16) : "memory");
}
__device__ __forceinline__ float pp_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pp_pack(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ float pp_max3(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;\n" : "=f"(d) : "f"(a), "f"(b), "f"(c));      // (a score that is NaN makes the row's reference NaN, and so its sums)
    return d;
}
// 16 columns of this thread's lane, as one warp.
__device__ __forceinline__ void pp_st16(uint32_t taddr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
                 "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
__global__ void __launch_bounds__(PP_THREADS, 1) attn_prefill_pair_kernel(
    const __grid_constant__ CUtensorMap kv_map, const __nv_bfloat16* q, long long q_stride, __nv_bfloat16* out, const int* block_table, int bt_stride,
    const int* entry_qstart, const int* entry_kvlen, int first_entry, int n_entries, int nh, int nkv, float scale_log2, int window, int tpt, int* status) {
    extern __shared__ __align__(1024) unsigned char smem[];
    if (t5_smem(smem) & 1023u) {                  // the swizzled tiles need 1 KB alignment; dynamic shared memory starts on it
        if (threadIdx.x == 0) atomicExch(status, 101);
        return;
    }
    const int G = nh / nkv, g = blockIdx.x % nkv, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // Which entry and which tokens: tiles are taken from the last to the first, so that of a request the longest blocks start first, kv heads side by side (one kv head behind the other: 495 for
    // 485 us, 8,192 tokens, 32 heads on 8 of 128; the requests by length instead: 161 for 154, five of 37 to 1,024 tokens behind up to 4,096).
    int tile = (int)(gridDim.x / nkv - 1 - blockIdx.x / nkv), e = first_entry;
    for (; e < n_entries; ++e) {
        const int nt = (entry_qstart[e + 1] - entry_qstart[e] + 2 * tpt - 1) / (2 * tpt);
        if (tile < nt) break;
        tile -= nt;
    }
    if (e >= n_entries) return;                   // the whole block
    const int q0 = entry_qstart[e], q1 = entry_qstart[e + 1], kvlen = entry_kvlen[e], start_pos = kvlen - (q1 - q0);
    const int tok0 = q0 + tile * 2 * tpt, n_tok = min(2 * tpt, q1 - tok0), n_a = min(n_tok, tpt), n_b = n_tok - n_a;
    const int* bt = block_table + (size_t)e * bt_stride;
    const int pos0 = start_pos + (tok0 - q0);     // A's first position
    const int page_first = il_mask_lo(pos0, window) / PP_PAGE, page_last = (pos0 + n_tok - 1) / PP_PAGE;
    const int tiles_a = ((pos0 + n_a - 1) / PP_PAGE - page_first) / PP_TILE_PAGES + 1;       // key tiles that A's rows can see some of
    const int n_tiles = (page_last - page_first) / PP_TILE_PAGES + 1, tiles_b = n_b > 0 ? n_tiles : 0;

    unsigned char* q_smem = smem;
    unsigned char* k_smem = smem + 2 * PP_Q_BYTES;
    unsigned char* v_smem = k_smem + PP_STAGES * PP_K_BYTES;
    uint64_t* bars = reinterpret_cast<uint64_t*>(v_smem + PP_STAGES * PP_K_BYTES);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + PP_N_BARS);
    const uint32_t bar0 = t5_smem(bars);
    const uint32_t q_full = bar0;                                     // Q is in shared memory (8 warps)
    const uint32_t k_full0 = bar0 + 8, k_empty0 = k_full0 + 8 * PP_STAGES, v_full0 = k_empty0 + 8 * PP_STAGES, v_empty0 = v_full0 + 8 * PP_STAGES;
    const uint32_t s_full0 = v_empty0 + 8 * PP_STAGES;                // a row tile's scores are complete, and so is all that O got before (tcgen05.commit)
    const uint32_t p_full0 = s_full0 + 16;                            // a row tile's P is in tensor memory (4 warps), and the keys and values that are needed next in shared memory (warp 3)
    const uint32_t o_done0 = p_full0 + 16;                            // a row tile's last product is through (tcgen05.commit)
    const uint32_t drained = o_done0 + 16;                            // after a wait that ran out: all products are (tcgen05.commit)
    if (threadIdx.x == 0) {
        t5_mbar_init(q_full, 8);
        for (int s = 0; s < PP_STAGES; ++s) t5_mbar_init(k_full0 + 8 * s, 1), t5_mbar_init(k_empty0 + 8 * s, 1), t5_mbar_init(v_full0 + 8 * s, 1), t5_mbar_init(v_empty0 + 8 * s, 1);
        t5_mbar_init(drained, 1);
        for (int t = 0; t < 2; ++t) t5_mbar_init(s_full0 + 8 * t, 1), t5_mbar_init(p_full0 + 8 * t, 5), t5_mbar_init(o_done0 + 8 * t, 1);
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
    }
    if (warp == 1) t5_alloc(tmem_slot, 512);
    t5_fence_before();
    __syncthreads();
    t5_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0) {
        // ---------------- producer: K and V pages by TMA, K one tile ahead of V ----------------
        // Page ids come from the block table ahead of their use: lane l holds the id of page base + l (`cur`) and of page base + 32 + l (`nxt`).
        int base = page_first;
        int cur = bt[min(base + lane, page_last)], nxt = bt[min(base + 32 + lane, page_last)];
        const auto issue = [&](int j, int kv) -> bool {
            const int stage = j % PP_STAGES, round = j / PP_STAGES;
            const uint32_t full = (kv ? v_full0 : k_full0) + 8 * stage;
            while (kv && page_first + j * PP_TILE_PAGES >= base + 32) {           // V(j) is the tile furthest behind: the window follows it
                base += 32;
                cur = nxt;
                nxt = bt[min(base + 32 + lane, page_last)];
            }
            int ok = 1;
            if (lane == 0) {
                if (!t5_mbar_wait((kv ? v_empty0 : k_empty0) + 8 * stage, ((uint32_t)round & 1u) ^ 1u, PP_SPIN)) {
                    atomicExch(status, 102);
                    ok = 0;
                } else {
                    t5_mbar_expect_tx(full, PP_K_BYTES);
                }
            }
            ok = __shfl_sync(0xffffffffu, ok, 0);
            const int p = lane % PP_TILE_PAGES, off = min(page_first + j * PP_TILE_PAGES + p, page_last) - base;       // 0 .. 63 (pages behind the last: the last again, masked)
            const int id_cur = __shfl_sync(0xffffffffu, cur, off & 31), id_nxt = __shfl_sync(0xffffffffu, nxt, off & 31);
            if (ok && lane < PP_TILE_PAGES) {
                const int page = off < 32 ? id_cur : id_nxt;
                pp_tma_page(t5_smem((kv ? v_smem : k_smem) + stage * PP_K_BYTES + p * PP_PAGE_BYTES), &kv_map, (page * 2 + kv) * nkv + g, full);
            }
            return ok != 0;
        };
        bool ok = issue(0, 0);
        int n_k = ok, n_v = 0;
        for (int j = 0; j < n_tiles && ok; ++j) {
            if (j + 1 < n_tiles) ok = issue(j + 1, 0), n_k += ok;
            if (ok) ok = issue(j, 1), n_v += ok;
        }
        if (lane == 0) {                          // (whatever became of the other roles: no copy may come behind the block's end)
            for (int j = max(n_k - PP_STAGES, 0); j < n_k; ++j) t5_mbar_wait(k_full0 + 8 * (j % PP_STAGES), (uint32_t)(j / PP_STAGES) & 1u, PP_SPIN);
            for (int j = max(n_v - PP_STAGES, 0); j < n_v; ++j) t5_mbar_wait(v_full0 + 8 * (j % PP_STAGES), (uint32_t)(j / PP_STAGES) & 1u, PP_SPIN);
        }
    } else if (warp == 2) {
        // ---------------- the tensor cores' products, one thread ----------------
        if (lane == 0) {
            const uint32_t idesc_s = t5_idesc(PP_ROWS, PP_KEYS, false), idesc_o = t5_idesc(PP_ROWS, PP_HD, true);
            const uint64_t q_desc = t5_desc(t5_smem(q_smem), 16, 1024), k_desc = t5_desc(t5_smem(k_smem), 16, PP_ATOM), v_desc = t5_desc(t5_smem(v_smem), 1024, PP_ATOM);
            const auto scores = [&](int t, int j) {           // S of row tile t, key tile j
                const uint64_t qd = q_desc + (uint64_t)(t * (PP_Q_BYTES >> 4)), kd = k_desc + (uint64_t)((j % PP_STAGES) * (PP_K_BYTES >> 4));
#pragma unroll
                for (int kk = 0; kk < PP_HD / 16; ++kk)
                    t5_mma_ss(tmem + PP_COL_S + t * PP_KEYS, qd + (uint64_t)((kk >> 2) * (PP_Q_HALF >> 4) + (kk & 3) * 2), kd + (uint64_t)((kk >> 2) * (1024 >> 4) + (kk & 3) * 2), idesc_s,
                              kk > 0 ? 1u : 0u);
                t5_commit(s_full0 + 8 * t);
            };
            bool ok = t5_mbar_wait(q_full, 0, PP_SPIN);
            if (!ok) atomicExch(status, 103);
            if (ok && !(ok = t5_mbar_wait(k_full0, 0, PP_SPIN))) atomicExch(status, 104);
            if (ok) {
                t5_fence_after();
                scores(0, 0);
                if (tiles_b > 0) scores(1, 0);
                t5_commit(k_empty0);
            }
            for (int j = 0; j < n_tiles && ok; ++j) {
                const int sv = j % PP_STAGES, sk = (j + 1) % PP_STAGES;
                const uint64_t vd = v_desc + (uint64_t)(sv * (PP_K_BYTES >> 4));
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const int nt = t ? tiles_b : tiles_a;
                    if (j >= nt || !ok) continue;
                    if (!t5_mbar_wait(p_full0 + 8 * t, (uint32_t)j & 1u, PP_SPIN)) { atomicExch(status, 106); ok = false; continue; }
                    t5_fence_after();
#pragma unroll
                    for (int kk = 0; kk < PP_KEYS / 16; ++kk)         // 16 keys a product: 8 columns of P, one page of V
                        t5_mma_ts(tmem + PP_COL_O + t * PP_HD, tmem + PP_COL_S + t * PP_KEYS + kk * 8, vd + (uint64_t)(kk * (PP_PAGE_BYTES >> 4)), idesc_o, (j > 0 || kk > 0) ? 1u : 0u);
                    if (j + 1 < nt) scores(t, j + 1);
                    else t5_commit(o_done0 + 8 * t);
                }
                t5_commit(v_empty0 + 8 * sv);
                if (j + 1 < n_tiles) t5_commit(k_empty0 + 8 * sk);
            }
            if (!ok) t5_commit(drained), t5_mbar_wait(drained, 0, PP_SPIN);        // (no product may come behind the tensor memory's release)
        }
    } else if (warp == 3) {
        // ---------------- waits for K and V on behalf of the thread that issues: its arrival at P's barriers says that V(j) and K(j + 1) are there, too. (A wait costs a thread some
        // 250 clocks even when it is over already; two more of them a tile stood between the products of B and those of A.) ----------------
        if (lane == 0) {
            for (int j = 0; j < n_tiles; ++j) {
                const int sk = (j + 1) % PP_STAGES;
                if (!t5_mbar_wait(v_full0 + 8 * (j % PP_STAGES), (uint32_t)(j / PP_STAGES) & 1u, PP_SPIN)) { atomicExch(status, 105); break; }
                if (j + 1 < n_tiles && !t5_mbar_wait(k_full0 + 8 * sk, (uint32_t)((j + 1) / PP_STAGES) & 1u, PP_SPIN)) { atomicExch(status, 107); break; }
                if (j < tiles_a) t5_mbar_arrive(p_full0);
                if (j < tiles_b) t5_mbar_arrive(p_full0 + 8);
                // (one arrival a phase: the next only behind this one's end)
                if (j < tiles_a && !t5_mbar_wait(p_full0, (uint32_t)j & 1u, PP_SPIN)) { atomicExch(status, 102); break; }
                if (j < tiles_b && !t5_mbar_wait(p_full0 + 8, (uint32_t)j & 1u, PP_SPIN)) { atomicExch(status, 102); break; }
            }
        }
    } else if (warp >= 4) {
        // ---------------- softmax and output: warps 4 - 7 row tile A, 8 - 11 row tile B; a warp owns tensor-memory lanes 32 (warp % 4) .. + 31 ----------------
        const int t = (warp - 4) >> 2, qd = warp & 3, r = qd * 32 + lane, n_rows = (t ? n_b : n_a) * G, my_tiles = t ? tiles_b : tiles_a, tok = tok0 + t * tpt;
        const bool rvalid = r < n_rows;
        const int tl = rvalid ? r / G : 0, hh = rvalid ? r - tl * G : 0;
        const int rpos = rvalid ? pos0 + t * tpt + tl : -1;           // a row that is not there masks every key
        const int rlo = rvalid ? il_mask_lo(rpos, window) : 0;
        {   // Q: this row's head_dim values into the swizzled K-major tile (16-byte chunk c of row r at chunk c ^ (r % 8))
            const uint4* src = rvalid ? reinterpret_cast<const uint4*>(q + (size_t)(tok + tl) * q_stride + (size_t)(g * G + hh) * PP_HD) : nullptr;
#pragma unroll
            for (int kk = 0; kk < PP_HALVES; ++kk)
#pragma unroll
                for (int c = 0; c < 8; ++c)
                    *reinterpret_cast<uint4*>(q_smem + t * PP_Q_BYTES + kk * PP_Q_HALF + r * 128 + ((c ^ (r & 7)) << 4)) = src ? src[kk * 8 + c] : make_uint4(0u, 0u, 0u, 0u);
            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");      // the tensor core reads it through the async proxy
            __syncwarp();
            if (lane == 0) t5_mbar_arrive(q_full);
        }
        const uint32_t t_lane = tmem + ((uint32_t)(qd * 32) << 16), t_s = t_lane + PP_COL_S + t * PP_KEYS, t_o = t_lane + PP_COL_O + t * PP_HD;
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        for (int j = 0; j < my_tiles; ++j) {
            if (!t5_mbar_wait(s_full0 + 8 * t, (uint32_t)j & 1u, PP_SPIN)) { atomicExch(status, 108); ok = false; break; }
            t5_fence_after();
            const int kb = (page_first + j * PP_TILE_PAGES) * PP_PAGE;
            const bool edge = __any_sync(0xffffffffu, kb + PP_KEYS - 1 > rpos || kb < rlo);   // the tile touches a causal or window edge of some row of the warp
            // ---- the row's scores into registers, their maximum
            uint32_t sv[PP_KEYS];
#pragma unroll
            for (int c0 = 0; c0 < PP_KEYS; c0 += 32) t5_ld32(t_s + c0, sv + c0);
            t5_wait_ld();
            if (edge) {
#pragma unroll
                for (int c = 0; c < PP_KEYS; ++c) {
                    const int key = kb + c;
                    if (!(key <= rpos && key >= rlo)) sv[c] = __float_as_uint(-INFINITY);
                }
            }
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int c = 0; c < PP_KEYS; c += 8)
#pragma unroll
                for (int i = 0; i < 4; ++i) mx[i] = pp_max3(mx[i], __uint_as_float(sv[c + i]), __uint_as_float(sv[c + 4 + i]));
            const float mxs = pp_max3(pp_max3(mx[0], mx[1], mx[2]), mx[3], mx[3]) * scale_log2;        // scale > 0
            const bool raise = !(mxs <= m + PP_RAISE);        // also the first keys a row sees (m = -inf), and a NaN
            float corr = 1.f;
            if (raise) corr = pp_ex2(m - mxs), m = mxs, l *= corr;        // (0 when nothing was summed yet)
            const bool rescale = j > 0 && __any_sync(0xffffffffu, raise);
            // ---- weights, P over the scores
            const il_f2 sc = il_f2_dup(scale_log2), neg_m = il_f2_dup(m == -INFINITY ? 0.f : -m);
            il_f2 sum[2] = {il_f2_dup(0.f), il_f2_dup(0.f)};
#pragma unroll
            for (int k = 0; k < PP_KEYS / 32; ++k) {
#pragma unroll
                for (int c = 32 * k; c < 32 * k + 32; c += 2) {
                    float a, b;
                    il_f2_get(il_f2_fma(il_f2_make(__uint_as_float(sv[c]), __uint_as_float(sv[c + 1])), sc, neg_m), a, b);
                    a = pp_ex2(a), b = pp_ex2(b);
                    sum[(c >> 1) & 1] = il_f2_add(sum[(c >> 1) & 1], il_f2_make(a, b));
                    sv[c >> 1] = pp_pack(a, b);
                }
                pp_st16(t_s + 16 * k, sv + 16 * k);
            }
            if (rescale) {                        // (O holds every tile before: the scores were issued behind their products)
#pragma unroll
                for (int c0 = 0; c0 < PP_HD; c0 += 32) {
                    uint32_t ov[32];
                    t5_ld32(t_o + c0, ov);
                    t5_wait_ld();
#pragma unroll
                    for (int c = 0; c < 32; ++c) ov[c] = __float_as_uint(__uint_as_float(ov[c]) * corr);
                    t5_st32(t_o + c0, ov);
                }
            }
            float s0, s1;
            il_f2_get(il_f2_add(sum[0], sum[1]), s0, s1);
            l += s0 + s1;
            t5_wait_st();
            t5_fence_before();
            __syncwarp();
            if (lane == 0) t5_mbar_arrive(p_full0 + 8 * t);
        }
        if (my_tiles > 0 && ok) {
            ok = t5_mbar_wait(o_done0 + 8 * t, 0, PP_SPIN);
            if (!ok) atomicExch(status, 109);
            t5_fence_after();
        }
        if (my_tiles > 0 && ok) {
            const float inv = l == 0.f ? 0.f : 1.f / l;
            // The rows go out through shared memory (Q's place: every product that reads Q is through), 32 / CH rows at a time, each row's bytes contiguous.
            constexpr int CH = PP_HD / 8;                 // 16-byte chunks of a row
            unsigned char* stage = q_smem + t * PP_Q_BYTES + qd * 32 * (PP_HD * 2);
#pragma unroll
            for (int c0 = 0; c0 < PP_HD; c0 += 32) {
                uint32_t ov[32];
                t5_ld32(t_o + c0, ov);
                t5_wait_ld();
#pragma unroll
                for (int c = 0; c < 32; c += 8) {
                    uint4 v;
                    v.x = pp_pack(__uint_as_float(ov[c]) * inv, __uint_as_float(ov[c + 1]) * inv);
                    v.y = pp_pack(__uint_as_float(ov[c + 2]) * inv, __uint_as_float(ov[c + 3]) * inv);
                    v.z = pp_pack(__uint_as_float(ov[c + 4]) * inv, __uint_as_float(ov[c + 5]) * inv);
                    v.w = pp_pack(__uint_as_float(ov[c + 6]) * inv, __uint_as_float(ov[c + 7]) * inv);
                    const int ch = (c0 + c) >> 3;
                    *reinterpret_cast<uint4*>(stage + lane * (PP_HD * 2) + ((ch ^ (lane & 7)) << 4)) = v;
                }
            }
            __syncwarp();
#pragma unroll
            for (int it = 0; it < CH; ++it) {
                const int wr = it * (32 / CH) + lane / CH, ch = lane % CH, rr = qd * 32 + wr;      // row of this warp, chunk of the row
                if (rr < n_rows) {
                    const int t2 = rr / G, h2 = rr - t2 * G;
                    *reinterpret_cast<uint4*>(out + (size_t)(tok + t2) * nh * PP_HD + (size_t)(g * G + h2) * PP_HD + ch * 8) =
                        *reinterpret_cast<const uint4*>(stage + wr * (PP_HD * 2) + ((ch ^ (wr & 7)) << 4));
                }
            }
        }
    }
    t5_fence_before();
    __syncthreads();
    if (warp == 1) {
        t5_fence_after();
        t5_dealloc(tmem, 512);
    }
}

// Rows a block owns: it takes twice rows / 2 / (heads per kv head) consecutive tokens.
IL_EXPORT int il_attn_prefill_pair_rows() { return 2 * PP_ROWS; }

// Arguments as one struct, addresses and strides first. kv_map: the 128 bytes of the cache's third tensor map (il_attn_decode_kv_map), on the host.
// n_tiles_total: sum over entries [first_entry, n_entries) of ceil(q_len / (2 tpt)), tpt = rows / 2 / (nh / nkv); more than that is allowed.
struct PpArgs {
    const void* q;
    long long q_stride;
    void* out;
    const void* kv_map;
    const int *block_table, *entry_qstart, *entry_kvlen;
    int* status;
    cudaStream_t stream;
    int bt_stride, first_entry, n_entries, n_tiles_total, nh, nkv, hd, window;
    float scale;
};
static_assert(sizeof(PpArgs) == 112, "what ops.py packs, padding included");
IL_EXPORT int il_attn_prefill_pair(const PpArgs* args) {
    const auto [q, q_stride, out, kv_map, block_table, entry_qstart, entry_kvlen, status, stream, bt_stride, first_entry, n_entries, n_tiles_total, nh, nkv, hd, window, scale] = *args;
    if (n_tiles_total <= 0 || first_entry >= n_entries) return IL_OK;
    if (hd != HEAD_DIM || !kv_map || !status) return IL_UNSUPPORTED;
    if (nh <= 0 || nkv <= 0 || nh % nkv != 0 || first_entry < 0) return IL_BAD_ARG;
    const int G = nh / nkv;
    if (G > PP_ROWS || !(scale > 0.f) || (long long)n_tiles_total * nkv > 0x7fffffffLL) return IL_UNSUPPORTED;
    if ((((uintptr_t)q | (uintptr_t)out) & 15) || (q_stride & 7)) return IL_UNSUPPORTED;
    int dev = 0;
    cudaGetDevice(&dev);
    static bool attr_set[64];
    if (dev >= 0 && dev < 64 && !attr_set[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(attn_prefill_pair_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, PP_SMEM);
        if (e != cudaSuccess) return 1000 + (int)e;
        attr_set[dev] = true;
    }
    CUtensorMap map;
    memcpy(&map, kv_map, sizeof(map));
    attn_prefill_pair_kernel<<<(unsigned)(n_tiles_total * nkv), PP_THREADS, PP_SMEM, stream>>>(map, (const __nv_bfloat16*)q, q_stride, (__nv_bfloat16*)out, block_table, bt_stride, entry_qstart, entry_kvlen,
                                                                                       first_entry, n_entries, nh, nkv, scale * 1.4426950408889634f, window, PP_ROWS / G, status);
    IL_LAUNCH_CHECK();
    return IL_OK;
}
