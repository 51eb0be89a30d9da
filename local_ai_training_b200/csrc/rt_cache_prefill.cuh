// rt_cache_prefill.cuh — attention of many query rows over the paged int8 cache (prompts and pieces of
// prompts): the mathematics and the work split of rt_cache_attn.cuh with tiles of 256 rows x 128 keys
// on tcgen05.
//
// 2 · D operations of each product per (row, key) on the tensor pipe and one exponential per score
// bound it: a 256 x 128 step is 2048 cycles of tcgen05 bf16 at D = 128 and 2048 cycles of the
// exponential unit (16 a cycle and SM), so the two row tiles of 128 take turns: while one's scores
// are in its softmax warps, the other's products run.
//   warps 0-3 / 4-7  softmax of row tile A / B, one row per thread (its TMEM lane): scores from tensor
//                    memory, running maximum, weights back to tensor memory as bf16 over the scores
//   warps 8-11       codes from the pages -> bf16 (exact) -> shared memory in the 128-byte swizzle
//   warp 12          one thread issues S = Q K^T (both from shared memory) and O += P V (P from
//                    tensor memory); completion by tcgen05.commit
// The block scales are folded into the scores and the weights (a factor per 16 keys).  The weight
// 2^(t - m)·sv is rounded to bf16 (bf16 queries only; the sum of weights keeps 32 bits).  The running
// maximum moves, and O is rescaled, only when a score exceeds it by 2^8.
#pragma once

#include "rt_cache_attn.cuh"

namespace rt {

// D[tmem] (+)= A[tmem] * B[smem desc], kind::f16.
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc,
                                            uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_32x32b_x32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]),
      "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
      "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

template <int D>
struct KpShape {
  static constexpr int ROWS = 128, RT = 2 * ROWS, KEYS = 128;
  static constexpr int SUB = 128 * 128;          // bytes of 128 rows x 64 bf16, 128-byte swizzle
  static constexpr int SUBS = D / 64;
  static constexpr int TILE = SUB * SUBS;        // a K, V or Q tile
  static constexpr int STAGES = 2;
  static constexpr int SCALES = 4;               // ring of the block factors
  static constexpr int Q_OFF = 0, K_OFF = 2 * TILE, V_OFF = K_OFF + STAGES * TILE;
  static constexpr int F_OFF = V_OFF + STAGES * TILE;
  static constexpr int BAR_OFF = F_OFF + SCALES * 80;
  // one CTA per SM: each takes all 512 columns of tensor memory
  static constexpr int SMEM_USED = BAR_OFF + 256 + 1024;
  static constexpr int SMEM = SMEM_USED > 120 * 1024 ? SMEM_USED : 120 * 1024;
  static constexpr int THREADS = 13 * 32;
  static constexpr uint32_t COL_S = 0, COL_O = 256;  // + 128 (scores) or + D (outputs) for row tile B
  static constexpr uint32_t IDESC_QK = (1u << 4) | (1u << 7) | (1u << 10) | ((KEYS >> 3) << 17) | ((ROWS >> 4) << 24);
  static constexpr uint32_t IDESC_PV =
      (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((D >> 3) << 17) | ((ROWS >> 4) << 24);
};
struct KpBars {
  uint64_t q_ready, k_full[2], k_empty[2], v_full[2], v_empty[2], f_full[4], s_full[2], p_ready[2], o_done[2];
  uint32_t tmem;
};
static_assert(sizeof(KpBars) <= 256, "KpBars");
struct KpFactors {  // one tile's block factors
  float k[8], v[8];
  uint32_t blocks;  // bit i: block i has a page
};

// four int8 -> four bf16
__device__ __forceinline__ uint2 bf16x4_of_bytes(uint32_t w) {
  return make_uint2(bf16x2_of_bytes<false>(w), bf16x2_of_bytes<true>(w));
}

template <int D>
__global__ void __launch_bounds__(KpShape<D>::THREADS, 1)
    kv_prefill_kernel(KvCache c, KvBatch bt, KvAttn a, int min_blocks) {
  using SH = KpShape<D>;
  using Walk = KvWalk<SH::RT, SH::KEYS>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  KpBars *bar = reinterpret_cast<KpBars *>(smem + SH::BAR_OFF);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) {
    mbar_init(&bar->q_ready, 256);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar->k_full[i], 128), mbar_init(&bar->k_empty[i], 1);
      mbar_init(&bar->v_full[i], 128), mbar_init(&bar->v_empty[i], 1);
      mbar_init(&bar->s_full[i], 1), mbar_init(&bar->p_ready[i], 128), mbar_init(&bar->o_done[i], 1);
    }
    for (int i = 0; i < 4; ++i) mbar_init(&bar->f_full[i], 1);
    fence_barrier_init();
  }
  if (warp == 12) {
    tmem_alloc(&bar->tmem, 512);
    tmem_relinquish();
  }
  pdl_wait();
  kv_zero_rest<__nv_bfloat16>(bt, a);
  Walk w;
  const bool busy = kv_walk_start<SH::THREADS>(w, c, bt, a, min_blocks);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_trigger();  // the next kernel comes up only now that this one has its tensor memory
  if (!busy) {
    if (tid == 0) a.meta[blockIdx.x] = make_int4(-1, 0, 0, 0);
    if (warp == 12) tmem_dealloc(bar->tmem, 512);
    return;
  }
  const uint32_t tmem = bar->tmem;

  // tiles [w.b, count) of the piece that row tile x has keys in, counted from the unit's beginning
  const auto tiles_of = [&](int x) {
    const int row0 = w.tile * SH::RT + x * SH::ROWS, rows = w.q.n * a.group;
    if (row0 >= rows) return w.b;
    const int nb = max((w.seen(a, min(row0 + SH::ROWS, rows)) + SH::KEYS - 1) / SH::KEYS, 1);
    return max(min(nb, w.e), w.b);
  };

  if (warp < 8) {
    // ================================================================ softmax of row tile x
    const int x = warp >> 2, r = tid & 127;  // r: row of the tile, TMEM lane
    const uint32_t t_s = tmem + SH::COL_S + x * 128 + (static_cast<uint32_t>(warp & 3) << 21);
    const uint32_t t_o = tmem + SH::COL_O + x * D + (static_cast<uint32_t>(warp & 3) << 21);
    uint32_t n_q = 0, n_s = 0, n_o = 0, n_f = 0;  // phases of q_ready, s_full, o_done; tiles of the CTA
    bool ok = true, first_piece = true;
    const bool flip = a.scale_log2 < 0.0f;  // the factors are kept >= 0 (maxima): q takes the sign
    while (w.left > 0) {
      const int row0 = w.tile * SH::RT + x * SH::ROWS, all = w.q.n * a.group;
      const int rows = max(min(SH::ROWS, all - row0), 0);
      // ---- Q tile, rows beyond the unit as zeros
      {
        constexpr int CH = D / 8;  // 16-byte chunks of a row
        uint8_t *qt = smem + SH::Q_OFF + x * SH::TILE;
#pragma unroll 4
        for (int i = 0; i < CH; ++i) {
          const int id = i * 128 + r, qr = id / CH, ch = id % CH;
          uint4 v = make_uint4(0, 0, 0, 0);
          if (qr < rows) {
            const int row = row0 + qr;
            const __nv_bfloat16 *qp = static_cast<const __nv_bfloat16 *>(a.q) +
                                      (w.q.c0 + static_cast<int64_t>(row / a.group)) * a.q_token +
                                      static_cast<int64_t>(w.head * a.group + row % a.group) * a.q_head;
            if (a.q_vec) {
              v = *reinterpret_cast<const uint4 *>(qp + ch * 8);
            } else {
              uint32_t u[8];
#pragma unroll
              for (int k = 0; k < 8; ++k)
                u[k] = ch * 8 + k < a.head_dim
                           ? *reinterpret_cast<const uint16_t *>(qp + ch * 8 + k)
                           : 0u;
              v = make_uint4(u[0] | u[1] << 16, u[2] | u[3] << 16, u[4] | u[5] << 16, u[6] | u[7] << 16);
            }
            if (flip) v.x ^= 0x80008000u, v.y ^= 0x80008000u, v.z ^= 0x80008000u, v.w ^= 0x80008000u;
          }
          *reinterpret_cast<uint4 *>(qt + (ch >> 3) * SH::SUB + qr * 128 + (((ch & 7) ^ (qr & 7)) << 4)) = v;
        }
        fence_proxy_async_smem();
        tc_fence_before();
        mbar_arrive(&bar->q_ready);
        // (also keeps a row tile without rows from running a piece ahead of the other)
        ok = __all_sync(0xffffffffu, mbar_wait(&bar->q_ready, n_q & 1));
        ++n_q;
      }
      const int end = tiles_of(x);
      const int tok = (row0 + min(r, max(rows - 1, 0))) / a.group;
      const int lim = min(w.q.start + tok + 1, w.q.len);  // keys this row sees
      float m = -1e30f, l = 0.0f;
      for (int j = w.b; j < end && ok; ++j) {
        const uint32_t f_at = n_f + static_cast<uint32_t>(j - w.b);
        ok = __all_sync(0xffffffffu, mbar_wait(&bar->f_full[f_at & 3], (f_at >> 2) & 1) &&
                                         mbar_wait(&bar->s_full[x], n_s & 1));
        if (!ok) break;
        ++n_s;
        tc_fence_after();
        const KpFactors *f = reinterpret_cast<const KpFactors *>(smem + SH::F_OFF + (f_at & 3) * 80);
        const int seen = lim - j * SH::KEYS;  // keys of this tile the row sees
        const uint32_t blocks = f->blocks;
        const bool cut = __any_sync(0xffffffffu, seen < SH::KEYS) || blocks != 0xFFu;
        const auto hidden = [&](int col) { return col >= seen || ((blocks >> (col >> 4)) & 1) == 0; };
        // ---- the tile's maximum
        float top = -INFINITY;
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          uint32_t s[32];
          tmem_ld_32x32b_x32(t_s + h * 32, s);
          tmem_ld_wait_regs(s);
          if (cut) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (hidden(h * 32 + i)) s[i] = 0xFF800000u;  // -inf
          }
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            float v = __uint_as_float(s[b * 16]);
#pragma unroll
            for (int i = 1; i < 16; ++i) v = fmaxf(v, __uint_as_float(s[b * 16 + i]));
            top = fmaxf(top, v * f->k[h * 2 + b]);
          }
        }
        if (__any_sync(0xffffffffu, top > m + 8.0f)) {
          const float mn = fmaxf(m, top), g = ex2(m - mn);
          m = mn;
          l *= g;
          if (j > w.b) {
            // the products so far have been added up; the next ones wait for this tile's weights
            ok = __all_sync(0xffffffffu, mbar_wait(&bar->o_done[x], (n_o + 1) & 1));
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int h = 0; h < D / 32; ++h) {
              uint32_t o[32];
              tmem_ld_32x32b_x32(t_o + h * 32, o);
              tmem_ld_wait_regs(o);
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * g);
              tmem_st_32x32b_x32(t_o + h * 32, o);
            }
          }
        }
        // ---- weights
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          uint32_t s[32], p[16];
          tmem_ld_32x32b_x32(t_s + h * 32, s);
          tmem_ld_wait_regs(s);
#pragma unroll
          for (int i = 0; i < 32; ++i)
            s[i] = __float_as_uint(fmaf(__uint_as_float(s[i]), f->k[h * 2 + (i >> 4)], -m));
          if (cut) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (hidden(h * 32 + i)) s[i] = 0xFF800000u;
          }
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const float p0 = ex2(__uint_as_float(s[i])), p1 = ex2(__uint_as_float(s[i + 1]));
            const float fv = f->v[h * 2 + (i >> 4)];
            l += p0 + p1;
            p[i / 2] = pack_bf16x2(p0 * fv, p1 * fv);
          }
          tmem_st_32x32b_x16(t_s + h * 16, p);
        }
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&bar->p_ready[x]);
        ++n_o;  // phases of o_done that will have completed when this tile's products are in
      }
      // ---- the piece's rows
      const bool whole = w.b == 0 && w.e == w.nb;
      if (ok && end > w.b) {
        ok = __all_sync(0xffffffffu, mbar_wait(&bar->o_done[x], (n_o + 1) & 1));
        tc_fence_after();
      }
      if (ok) {
        const int slot = blockIdx.x * 2 + (w.b > 0 ? 0 : 1);
        const int row = row0 + r;
        const float inv = l > 0.0f ? __fdividef(1.0f, l) : 0.0f;
        float *ws = a.ws + (static_cast<int64_t>(slot) * SH::RT + x * SH::ROWS + r) * (D + 2);
        __nv_bfloat16 *op = static_cast<__nv_bfloat16 *>(a.out) +
                            (w.q.c0 + static_cast<int64_t>(row / a.group)) * a.o_token +
                            static_cast<int64_t>(w.head * a.group + row % a.group) * a.o_head;
#pragma unroll
        for (int h = 0; h < D / 32; ++h) {
          uint32_t o[32];
          if (end > w.b) {
            tmem_ld_32x32b_x32(t_o + h * 32, o);
            tmem_ld_wait_regs(o);
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = 0;
          }
          if (r >= rows) {
          } else if (!whole) {
#pragma unroll
            for (int i = 0; i < 32; i += 2)
              *reinterpret_cast<uint2 *>(ws + 2 + h * 32 + i) = make_uint2(o[i], o[i + 1]);
          } else if (a.o_vec) {
#pragma unroll
            for (int i = 0; i < 32; i += 8) {
              uint32_t u[4];
#pragma unroll
              for (int k = 0; k < 4; ++k)
                u[k] = pack_bf16x2(__uint_as_float(o[i + 2 * k]) * inv, __uint_as_float(o[i + 2 * k + 1]) * inv);
              *reinterpret_cast<uint4 *>(op + h * 32 + i) = make_uint4(u[0], u[1], u[2], u[3]);
            }
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (h * 32 + i < a.head_dim) op[h * 32 + i] = __float2bfloat16_rn(__uint_as_float(o[i]) * inv);
          }
          __syncwarp();
        }
        if (!whole && r < rows) ws[0] = m, ws[1] = l;
        tc_fence_before();
      }
      if (tid == 0) {
        int4 *mt = a.meta + blockIdx.x;
        if (first_piece) *mt = make_int4(-1, 0, 0, 0);
        if (w.b > 0) mt->w = w.e == w.nb;
        if (w.b == 0 && !whole) mt->x = w.s, mt->y = w.tile, mt->z = w.head;
      }
      first_piece = false;
      n_f += static_cast<uint32_t>(w.e - w.b);
      if (!ok) break;
      w.next(c, bt, a);
    }
  } else if (warp < 12) {
    // ================================================================ codes -> bf16 tiles
    // Thread t takes 16-byte piece t % P of row t / P of each 16-token block (P pieces a row, 2 blocks
    // a pass at D = 64); a block's page is looked up once per tile.
    const int t = tid - 256;
    constexpr int P = D / 16, RPI = 128 / P, N = SH::KEYS / RPI;  // pieces, rows a pass, passes
    const int prow = t / P, pcol = t % P;
    const float fscale = fabsf(a.scale_log2);
    uint32_t n = 0;
    bool ok = true;
    const int64_t part = static_cast<int64_t>(c.kv_heads) * c.page_size * D;
    Walk ld = w;     // the tile whose codes are fetched next
    int ld_j = ld.b;
    uint4 raw[2][N];
    float fk = 0.0f, fv = 0.0f;  // thread t < 8: factors of block t
    bool has = false;
    const auto fetch = [&] {
      if (ld.left <= 0) return;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int row = i * RPI + prow, blk = ld_j * 8 + (row >> 4);
        raw[0][i] = raw[1][i] = make_uint4(0, 0, 0, 0);
        const int64_t page = blk * KV_BLOCK < ld.q.len ? kv_page(c, bt, ld.s, blk) : -1;
        if (page >= 0) {
          const int8_t *kp = c.block(page, 0, ld.head, blk & ((c.page_size >> 4) - 1)) + (row & 15) * D + pcol * 16;
          raw[0][i] = *reinterpret_cast<const uint4 *>(kp);
          raw[1][i] = *reinterpret_cast<const uint4 *>(kp + part);
        }
      }
      if (t < 8) {
        const int blk = ld_j * 8 + t;
        const int64_t page = blk * KV_BLOCK < ld.q.len ? kv_page(c, bt, ld.s, blk) : -1;
        has = page >= 0;
        fk = has ? *c.scale(page, 0, ld.head, blk & ((c.page_size >> 4) - 1)) * fscale : 0.0f;
        fv = has ? *c.scale(page, 1, ld.head, blk & ((c.page_size >> 4) - 1)) : 0.0f;
      }
      if (++ld_j >= ld.e) {
        ld.next(c, bt, a);
        ld_j = ld.b;
      }
    };
    const auto put = [&](uint8_t *tile, const uint4 (&v)[N]) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int row = i * RPI + prow;
        const uint2 b0 = bf16x4_of_bytes(v[i].x), b1 = bf16x4_of_bytes(v[i].y);
        const uint2 b2 = bf16x4_of_bytes(v[i].z), b3 = bf16x4_of_bytes(v[i].w);
        uint8_t *at = tile + (pcol >> 2) * SH::SUB + row * 128;
        const int ch = (pcol & 3) * 2;
        const uint4 lo = make_uint4(b0.x, b0.y, b1.x, b1.y), hi = make_uint4(b2.x, b2.y, b3.x, b3.y);
        // lanes of the second sub-tile store their halves in the other order: no bank is hit twice
        const bool sw = pcol & 4;
        *reinterpret_cast<uint4 *>(at + (((ch + sw) ^ (row & 7)) << 4)) = sw ? hi : lo;
        *reinterpret_cast<uint4 *>(at + (((ch + 1 - sw) ^ (row & 7)) << 4)) = sw ? lo : hi;
      }
    };
    fetch();
    while (w.left > 0 && ok) {
      for (int j = w.b; j < w.e; ++j, ++n) {
        const int st = n & 1;
        const uint32_t free_parity = ((n >> 1) & 1) ^ 1;  // a fresh barrier passes for its first use
        if (warp == 8) {
          KpFactors *f = reinterpret_cast<KpFactors *>(smem + SH::F_OFF + (n & 3) * 80);
          // the slot's last readers are past: tile n - 2's scores, complete here, were issued after the
          // softmax of tile n - 3, and the slot held tile n - 4
          ok = __all_sync(0xffffffffu, mbar_wait(&bar->k_empty[st], free_parity));
          const uint32_t blocks = __ballot_sync(0xffffffffu, has) & 0xFFu;
          if (lane < 8) f->k[lane] = fk, f->v[lane] = fv;
          if (lane == 0) f->blocks = blocks;
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar->f_full[n & 3]);
        } else if (!mbar_wait(&bar->k_empty[st], free_parity)) {
          ok = false;
        }
        if (!ok) break;
        put(smem + SH::K_OFF + st * SH::TILE, raw[0]);
        fence_proxy_async_smem();
        mbar_arrive(&bar->k_full[st]);
        if (!mbar_wait(&bar->v_empty[st], free_parity)) {
          ok = false;
          break;
        }
        put(smem + SH::V_OFF + st * SH::TILE, raw[1]);
        fence_proxy_async_smem();
        mbar_arrive(&bar->v_full[st]);
        fetch();
      }
      w.next(c, bt, a);
    }
  } else {
    if (lane == 0) {
    // ================================================================ MMA issue
    const uint32_t q0 = smem_u32(smem + SH::Q_OFF), k0 = smem_u32(smem + SH::K_OFF), v0 = smem_u32(smem + SH::V_OFF);
    uint32_t n = 0, n_q = 0, n_p[2] = {0, 0};
    bool ok = true;
    const auto qk = [&](int x, uint32_t tile) {
      tc_fence_after();
      const uint32_t qa = q0 + x * SH::TILE, ka = k0 + (tile & 1) * SH::TILE;
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
        umma_f16(tmem + SH::COL_S + x * 128, make_sw128_desc(qa + (i >> 2) * SH::SUB + (i & 3) * 32, 16, 1024),
                 make_sw128_desc(ka + (i >> 2) * SH::SUB + (i & 3) * 32, 16, 1024), SH::IDESC_QK, i > 0);
      umma_commit(&bar->s_full[x]);
    };
    const auto pv = [&](int x, uint32_t tile, bool fresh) {
      tc_fence_after();
      const uint32_t va = v0 + (tile & 1) * SH::TILE;
#pragma unroll
      for (int i = 0; i < SH::KEYS / 16; ++i)
        umma_f16_ts(tmem + SH::COL_O + x * D, tmem + SH::COL_S + x * 128 + i * 8,
                    make_sw128_desc(va + i * 2048, SH::SUB, 1024), SH::IDESC_PV, !fresh || i > 0);
      umma_commit(&bar->o_done[x]);
    };
    while (w.left > 0 && ok) {
      const int end[2] = {tiles_of(0), tiles_of(1)};
      ok = mbar_wait(&bar->q_ready, n_q & 1) && mbar_wait(&bar->k_full[n & 1], (n >> 1) & 1);
      ++n_q;
      if (!ok) break;
      for (int x = 0; x < 2; ++x)
        if (end[x] > w.b) qk(x, n);
      umma_commit(&bar->k_empty[n & 1]);
      for (int j = w.b; j < w.e && ok; ++j, ++n) {
        ok = mbar_wait(&bar->v_full[n & 1], (n >> 1) & 1);
        const bool more = j + 1 < w.e;
        for (int x = 0; x < 2 && ok; ++x) {
          if (j < end[x]) {
            ok = mbar_wait(&bar->p_ready[x], n_p[x] & 1);
            ++n_p[x];
            if (!ok) break;
            pv(x, n, j == w.b);
          }
          if (x == 1) umma_commit(&bar->v_empty[n & 1]);
          if (more && j + 1 < end[x]) {
            ok = mbar_wait(&bar->k_full[(n + 1) & 1], ((n + 1) >> 1) & 1);
            if (ok) qk(x, n + 1);
          }
        }
        if (more && ok) umma_commit(&bar->k_empty[(n + 1) & 1]);
      }
      if (ok) w.next(c, bt, a);
    }
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 12) tmem_dealloc(tmem, 512);
}

}  // namespace rt
