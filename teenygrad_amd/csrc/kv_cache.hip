// The 8-bit paged K/V cache: a step's plan (pages, slots) and its writes.
//
// No counterpart in the reference, whose attention reads dense K and V
// (kernels/teeny-kernels/src/nn/attention/flash_attn2.rs:18-21); the codes
// follow teeny-quant's symmetric int8 (utilities/teeny-quant/src/quant/
// affine.rs:55-148: scale = amax / 127, zero point 0), with one group per
// (page, head) and ties to even.
//
// Pages: K [pages, heads, page_size, D], V transposed [pages, heads, D,
// page_size]: kv_attn.hip multiplies both straight from memory, and V^T's
// operand wants consecutive tokens of one d.
#include "mfma.hpp"

namespace teeny {

// ── plan ────────────────────────────────────────────────────────────────────
//
// The sums over requests (tokens, pages given back, pages needed) are prefix
// sums; everything else follows from them without a further dependency: page
// k of a step is entry avail - 1 - k of the free stack with the returned pages
// on top, and an entry at or above the old count is found in its request's
// row of the table.  So every workgroup does the sums for itself (a few KB
// that come from L2), and then its share of the tokens and pages: one launch.
// Bound by latency, the launch, two or three rounds of loads and the scans: 2.9
// us on the device for 8 requests and 8 tokens, 7.1 us for 512 requests, 13500
// tokens and 5000 pages taken or given back (9.8 with 256 threads for the sums,
// and the three kinds of work one after the other).

constexpr int kPlanMost = 4096;

struct KvPlanArgs {
  const int32_t *new_lens, *seq_lens;
  int32_t *table, *free_list;
  const int32_t *free_count;
  int32_t *q_starts, *slots, *positions, *context_lens, *granted, *free_after;
  int batch, width, pages, shift, tokens;
  int state, work;  // what this launch does: the per-request outputs; tokens, pages and the table
};

// Smallest i with cum[i] > x (cum ascending, cum[n - 1] > x).
__device__ __forceinline__ int upper(const uint32_t *cum, int n, uint32_t x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (cum[mid] > x) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

template <int THREADS>
__global__ __launch_bounds__(THREADS) void kv_plan(KvPlanArgs p) {
  constexpr int WAVES = THREADS / 64;
  __shared__ uint32_t ends[kPlanMost], backs[kPlanMost], needs[kPlanMost];  // inclusive sums
  __shared__ int32_t seqs[kPlanMost];
  __shared__ uint32_t part[2][WAVES], given_pages;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int64_t room = static_cast<int64_t>(p.width) << p.shift;  // tokens of a table row
  const uint32_t held = min(max(p.free_count[0], 0), p.pages);
  auto pages_of = [&](int64_t n) { return static_cast<uint32_t>((n + (1 << p.shift) - 1) >> p.shift); };
  // inclusive prefix sums of two values over the workgroup, behind the carries (lengths come from the caller and may
  // be anything: sums saturate)
  auto scan2 = [&](uint32_t &a, uint32_t &b, uint32_t &ca, uint32_t &cb) {
    a = wave_scan(a);
    b = wave_scan(b);
    __syncthreads();
    if (lane == 63) part[0][w] = a, part[1][w] = b;
    __syncthreads();
    uint32_t sa = ca, sb = cb;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) {
      if (i == w) {
        a = __builtin_elementwise_add_sat(a, sa);
        b = __builtin_elementwise_add_sat(b, sb);
      }
      sa = __builtin_elementwise_add_sat(sa, part[0][i]);
      sb = __builtin_elementwise_add_sat(sb, part[1][i]);
    }
    ca = sa;
    cb = sb;
  };
  // pages that request b needs, 0 if it does not fit; end: tokens up to and with it
  auto need_of = [&](int64_t nw, int64_t seq, uint32_t end, bool &fits) -> uint32_t {
    fits = nw > 0 && seq >= 0 && seq + nw <= room && end <= static_cast<uint32_t>(p.tokens);
    return fits ? pages_of(seq + nw) - pages_of(seq) : 0;
  };
  if (tid == 0) given_pages = 0;
  uint32_t all_tokens = 0, all_back = 0, all_need = 0, none = 0;
  bool fits;
  for (int b0 = 0; b0 < p.batch; b0 += THREADS) {
    const int b = b0 + tid;
    const int nw = b < p.batch ? p.new_lens[b] : 0, seq = b < p.batch ? p.seq_lens[b] : 0;
    uint32_t add = nw > 0 ? nw : 0;
    uint32_t back = nw < 0 ? pages_of(min(max(int64_t{seq}, int64_t{0}), room)) : 0;
    scan2(add, back, all_tokens, all_back);
    uint32_t need = need_of(nw, seq, add, fits), zero = 0;
    scan2(need, zero, all_need, none);
    if (b < p.batch) ends[b] = add, backs[b] = back, needs[b] = need, seqs[b] = seq;
  }
  __syncthreads();
  const uint32_t avail = min(held + min(all_back, static_cast<uint32_t>(p.pages)), static_cast<uint32_t>(p.pages));
  // whether request b, of nw new tokens, gets its pages
  auto gets = [&](int b, int nw) {
    const uint32_t need = need_of(nw, seqs[b], ends[b], fits);
    return fits && (needs[b] <= avail || need == 0);
  };
  // what the granted requests take together: the largest sum that the pool covers
  uint32_t most = 0;
  for (int b = tid; b < p.batch; b += THREADS)
    if (needs[b] <= avail) most = max(most, needs[b]);
  if (most > 0) atomicMax(&given_pages, most);
  __syncthreads();
  const uint32_t taken = given_pages;

  // entry i < avail of the stack with the returned pages on top
  auto entry = [&](uint32_t i) -> int32_t {
    if (i < held) return p.free_list[i];
    const uint32_t r = i - held;
    const int b = upper(backs, p.batch, r);
    return p.table[static_cast<int64_t>(b) * p.width + (r - (b > 0 ? backs[b - 1] : 0))];
  };
  if (p.work) {
    // the tokens, then the pages that are taken, then those that come back: all of one launch's threads at once
    const uint32_t step = gridDim.x * THREADS, to_take = p.tokens + taken, all = to_take + (avail - held);
    for (uint32_t i = blockIdx.x * THREADS + tid; i < all; i += step) {
      if (i < static_cast<uint32_t>(p.tokens)) {
        int32_t slot = -1, pos = -1;
        if (i < all_tokens) {
          const int b = upper(ends, p.batch, i);
          const uint32_t from = b > 0 ? ends[b - 1] : 0;
          const int64_t seq = seqs[b];
          if (gets(b, static_cast<int>(min(ends[b] - from, 0x7fffffffu)))) {
            pos = static_cast<int32_t>(seq) + static_cast<int32_t>(i - from);
            const uint32_t at = static_cast<uint32_t>(pos) >> p.shift, had = pages_of(seq);
            const int32_t page = at < had ? p.table[static_cast<int64_t>(b) * p.width + at]
                                          : entry(avail - 1 - ((b > 0 ? needs[b - 1] : 0) + at - had));
            // a page that is none (a table that was never filled) takes no token
            if (page >= 0 && page < p.pages) slot = (page << p.shift) + (pos & ((1 << p.shift) - 1));
          }
        }
        p.slots[i] = slot;
        p.positions[i] = pos;
      } else if (i < to_take) {
        const uint32_t k = i - p.tokens;
        const int b = upper(needs, p.batch, k);
        p.table[static_cast<int64_t>(b) * p.width + pages_of(seqs[b]) + (k - (b > 0 ? needs[b - 1] : 0))] =
            entry(avail - 1 - k);
      } else {
        const uint32_t r = held + (i - to_take);
        p.free_list[r] = entry(r);
      }
    }
  }
  if (p.state && blockIdx.x == 0) {
    // the outputs may be the inputs themselves: everything above has been read
    __syncthreads();
    for (int b = tid; b < p.batch; b += THREADS) {
      const int nw = p.new_lens[b];
      const int got = gets(b, nw) ? nw : 0;
      p.q_starts[b + 1] = static_cast<int32_t>(min(ends[b], static_cast<uint32_t>(p.tokens)));
      p.granted[b] = got;
      p.context_lens[b] = nw < 0 ? 0 : seqs[b] + got;
    }
    if (tid == 0) {
      p.q_starts[0] = 0;
      p.free_after[0] = static_cast<int32_t>(avail - taken);
    }
  }
}

// ── write ───────────────────────────────────────────────────────────────────
//
// s' = max(s, amax / 127) over a page's old and new tokens, old codes q ->
// rint(q s / s'), new ones rint(x / s').  A page's new tokens are a run of
// consecutive slots; the run's first token finds itself from the slots, and
// a team of page_size / 16 waves does the page of one head and one cache, 16
// tokens a wave, held in registers between the two passes over them.  A page
// that a run begins at its first slot forgets its old scale.  Bound by
// reading the tokens and writing the codes, and by latency for few tokens:
// 5 x 1600 tokens of 8 heads of 128 take 13.8 us (49 MB, 3.6 TB/s; 20.0 with
// a division of its own for each code), 64 requests' single tokens 5.1 us.

struct KvWriteArgs {
  const bf16 *k, *v;
  int64_t k_stride, v_stride;
  const int32_t *slots;
  int8_t *kc, *vc;
  float *ks, *vs;
  int tokens, heads, pages, shift, share;  // share: workgroups to 64 tokens, a head and a cache
};

// bits[i]: a word whose low byte is rint(x[i] / s), in -127..127, the quotient
// rounded to fp32 first as division does: x inv, inv the rounded reciprocal, and
// two corrections by the exact remainder, the last of which rounds correctly
// (Markstein, 1990).  Adding 1.5 * 2^23 rounds to an integer and leaves it in the
// low bits.  tiny: s and x were scaled up from where fp32 has fewer bits, and s
// may be too small for its largest x.
template <int N>
__device__ __forceinline__ void kv_codes(float (&x)[N], float s, float inv, bool tiny, uint32_t (&bits)[N]) {
  if (tiny)
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] *= 0x1p100f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float t = x[i] * inv;
    t = __builtin_fmaf(__builtin_fmaf(-t, s, x[i]), inv, t);
    x[i] = __builtin_fmaf(__builtin_fmaf(-t, s, x[i]), inv, t);
  }
  if (tiny)
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = fminf(fmaxf(x[i], -127.0f), 127.0f);
#pragma unroll
  for (int i = 0; i < N; ++i) bits[i] = __float_as_uint(x[i] + 12582912.0f);
}
// An old code under a larger scale: ratio = old scale / new scale.
__device__ __forceinline__ int kv_recode(int q, float ratio) {
  return static_cast<int>(__builtin_rintf(static_cast<float>(q) * ratio));
}
// The low bytes of four words.
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0c0c0400u), __builtin_amdgcn_perm(b, a, 0x0c0c0400u), 0x05040100u);
}
__device__ __forceinline__ int byte_of(uint32_t word, int i) {
  return static_cast<int8_t>((word >> (8 * i)) & 0xffu);
}

// D: head size; WPP: waves per page (page_size / 16); blockIdx.y: head, blockIdx.z: K or V.
template <int D, int WPP>
__global__ __launch_bounds__(64 * (WPP > 4 ? WPP : 4)) void kv_write(KvWriteArgs p) {
  constexpr int TEAMS = WPP > 4 ? 1 : 4 / WPP, PAGE = 16 * WPP;
  __shared__ uint32_t big[2][TEAMS][WPP];
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int team = w / WPP, part = w % WPP, head = blockIdx.y;
  const bool is_v = blockIdx.z == 1;
  // worker by worker, so that those without a run, the later ones, are not always the same XCD's
  const int chunks = (p.tokens + 63) / 64, worker = blockIdx.x / chunks, t0 = (blockIdx.x - worker * chunks) * 64;
  const int limit = p.pages << p.shift;  // slots of the cache, below 2^31

  // 64 tokens' slots and the runs that begin among them, dealt out to the workers' teams in turn
  const int mine = t0 + lane < p.tokens ? p.slots[t0 + lane] : -1;
  int before = __shfl_up(mine, 1, 64);
  if (lane == 0) before = t0 > 0 ? p.slots[t0 - 1] : -2;
  const bool leads = mine >= 0 && mine < limit && (mine % PAGE == 0 || mine != before + 1);
  const uint64_t runs = __ballot(leads);
  const int rank = __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(runs >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(runs), 0));
  const int stride = p.share * TEAMS, count = __popcll(runs);
  for (int round = 0, turn = worker * TEAMS; turn < count; ++round, turn += stride) {
    const uint64_t own = __ballot(leads && rank == turn + team);
    const bool live = own != 0;
    const int at0 = live ? __builtin_ctzll(own) : 0, first = t0 + at0;
    const int slot = live ? __builtin_amdgcn_readlane(mine, at0) : 0;
    const int page = slot / PAGE, old = slot % PAGE;
    int n = 0;  // the run's length
    if (live) {
      const uint64_t in = __ballot(lane >= at0 && lane - at0 < PAGE - old && mine == slot + lane - at0) >> at0;
      n = in == ~0ull ? 64 : __builtin_ctzll(~in);
      // past the slots at hand
      while (n < PAGE - old && at0 + n >= 64) {
        const int at = n + lane;
        const uint64_t more = __ballot(at < PAGE - old && first + at < p.tokens && p.slots[first + at] == slot + at);
        const int m = more == ~0ull ? 64 : __builtin_ctzll(~more);
        n += m;
        if (m < 64) break;
      }
    }
    const int64_t unit = static_cast<int64_t>(page) * p.heads + head;
    float *scale_at = (is_v ? p.vs : p.ks) + unit;
    const float scale0 = live && old > 0 ? *scale_at : 0.0f;
    // offsets of this wave's 16 tokens: [lo, hi) are new
    const int base = 16 * part, lo = max(old - base, 0), hi = min(old + n - base, 16);
    const bool news = live && hi > lo, whole = lo == 0 && hi == 16;
    uint32_t mx = 0;  // the largest magnitude as bf16 bits: ordered like the values, NaN above all
    constexpr int VPR = D / 8, RPI = 64 / VPR, NK = 16 / RPI;  // K: lanes per row, rows per round
    constexpr int DPL = D / 64;                                // V: d's per lane
    u32x4 kr[NK], vc[DPL];
    uint32_t vr[16];
    u32x4 *v_at = reinterpret_cast<u32x4 *>(p.vc + unit * (PAGE * D) + DPL * lane * PAGE + base);
    // (outside of [lo, hi) the nearest new token once more: it changes no maximum)
    if (news && !is_v) {
      const bf16 *src = p.k + (first + base - old) * p.k_stride + head * D + 8 * (lane % VPR);
#pragma unroll
      for (int i = 0; i < NK; ++i)
        kr[i] = *reinterpret_cast<const u32x4 *>(src + min(max(i * RPI + lane / VPR, lo), hi - 1) * p.k_stride);
#pragma unroll
      for (int i = 0; i < NK; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) mx = max(mx, max(kr[i][j] & 0x7fffu, (kr[i][j] >> 16) & 0x7fffu));
    } else if (live && is_v) {
      // bytes of other tokens stay as they are (or take the new scale)
      if (!whole)
#pragma unroll
        for (int dd = 0; dd < DPL; ++dd) vc[dd] = v_at[dd * (PAGE / 16)];
      if (news) {
        const bf16 *src = p.v + (first + base - old) * p.v_stride + head * D + DPL * lane;
#pragma unroll
        for (int o = 0; o < 16; ++o) {
          const bf16 *at = src + min(max(o, lo), hi - 1) * p.v_stride;
          if constexpr (DPL == 2) vr[o] = *reinterpret_cast<const uint32_t *>(at);
          else vr[o] = *reinterpret_cast<const uint16_t *>(at);
        }
#pragma unroll
        for (int o = 0; o < 16; ++o) mx = max(mx, max(vr[o] & 0x7fffu, (vr[o] >> 16) & 0x7fffu));
      }
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) mx = max(mx, static_cast<uint32_t>(__shfl_xor(static_cast<int>(mx), off, 64)));
    if constexpr (WPP > 1) {  // two sets in turn: a wave writes the next one at most before the last reads this one
      if (lane == 0) big[round & 1][team][part] = mx;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < WPP; ++i) mx = max(mx, big[round & 1][team][i]);
    }
    if (!live) continue;
    const float scale = __builtin_elementwise_maximum(scale0, __uint_as_float(mx << 16) / 127.0f);
    const bool fine = scale > 0.0f && scale < INFINITY;  // else every code is 0
    const bool tiny = scale < 1e-30f;
    const float div = tiny ? scale * 0x1p100f : scale, inv = fine ? 1.0f / div : 0.0f, ratio = fine ? scale0 / scale : 0.0f;
    const bool again = old > base && scale != scale0;  // old codes here, under another scale (also NaN)
    if (!is_v) {
      if (news || again) {
        u32x2 *at = reinterpret_cast<u32x2 *>(p.kc + unit * (PAGE * D) + (base + lane / VPR) * D + 8 * (lane % VPR));
#pragma unroll
        for (int i = 0; i < NK; ++i) {
          const int o = i * RPI + lane / VPR;
          u32x2 c;
          if (news && o >= lo && o < hi) {
            float x[8];
            uint32_t q[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              x[2 * j] = __uint_as_float(kr[i][j] << 16);
              x[2 * j + 1] = __uint_as_float(kr[i][j] & 0xffff0000u);
            }
            kv_codes(x, div, inv, tiny, q);
#pragma unroll
            for (int j = 0; j < 2; ++j) c[j] = fine ? pack4(q[4 * j], q[4 * j + 1], q[4 * j + 2], q[4 * j + 3]) : 0u;
            at[i * (RPI * D / 8)] = c;
          } else if (again && o < lo) {
            c = at[i * (RPI * D / 8)];
#pragma unroll
            for (int j = 0; j < 2; ++j)
              c[j] = pack4(kv_recode(byte_of(c[j], 0), ratio), kv_recode(byte_of(c[j], 1), ratio),
                           kv_recode(byte_of(c[j], 2), ratio), kv_recode(byte_of(c[j], 3), ratio));
            at[i * (RPI * D / 8)] = c;
          }
        }
      }
    } else if (news || again) {
      auto below = [](int n) { return n <= 0 ? 0u : n >= 4 ? ~0u : (1u << (8 * n)) - 1; };
      uint32_t fresh[4];  // bytes of the new tokens
#pragma unroll
      for (int j = 0; j < 4; ++j) fresh[j] = below(hi - 4 * j) & ~below(lo - 4 * j);
#pragma unroll
      for (int dd = 0; dd < DPL; ++dd) {
        u32x4 c = u32x4{0u, 0u, 0u, 0u};
        if (!whole) {
          c = vc[dd];
          if (again) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              uint32_t word = 0;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int q = byte_of(c[j], e);
                word |= (static_cast<uint32_t>(4 * j + e < lo ? kv_recode(q, ratio) : q) & 0xffu) << (8 * e);
              }
              c[j] = word;
            }
          }
        }
        if (news) {
          float x[16];
          uint32_t q[16];
#pragma unroll
          for (int o = 0; o < 16; ++o) x[o] = __uint_as_float(dd ? vr[o] & 0xffff0000u : vr[o] << 16);
          kv_codes(x, div, inv, tiny, q);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t word = fine ? pack4(q[4 * j], q[4 * j + 1], q[4 * j + 2], q[4 * j + 3]) : 0u;
            c[j] = whole ? word : (c[j] & ~fresh[j]) | (word & fresh[j]);
          }
        }
        v_at[dd * (PAGE / 16)] = c;
      }
    }
    if (part == 0 && lane == 0) *scale_at = scale;
  }
}

template <int D>
static void launch_kv_write(const KvWriteArgs &p, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(cdiv(p.tokens, 64) * p.share), static_cast<unsigned>(p.heads), 2);
  switch (p.shift) {
    case 4: hipLaunchKernelGGL((kv_write<D, 1>), grid, dim3(256), 0, s, p); break;
    case 5: hipLaunchKernelGGL((kv_write<D, 2>), grid, dim3(256), 0, s, p); break;
    case 6: hipLaunchKernelGGL((kv_write<D, 4>), grid, dim3(256), 0, s, p); break;
    default: hipLaunchKernelGGL((kv_write<D, 8>), grid, dim3(512), 0, s, p); break;
  }
}

int kv_page_shift(int64_t page_size) {
  return page_size == 16 ? 4 : page_size == 32 ? 5 : page_size == 64 ? 6 : page_size == 128 ? 7 : -1;
}

}  // namespace teeny

using namespace teeny;

extern "C" {

teeny_status teeny_kv_cache_plan(const int32_t *new_lens, const int32_t *seq_lens, int32_t *block_table,
                                 int32_t *free_list, const int32_t *free_count, int32_t *q_starts, int32_t *slots,
                                 int32_t *positions, int32_t *context_lens, int32_t *granted, int32_t *free_after,
                                 int64_t batch, int64_t max_pages, int64_t num_pages, int64_t page_size,
                                 int64_t n_tokens, teeny_stream stream) {
  const char *nm = "kv_cache_plan";
  TEENY_REQUIRE(batch >= 0 && max_pages >= 0 && num_pages >= 0 && n_tokens >= 0, TEENY_ERR_SHAPE_MISMATCH,
                "kv_cache_plan: negative size");
  TEENY_REQUIRE(batch <= kPlanMost, TEENY_ERR_SHAPE_MISMATCH, "kv_cache_plan: more than 4096 requests");
  const int shift = kv_page_shift(page_size);
  TEENY_REQUIRE(shift > 0, TEENY_ERR_UNSUPPORTED, "kv_cache_plan: page_size must be 16, 32, 64 or 128");
  TEENY_REQUIRE(num_pages <= 0x7fffffff / page_size && max_pages <= 0x7fffffff / page_size && n_tokens <= 1 << 30,
                TEENY_ERR_SHAPE_MISMATCH, "kv_cache_plan: slots or a row's tokens exceed 2^31-1, or the step's tokens 2^30");
  TEENY_REQUIRE(q_starts != nullptr && free_count != nullptr && free_after != nullptr, TEENY_ERR_NULL_POINTER,
                "kv_cache_plan: q_starts/free_count/free_after");
  TEENY_REQUIRE(batch == 0 || (new_lens != nullptr && seq_lens != nullptr && context_lens != nullptr && granted != nullptr),
                TEENY_ERR_NULL_POINTER, "kv_cache_plan: new_lens/seq_lens/context_lens/granted");
  TEENY_REQUIRE((batch == 0 || max_pages == 0 || block_table != nullptr) && (num_pages == 0 || free_list != nullptr),
                TEENY_ERR_NULL_POINTER, "kv_cache_plan: block_table/free_list");
  TEENY_REQUIRE(n_tokens == 0 || (slots != nullptr && positions != nullptr), TEENY_ERR_NULL_POINTER,
                "kv_cache_plan: slots/positions");
  hipStream_t s = static_cast<hipStream_t>(stream);
  KvPlanArgs p{new_lens, seq_lens, block_table, free_list, free_count, q_starts, slots, positions, context_lens, granted,
               free_after, static_cast<int>(batch), static_cast<int>(max_pages), static_cast<int>(num_pages), shift,
               static_cast<int>(n_tokens), 1, 1};
  // Threads for the requests' sums, workgroups for two items (tokens and pages) to a token.  How many pages come back is
  // on the device: where few tokens stand against many of them, one workgroup moves 1024 in 3 us, one round of searches
  // and loads after the other (256 requests, 256 tokens, us with 0 / 20 / 200 requests that end with 500 pages each: 5 /
  // 33 / 290).
  const int threads = batch > 256 ? 1024 : 256;
  const auto kern = batch > 256 ? kv_plan<1024> : kv_plan<256>;
  const unsigned grid = static_cast<unsigned>(
      n_tokens <= threads ? 1 : std::min<int64_t>(cdiv(2 * n_tokens, threads), device_cu_count()));
  // outputs in place of inputs that other workgroups still read: a launch of their own
  const bool in_place = context_lens == seq_lens || context_lens == new_lens || granted == new_lens ||
                        granted == seq_lens || free_after == free_count;
  if (grid > 1 && in_place) {
    p.state = 0;
    hipLaunchKernelGGL(kern, dim3(grid), dim3(threads), 0, s, p);
    p.state = 1;
    p.work = 0;
    hipLaunchKernelGGL(kern, dim3(1), dim3(threads), 0, s, p);
  } else {
    hipLaunchKernelGGL(kern, dim3(grid), dim3(threads), 0, s, p);
  }
  return after_launch(nm, s);
}

teeny_status teeny_kv_cache_write(const void *k, const void *v, const int32_t *slots, int8_t *k_cache, int8_t *v_cache,
                                  float *k_scale, float *v_scale, int64_t n_tokens, int64_t kv_heads, int64_t head_dim,
                                  int64_t num_pages, int64_t page_size, int64_t k_stride, int64_t v_stride,
                                  teeny_stream stream) {
  const char *nm = "kv_cache_write";
  TEENY_REQUIRE(n_tokens >= 0 && kv_heads >= 0 && num_pages >= 0, TEENY_ERR_SHAPE_MISMATCH,
                "kv_cache_write: negative size");
  TEENY_REQUIRE(head_dim == 64 || head_dim == 128, TEENY_ERR_UNSUPPORTED, "kv_cache_write: head_dim must be 64 or 128");
  const int shift = kv_page_shift(page_size);
  TEENY_REQUIRE(shift > 0, TEENY_ERR_UNSUPPORTED, "kv_cache_write: page_size must be 16, 32, 64 or 128");
  // (a launch has less than 2^32 threads: 2^27 / 64 * 2 workgroups of 512 at most)
  TEENY_REQUIRE(num_pages <= 0x7fffffff / page_size && n_tokens <= 1 << 27 && kv_heads <= 65535,
                TEENY_ERR_SHAPE_MISMATCH, "kv_cache_write: slots exceed 2^31-1, tokens 2^27 or kv_heads 65535");
  if (n_tokens == 0 || kv_heads == 0 || num_pages == 0) return TEENY_OK;
  TEENY_REQUIRE(k != nullptr && v != nullptr && slots != nullptr && k_cache != nullptr && v_cache != nullptr &&
                    k_scale != nullptr && v_scale != nullptr,
                TEENY_ERR_NULL_POINTER, "kv_cache_write: k/v/slots/cache/scale");
  TEENY_REQUIRE(k_stride >= kv_heads * head_dim && v_stride >= kv_heads * head_dim, TEENY_ERR_SHAPE_MISMATCH,
                "kv_cache_write: token strides below kv_heads * head_dim");
  TEENY_REQUIRE(aligned(k, 16) && aligned(v, 16) && aligned(k_cache, 16) && aligned(v_cache, 16) && k_stride % 8 == 0 &&
                    v_stride % 8 == 0,
                TEENY_ERR_MISALIGNED, "kv_cache_write: 16-byte aligned tensors and token strides");
  hipStream_t s = static_cast<hipStream_t>(stream);
  KvWriteArgs p{static_cast<const bf16 *>(k), static_cast<const bf16 *>(v), k_stride, v_stride, slots, k_cache, v_cache,
                k_scale, v_scale, static_cast<int>(n_tokens), static_cast<int>(kv_heads), static_cast<int>(num_pages),
                shift,
                // 64 tokens are between one page and 64 of them, which only the device knows.  8 heads of 128, us with
                // 1 / 2 / 4 / 8 / 16 workgroups: 5 prompts of 1600 tokens 15.6 / 14.6 / 16.4 / 19.5 / 25.8, one of 500
                // 6.5 / 5.4 / 5.3 / 6.2 / 6.8; single tokens of 64 requests (pages of 16) 34 / 18 / 10.4 / 6.3 / 5.7, of
                // 500 36 / 20 / 12.8 / 10.0 / 10.1, of 2000 (heads of 64) 36 / 25 / 24 / 23 / 24
                n_tokens <= 256 ? 16 : n_tokens <= 1024 ? 8 : 2};
  if (head_dim == 64) launch_kv_write<64>(p, s);
  else launch_kv_write<128>(p, s);
  return after_launch(nm, s);
}

}  // extern "C"
