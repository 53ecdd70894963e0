// Keys and values in 8 bits: rotary positions, writing into a quantized cache and reading it back, attention of new
// tokens over it, the accepted drafts' move.  Declarations: include/marian_hip_ops.h
#include "../../include/marian_hip_ops.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "../../include/marian_hip_int8.h"
#include "abi_common.h"
#include "cache_args.h"
#include "cache_attention.h"
#include "cache_codes.h"
#include "cache_plan.h"

using namespace marian_hip;

namespace {

// ---------------------------------------------------------------- rotary positions
// A pair's angle in half turns, -1 .. 1: position times turns mod 2^64 is the fraction of a turn exactly.
__device__ __forceinline__ float half_turns(long long position, unsigned long long turns) {
  const long long f = (long long)(turns * (unsigned long long)position);
  return __builtin_fmaf((float)(unsigned)f, 0x1p-63f, (float)(int)(f >> 32) * 0x1p-31f);
}

// A thread turns one unit - four pairs, or eight values behind the turned ones - of up to HEADS heads of a position: the
// angles are the same for all of them.  Units of a row are side by side, then heads, then positions.
// out = x turned, in float32 with the angle's fraction of a turn exact: the error does not grow with the position.  (The fraction is rounded to 24
// bits ahead of sine and cosine: float32 results are off by 4.9e-8 of their norm, where angles in 64 bits leave 4.3e-8.)
// Memory bounds it: 4 sequences of 4093 positions, 32 heads of 128 values, bfloat16, 54 us, 5.0 TB/s (a copy: 5.1); a single token's 2.3 us are a
// launch's.
template <typename T, int HEADS>
__global__ __launch_bounds__(256) void rotary_kernel(const T* x, Strides xs, T* out, Strides os, const int* __restrict__ positions, int each,
                                                     const unsigned long long* __restrict__ turns, int dims, float magnitude, int interleaved,
                                                     int heads, int n, int dk) {
  const int units = dk / 8, groups = (heads + HEADS - 1) / HEADS;
  const unsigned id = blockIdx.x * 256u + threadIdx.x;
  const int u = id % units, hg = id / units % groups, i = id / units / groups, s = blockIdx.y;
  if(i >= n) return;
  const bool turned = 8 * u < dims;
  const long long at = each ? positions[(long long)s * n + i] : (long long)positions[s] + i;
  const int d0 = turned && !interleaved ? 4 * u : 8 * u, d1 = turned && !interleaved ? dims / 2 + 4 * u : 8 * u + 4;
  x += s * xs.s + i * xs.n;
  out += s * os.s + i * os.n;
  float a[HEADS][4], b[HEADS][4];
#pragma unroll
  for(int j = 0; j < HEADS; ++j) {
    const int h = hg + j * groups;
    if(h < heads) {
      load_row<4>(x + h * xs.h + d0, a[j]);
      load_row<4>(x + h * xs.h + d1, b[j]);
    }
  }
  float c[4], sn[4];
  if(turned) {
#pragma unroll
    for(int p = 0; p < 4; ++p) {
      sincospif(half_turns(at, turns[4 * u + p]), &sn[p], &c[p]);
      c[p] *= magnitude;
      sn[p] *= magnitude;
    }
  }
#pragma unroll
  for(int j = 0; j < HEADS; ++j) {
    const int h = hg + j * groups;
    if(h >= heads) break;
    if(turned) {
      auto turn = [&](float& va, float& vb, int p) __attribute__((always_inline)) {
        const float ra = __builtin_fmaf(va, c[p], -(vb * sn[p])), rb = __builtin_fmaf(va, sn[p], vb * c[p]);
        va = ra;
        vb = rb;
      };
      if(interleaved) {
        turn(a[j][0], a[j][1], 0);
        turn(a[j][2], a[j][3], 1);
        turn(b[j][0], b[j][1], 2);
        turn(b[j][2], b[j][3], 3);
      } else {
#pragma unroll
        for(int p = 0; p < 4; ++p) turn(a[j][p], b[j][p], p);
      }
    }
    store_row<4, T>(out + h * os.h + d0, a[j]);
    store_row<4, T>(out + h * os.h + d1, b[j]);
  }
}

// ---------------------------------------------------------------- writing
struct AppendArgs {
  unsigned char *k, *v;
  float *ks, *vs;
  const int *lens, *counts, *parents;
  const unsigned long long* turns;
  double magnitude;
  Strides kx, vx, qx, qo;
  int dims, interleaved, heads, q_heads, n, cap, dk;
};

// A row - a head's key, value or query of one token - to LANES lanes, eight values each; a workgroup takes 256 / LANES
// rows at a time of up to TOKENS tokens, whose sines and cosines its threads make first (in 64 bits: keys are
// rounded once to float32 and then quantized, so that a key next to a border of a code falls on its own side).
//   scale = largest magnitude of the row / 127 (448), code = value / scale rounded to the nearest, ties to even.
// A row's lanes are side by side, its largest value a few exchanges away; a value and the one it is turned with are both loaded, the second
// from a cache, in place of an exchange.  3 sequences of 2731 tokens, 32 + 8 + 8 heads of 128 values, float16 to e4m3: 50 us,
// 3.7 TB/s.  Without a rotation they take 36, as a copy of these bytes does, so turning is what the rest goes to: angles made by each of the three
// workgroups that share a token, ahead of its rows' loads, and turns in 64 bits, of queries like keys (in 32 bits, which would move codes of keys
// at borders, 4 us less).  128 sequences' single tokens, 48 heads of 64 values, float32: 4.4 us, 3.8 without a rotation, one step after the
// other, where a launch alone takes 2.3.
template <typename T, CacheFormat F, int LANES, int TOKENS>
__global__ __launch_bounds__(256) void append_kernel(const T* k, const T* v, const T* q, T* q_out, AppendArgs a) {
  constexpr int kRows = 256 / LANES;
  __shared__ double2 turn[TOKENS][LANES * 4];
  __shared__ int stands[64];   // tokens of a tree: how many they descend from
  const int tid = threadIdx.x, s = blockIdx.z, first = blockIdx.y * TOKENS;
  const int len = clamp_int(a.lens[s], 0, a.cap), count = a.counts ? clamp_int(a.counts[s], 0, a.n) : a.n;
  const int tokens = min(TOKENS, a.n - first), half = a.dims / 2;
  if(a.dims) {
    if(a.parents) {
      if(tid < 64) stands[tid] = __popcll(lineage(a.parents + (long long)s * a.n, a.n, tid)) - 1;
      __syncthreads();
    }
    for(int i = tid; i < tokens * half; i += 256) {
      const int t = i / half, p = i - t * half, token = first + t;
      const long long at = (long long)len + (a.parents ? stands[token] : token);
      const long long f = (long long)(a.turns[p] * (unsigned long long)at);
      double sn, c;
      sincospi((double)f * 0x1p-63, &sn, &c);
      turn[t][p] = double2{c * a.magnitude, sn * a.magnitude};
    }
    __syncthreads();
  }
  const int lane = tid % LANES, all = 2 * a.heads + a.q_heads, row = blockIdx.x * kRows + tid / LANES;
  const int d = 8 * lane;
  const bool there = row < all && d < a.dk;
  const int what = row < a.heads ? 0 : row < 2 * a.heads ? 1 : 2, h = there ? row - what * a.heads : 0;
  const Strides& st = what == 0 ? a.kx : what == 1 ? a.vx : a.qx;
  const T* const x = (!there || what == 0 ? k : what == 1 ? v : q) + s * (there ? st.s : a.kx.s) + h * st.h + (there ? d : 0);
  const long long step = there ? st.n : a.kx.n;
  // Halves: where the values that the lane's two fours are turned with lie (a four beyond the turned ones: itself).
  int other[2];
#pragma unroll
  for(int quad = 0; quad < 2; ++quad) {
    const int e = 4 * quad;
    other[quad] = e + (d + e < half ? half : d + e < a.dims ? -half : 0);
    if(!there || a.interleaved || what == 1) other[quad] = e;
  }
  // All tokens are asked for at once.
  float y[TOKENS][8], z[TOKENS][2][4];
#pragma unroll
  for(int t = 0; t < TOKENS; ++t) {
    const T* const in = x + min(first + t, a.n - 1) * step;
    load_row<8>(in, y[t]);
#pragma unroll
    for(int quad = 0; quad < 2; ++quad) load_row<4>(in + other[quad], z[t][quad]);
  }
#pragma unroll
  for(int t = 0; t < TOKENS; ++t) {
    const int token = first + t, slot = len + token;
    if(t && token >= a.n) break;
    const bool kept = token < count && (what == 2 || slot < a.cap);
    if(what != 1) {
#pragma unroll
      for(int quad = 0; quad < 2; ++quad) {
        const int e = 4 * quad;
        if(d + e >= a.dims) continue;
        if(a.interleaved) {
#pragma unroll
          for(int p = 0; p < 2; ++p) {
            const double2 w = turn[t][(d + e) / 2 + p];
            const double va = y[t][e + 2 * p], vb = y[t][e + 2 * p + 1];
            y[t][e + 2 * p] = (float)__builtin_fma(va, w.x, -(vb * w.y));
            y[t][e + 2 * p + 1] = (float)__builtin_fma(va, w.y, vb * w.x);
          }
        } else {
          const bool upper = d + e >= half;   // (its sine counts the other way)
#pragma unroll
          for(int p = 0; p < 4; ++p) {
            const double2 w = turn[t][d + e - (upper ? half : 0) + p];
            const double mine = y[t][e + p], its = z[t][quad][p];
            y[t][e + p] = (float)__builtin_fma(mine, w.x, its * (upper ? w.y : -w.y));
          }
        }
      }
    }
    if(what == 2) {
      if(there && token < a.n) {
        float out[8];
#pragma unroll
        for(int e = 0; e < 8; ++e) out[e] = kept ? y[t][e] : 0.0f;
        store_row<8, T>(q_out + s * a.qo.s + h * a.qo.h + (long long)token * a.qo.n + d, out);
      }
      continue;
    }
    unsigned most = 0;   // bits of the largest magnitude, NaN above all
#pragma unroll
    for(int e = 0; e < 8; ++e) most = max(most, __builtin_bit_cast(unsigned, there ? y[t][e] : 0.0f) & 0x7fffffffu);
#pragma unroll
    for(int o = 1; o < LANES; o <<= 1) most = max(most, (unsigned)__shfl_xor((int)most, o, 64));
    if(!there || !kept) continue;
    const float m = __builtin_bit_cast(float, most);
    unsigned code[2] = {0, 0};
    if(most != 0 && most < 0x7f800000u) {
      const float fast = code_factor<F>(m);
#pragma unroll
      for(int e = 0; e < 8; ++e) code[e / 4] |= code_of<F>(y[t][e], fast, m) << (8 * (e % 4));
    }
    const long long at = ((long long)s * a.heads + h) * a.cap + slot;
    *reinterpret_cast<cache_u2*>((what == 0 ? a.k : a.v) + at * a.dk + d) = cache_u2{code[0], code[1]};
    if(lane == 0) (what == 0 ? a.ks : a.vs)[at] = most < 0x7f800000u ? m / kCodeMost<F> : __builtin_nanf("");
  }
}

// ---------------------------------------------------------------- reading back
// A thread takes sixteen bytes of output at a time - four float32, eight of the shorter types -, kReadTurns of them
// a workgroup's stride apart, of keys and values alike: all loads are out before the first is used.  Memory bounds it: 8 sequences, 8 heads,
// 4001 positions of 128 values, e4m3 to bfloat16, 35.6 us, 5.5 TB/s; 33 positions of 6 sequences 2.9 us.
constexpr int kReadTurns = 4;
template <typename T, CacheFormat F>
__global__ __launch_bounds__(256) void cache_read_kernel(const unsigned char* __restrict__ k, const unsigned char* __restrict__ v,
                                                         const float* __restrict__ ks, const float* __restrict__ vs, const int* __restrict__ first,
                                                         int heads, int cap, int dk, int n, int blocks, T* __restrict__ k_out, T* __restrict__ v_out) {
  constexpr int kEach = 16 / sizeof(T);
  const int entry = blockIdx.x / blocks, block = blockIdx.x % blocks, units = dk / kEach;
  const int from = first[entry / heads];
  const long long in = (long long)entry * cap, to = (long long)entry * n;
  unsigned code[2][kReadTurns][kEach / 4];
  float scale[2][kReadTurns];
#pragma unroll
  for(int t = 0; t < kReadTurns; ++t) {
    const unsigned id = (block * kReadTurns + t) * 256u + threadIdx.x;
    const int i = id / units, d = (id - i * units) * kEach;
    const long long p = (long long)from + i;
    scale[0][t] = scale[1][t] = 0.0f;
#pragma unroll
    for(int e = 0; e < kEach / 4; ++e) code[0][t][e] = code[1][t][e] = 0;
    if(i < n && p >= 0 && p < cap) {
      const long long at = in + p;
      if constexpr(kEach == 8) {
        const cache_u2 a = *reinterpret_cast<const cache_u2*>(k + at * dk + d), b = *reinterpret_cast<const cache_u2*>(v + at * dk + d);
        code[0][t][0] = a[0];
        code[0][t][1] = a[1];
        code[1][t][0] = b[0];
        code[1][t][1] = b[1];
      } else {
        code[0][t][0] = *reinterpret_cast<const unsigned*>(k + at * dk + d);
        code[1][t][0] = *reinterpret_cast<const unsigned*>(v + at * dk + d);
      }
      scale[0][t] = ks[at];
      scale[1][t] = vs[at];
    }
  }
#pragma unroll
  for(int t = 0; t < kReadTurns; ++t) {
    const unsigned id = (block * kReadTurns + t) * 256u + threadIdx.x;
    const int i = id / units, d = (id - i * units) * kEach;
    if(i >= n) break;
#pragma unroll
    for(int x = 0; x < 2; ++x) {
      float y[kEach];
#pragma unroll
      for(int e = 0; e < kEach / 4; ++e) {
        float z[4];
        values_of<F>(code[x][t][e], z);
#pragma unroll
        for(int j = 0; j < 4; ++j) y[4 * e + j] = z[j] * scale[x][t];
      }
      store_row<kEach, T>((x ? v_out : k_out) + (to + i) * dk + d, y);
    }
  }
}

// ---------------------------------------------------------------- accepted drafts
// A workgroup to the keys or the values of an entry: everything is read before anything is written, so a path may go anywhere, twice to
// the same row too.  A launch and the steps that follow each other (path, rows, stores) bound it: 16 to 32 rows of 128 codes in each of 64 sequences, 16
// heads, 5.2 us, 2.4 TB/s; all 64 rows 7.0 us, 4.9 TB/s; 16 rows of one sequence 2.4 us.
__global__ __launch_bounds__(256) void cache_keep_kernel(unsigned char* k, unsigned char* v, float* ks, float* vs, const int* __restrict__ lens,
                                                         const int* __restrict__ path, int path_len, const int* __restrict__ accepted,
                                                         int* __restrict__ new_lens, int heads, int cap, int dk) {
  const int entry = blockIdx.x, s = entry / heads, tid = threadIdx.x;
  unsigned char* const codes = (blockIdx.y ? v : k) + (long long)entry * cap * dk;
  float* const scales = (blockIdx.y ? vs : ks) + (long long)entry * cap;
  const int len = clamp_int(lens[s], 0, cap), count = min(clamp_int(accepted[s], 0, path_len), cap - len);
  auto source = [&](int j) {   // the row that moves to row len + j, or -1
    const int p = path[(long long)s * path_len + j];
    return p < 0 || p >= cap - len ? -1 : len + p;
  };
  const int pieces = dk / 16;
  cache_u4 x[4];   // 64 rows of up to 256 codes
  float scale = 0.0f;
#pragma unroll
  for(int t = 0; t < 4; ++t) {
    const int i = t * 256 + tid, j = i / pieces;
    x[t] = cache_u4{0, 0, 0, 0};
    if(j < count && source(j) >= 0) x[t] = *reinterpret_cast<const cache_u4*>(codes + (long long)source(j) * dk + 16 * (i - j * pieces));
  }
  if(tid < count && source(tid) >= 0) scale = scales[source(tid)];
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // every wave has what it read ...
  __syncthreads();                                   // ... before any writes
#pragma unroll
  for(int t = 0; t < 4; ++t) {
    const int i = t * 256 + tid, j = i / pieces;
    if(j < count && source(j) >= 0) *reinterpret_cast<cache_u4*>(codes + (long long)(len + j) * dk + 16 * (i - j * pieces)) = x[t];
  }
  if(tid < count && source(tid) >= 0) scales[len + tid] = scale;
  if(tid == 0 && blockIdx.y == 0 && entry % heads == 0) new_lens[s] = len + count;
}

// ---------------------------------------------------------------- arguments
template <CacheFormat F>
struct Format {
  static constexpr CacheFormat value = F;
};
template <typename F>
int for_format(int format, F f) {
  return format == MARIAN_HIP_CACHE_INT8 ? f(Format<CacheFormat::int8>()) : f(Format<CacheFormat::e4m3>());
}

int check_cache(const marian_hip_kv_cache* c) {
  if(!c) return MARIAN_HIP_ERR_NULL;
  if(c->sequences < 0 || c->heads < 1 || c->capacity < 1 || !row_size(c->dk) ||
     (c->format != MARIAN_HIP_CACHE_INT8 && c->format != MARIAN_HIP_CACHE_E4M3))
    return MARIAN_HIP_ERR_SHAPE;
  if(c->sequences > kMaxSequences || c->heads > kMaxHeads || c->capacity > 0x7fffffff / c->dk) return MARIAN_HIP_ERR_RANGE;
  return MARIAN_HIP_OK;
}
int check_cache_memory(const marian_hip_kv_cache* c) {
  if(!c->k || !c->v || !c->k_scale || !c->v_scale) return MARIAN_HIP_ERR_NULL;
  if(!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->k_scale, 4) || !aligned(c->v_scale, 4)) return MARIAN_HIP_ERR_ALIGN;
  return MARIAN_HIP_OK;
}
int check_drafts(const marian_hip_drafts* d) {
  if(!d) return MARIAN_HIP_ERR_NULL;
  if(d->n < 0 || (d->parents && d->n > MARIAN_HIP_TREE_MAX)) return MARIAN_HIP_ERR_SHAPE;
  if(d->n > kMaxTokens) return MARIAN_HIP_ERR_RANGE;
  return MARIAN_HIP_OK;
}
int check_drafts_memory(const marian_hip_drafts* d) {
  if(!d->lens) return MARIAN_HIP_ERR_NULL;
  if(!aligned(d->lens, 4) || !aligned(d->counts, 4) || !aligned(d->parents, 4)) return MARIAN_HIP_ERR_ALIGN;
  return MARIAN_HIP_OK;
}
int check_rotation(const marian_hip_rotation* r, int64_t dk) {
  if(r->dims < 8 || r->dims > dk || r->dims % 8 != 0 || !std::isfinite(r->magnitude)) return MARIAN_HIP_ERR_SHAPE;
  if(!r->turns) return MARIAN_HIP_ERR_NULL;
  return aligned(r->turns, 8) ? MARIAN_HIP_OK : MARIAN_HIP_ERR_ALIGN;
}
inline int64_t cache_rows(const marian_hip_kv_cache* c) { return c->sequences * c->heads * c->capacity; }

__global__ __launch_bounds__(256) void clear_kernel(unsigned* p, unsigned n) {
  const unsigned i = blockIdx.x * 256u + threadIdx.x;
  if(i < n) p[i] = 0;
}

}  // namespace

extern "C" {

int marian_hip_rotary_turns(uint64_t* host_turns, double* host_magnitude, int64_t dims, double base, int scaling, double factor,
                            int64_t original, double slow, double fast) {
  if(!host_turns || !host_magnitude) return MARIAN_HIP_ERR_NULL;
  if(dims < 2 || dims % 2 != 0 || dims > 65536 || !(base > 1.0) || !std::isfinite(base) || scaling < MARIAN_HIP_ROTARY_PLAIN ||
     scaling > MARIAN_HIP_ROTARY_BANDS)
    return MARIAN_HIP_ERR_SHAPE;
  if(scaling != MARIAN_HIP_ROTARY_PLAIN && (!(factor >= 1.0) || !std::isfinite(factor))) return MARIAN_HIP_ERR_SHAPE;
  if(scaling == MARIAN_HIP_ROTARY_BASE && dims < 4) return MARIAN_HIP_ERR_SHAPE;
  if(scaling == MARIAN_HIP_ROTARY_BANDS && (original < 1 || !(slow >= 0.0) || !(fast > slow) || !std::isfinite(fast))) return MARIAN_HIP_ERR_SHAPE;
  const long double circle = 6.283185307179586476925286766559005768L;
  long double b = base;
  if(scaling == MARIAN_HIP_ROTARY_BASE) b *= powl(factor, (long double)dims / (dims - 2));
  *host_magnitude = scaling == MARIAN_HIP_ROTARY_BANDS ? 0.1 * std::log(factor) + 1.0 : 1.0;
  for(int64_t p = 0; p < dims / 2; ++p) {
    long double radians = powl(b, -2.0L * p / dims);
    if(scaling == MARIAN_HIP_ROTARY_LINEAR) radians /= factor;
    if(scaling == MARIAN_HIP_ROTARY_BANDS) {
      long double keep = (original * radians / circle - slow) / ((long double)fast - slow);
      keep = keep < 0 ? 0 : keep > 1 ? 1 : keep;
      radians = radians * (keep + (1 - keep) / factor);
    }
    host_turns[p] = (uint64_t)roundl(ldexpl(radians / circle, 64));   // (at most 0.16 of a turn)
  }
  return MARIAN_HIP_OK;
}

int marian_hip_rotary(const void* x, const int64_t* x_strides, void* out, const int64_t* out_strides, int type, int64_t sequences,
                      int64_t heads, int64_t n, int64_t dk, const int32_t* positions, int each, const marian_hip_rotation* rotation,
                      void* stream) {
  MH_CHECK(check_type(type));
  if(sequences < 0 || heads < 1 || n < 0 || !row_size(dk)) return MARIAN_HIP_ERR_SHAPE;
  if(sequences > kMaxSequences || heads > kMaxHeads || n > kMaxTokens || n * heads * (dk / 8) > 0x7fffff00) return MARIAN_HIP_ERR_RANGE;
  if(!rotation) return MARIAN_HIP_ERR_NULL;
  if(rotation->dims < 8 || rotation->dims > dk || rotation->dims % 8 != 0) return MARIAN_HIP_ERR_SHAPE;
  if(sequences == 0 || n == 0) return MARIAN_HIP_OK;
  if(!positions) return MARIAN_HIP_ERR_NULL;
  MH_CHECK(check_rotation(rotation, dk));
  Span in, to;
  MH_CHECK(check_rows(x, x_strides, type, sequences, heads, n, dk, &in));
  MH_CHECK(check_written(out, out_strides, type, sequences, heads, n, dk, &to));
  if(!aligned(positions, 4)) return MARIAN_HIP_ERR_ALIGN;
  if(!same_rows(x, x_strides, out, out_strides, sequences, heads, n)) MH_CHECK(apart({to}, {in}));
  MH_CHECK(apart({to}, {{positions, 4 * (each ? sequences * n : sequences)}, {rotation->turns, 4 * rotation->dims}}));
  const hipStream_t st = static_cast<hipStream_t>(stream);
  // Four heads to a thread share its angles where that leaves two workgroups to a CU.
  const int64_t units = n * (dk / 8), many = (units * ((heads + 3) / 4) + 255) / 256;
  return for_type(type, [&](auto t) -> int {
    using T = decltype(t);
    const unsigned long long* turns = reinterpret_cast<const unsigned long long*>(rotation->turns);
    if(many * sequences >= 512)
      MH_LAUNCH((rotary_kernel<T, 4>), dim3((unsigned)many, (unsigned)sequences), dim3(256), 0, st, static_cast<const T*>(x), strides(x_strides),
                static_cast<T*>(out), strides(out_strides), positions, each, turns, (int)rotation->dims, (float)rotation->magnitude,
                rotation->interleaved, (int)heads, (int)n, (int)dk);
    else
      MH_LAUNCH((rotary_kernel<T, 1>), dim3((unsigned)((units * heads + 255) / 256), (unsigned)sequences), dim3(256), 0, st,
                static_cast<const T*>(x), strides(x_strides), static_cast<T*>(out), strides(out_strides), positions, each, turns,
                (int)rotation->dims, (float)rotation->magnitude, rotation->interleaved, (int)heads, (int)n, (int)dk);
    return MARIAN_HIP_OK;
  });
}

int marian_hip_cache_append(const marian_hip_kv_cache* cache, const marian_hip_drafts* drafts, const void* k, const int64_t* k_strides,
                            const void* v, const int64_t* v_strides, int type, const marian_hip_rotation* rotation, const void* q,
                            const int64_t* q_strides, int64_t q_heads, void* q_out, const int64_t* q_out_strides, void* stream) {
  MH_CHECK(check_cache(cache));
  MH_CHECK(check_drafts(drafts));
  MH_CHECK(check_type(type));
  const int64_t sequences = cache->sequences, n = drafts->n, dk = cache->dk;
  if(q && q_heads < 1) return MARIAN_HIP_ERR_SHAPE;
  if(q && q_heads > 4 * kMaxHeads) return MARIAN_HIP_ERR_RANGE;
  if(rotation && (rotation->dims < 8 || rotation->dims > dk || rotation->dims % 8 != 0)) return MARIAN_HIP_ERR_SHAPE;
  if(sequences == 0 || n == 0) return MARIAN_HIP_OK;
  MH_CHECK(check_cache_memory(cache));
  MH_CHECK(check_drafts_memory(drafts));
  if(rotation) MH_CHECK(check_rotation(rotation, dk));
  Span ks, vs, qs{nullptr, 0}, qo{nullptr, 0};
  MH_CHECK(check_rows(k, k_strides, type, sequences, cache->heads, n, dk, &ks));
  MH_CHECK(check_rows(v, v_strides, type, sequences, cache->heads, n, dk, &vs));
  if(q) {
    MH_CHECK(check_rows(q, q_strides, type, sequences, q_heads, n, dk, &qs));
    MH_CHECK(check_written(q_out, q_out_strides, type, sequences, q_heads, n, dk, &qo));
  }
  const int64_t rows = cache_rows(cache);
  const Span codes[2] = {{cache->k, rows * dk}, {cache->v, rows * dk}}, scales[2] = {{cache->k_scale, rows * 4}, {cache->v_scale, rows * 4}};
  const Span lens{drafts->lens, 4 * sequences}, counts{drafts->counts, 4 * sequences}, parents{drafts->parents, 4 * sequences * n};
  const Span turns{rotation ? rotation->turns : nullptr, rotation ? 4 * rotation->dims : 0};
  const bool in_place = q && same_rows(q, q_strides, q_out, q_out_strides, sequences, q_heads, n);
  MH_CHECK(apart({codes[0], codes[1], scales[0], scales[1], qo}, {ks, vs, lens, counts, parents, turns}));
  MH_CHECK(apart({codes[0], codes[1], scales[0], scales[1]}, {qs}));
  MH_CHECK(apart({codes[0]}, {codes[1], scales[0], scales[1], qo}));
  MH_CHECK(apart({codes[1]}, {scales[0], scales[1], qo}));
  MH_CHECK(apart({scales[0]}, {scales[1], qo}));
  MH_CHECK(apart({scales[1]}, {qo}));
  if(q && !in_place) MH_CHECK(apart({qo}, {qs}));
  const hipStream_t st = static_cast<hipStream_t>(stream);
  AppendArgs a{};
  a.k = static_cast<unsigned char*>(cache->k);
  a.v = static_cast<unsigned char*>(cache->v);
  a.ks = cache->k_scale;
  a.vs = cache->v_scale;
  a.lens = drafts->lens;
  a.counts = drafts->counts;
  a.parents = drafts->parents;
  a.turns = rotation ? reinterpret_cast<const unsigned long long*>(rotation->turns) : nullptr;
  a.magnitude = rotation ? rotation->magnitude : 1.0;
  a.kx = strides(k_strides);
  a.vx = strides(v_strides);
  if(q) {
    a.qx = strides(q_strides);
    a.qo = strides(q_out_strides);
  }
  a.dims = rotation ? (int)rotation->dims : 0;
  a.interleaved = rotation ? rotation->interleaved : 0;
  a.heads = (int)cache->heads;
  a.q_heads = q ? (int)q_heads : 0;
  a.n = (int)n;
  a.cap = (int)cache->capacity;
  a.dk = (int)dk;
  const int64_t all = 2 * a.heads + a.q_heads;
  // Four tokens to a workgroup, all asked for at once, where a workgroup each would be more than 32 to a CU: 512 tokens of 16 sequences, 48 rows
  // of 128 values a token, bfloat16, 47.8 us against 59.0 (a prompt's angles and the wait for memory count; float32 74 both); below that a workgroup
  // to each: 64 tokens 10.8 us against 11.9, 3 of 64 sequences 5.2 against 7.3.
  const int lanes = dk <= 64 ? 8 : dk <= 128 ? 16 : 32;
  const int64_t row_groups = (all * lanes + 255) / 256;
  const int each = row_groups * n * sequences > 8192 ? 4 : 1;
  const int64_t tokens = (n + each - 1) / each;
  if(tokens > 65535) return MARIAN_HIP_ERR_RANGE;
  return for_type(type, [&](auto t) -> int {
    using T = decltype(t);
    return for_format(cache->format, [&](auto f) -> int {
      constexpr CacheFormat F = decltype(f)::value;
      const T *kp = static_cast<const T*>(k), *vp = static_cast<const T*>(v), *qp = static_cast<const T*>(q);
      T* qop = static_cast<T*>(q_out);
      const dim3 grid((unsigned)row_groups, (unsigned)tokens, (unsigned)sequences);
      auto launch = [&](auto given) -> int {
        constexpr int LANES = decltype(given)::value;
        if(each == 1) MH_LAUNCH((append_kernel<T, F, LANES, 1>), grid, dim3(256), 0, st, kp, vp, qp, qop, a);
        else MH_LAUNCH((append_kernel<T, F, LANES, 4>), grid, dim3(256), 0, st, kp, vp, qp, qop, a);
        return MARIAN_HIP_OK;
      };
      if(lanes == 8) return launch(std::integral_constant<int, 8>());
      if(lanes == 16) return launch(std::integral_constant<int, 16>());
      return launch(std::integral_constant<int, 32>());
    });
  });
}

int marian_hip_cache_read(const marian_hip_kv_cache* cache, const int32_t* first, int64_t n, void* k_out, void* v_out, int type,
                          void* stream) {
  MH_CHECK(check_cache(cache));
  MH_CHECK(check_type(type));
  if(n < 0) return MARIAN_HIP_ERR_SHAPE;
  const int64_t entries = cache->sequences * cache->heads, dk = cache->dk;
  if(n > 0x7fffff00 / dk) return MARIAN_HIP_ERR_RANGE;
  if(entries == 0 || n == 0) return MARIAN_HIP_OK;
  const int64_t blocks = (n * dk * width_of(type) / 16 + 256 * kReadTurns - 1) / (256 * kReadTurns);
  if(blocks * entries > kMostThreads / 256) return MARIAN_HIP_ERR_RANGE;
  MH_CHECK(check_cache_memory(cache));
  if(!first || !k_out || !v_out) return MARIAN_HIP_ERR_NULL;
  if(!aligned(first, 4) || !aligned(k_out, 16) || !aligned(v_out, 16)) return MARIAN_HIP_ERR_ALIGN;
  const int64_t rows = cache_rows(cache), bytes = entries * n * dk * width_of(type);
  MH_CHECK(apart({{k_out, bytes}}, {{v_out, bytes}}));
  MH_CHECK(apart({{k_out, bytes}, {v_out, bytes}}, {{cache->k, rows * dk}, {cache->v, rows * dk}, {cache->k_scale, rows * 4},
                                                    {cache->v_scale, rows * 4}, {first, 4 * cache->sequences}}));
  const hipStream_t st = static_cast<hipStream_t>(stream);
  return for_type(type, [&](auto t) -> int {
    using T = decltype(t);
    return for_format(cache->format, [&](auto f) -> int {
      MH_LAUNCH((cache_read_kernel<T, decltype(f)::value>), dim3((unsigned)(blocks * entries)), dim3(256), 0, st,
                static_cast<const unsigned char*>(cache->k), static_cast<const unsigned char*>(cache->v), cache->k_scale, cache->v_scale, first,
                (int)cache->heads, (int)cache->capacity, (int)dk, (int)n, (int)blocks, static_cast<T*>(k_out), static_cast<T*>(v_out));
      return MARIAN_HIP_OK;
    });
  });
}

size_t marian_hip_cache_attention_workspace_bytes(int64_t sequences, int64_t heads, int64_t q_heads, int64_t n, int64_t dk) {
  if(sequences < 1 || heads < 1 || q_heads < heads || q_heads % heads != 0 || n < 1 || !row_size(dk)) return 0;
  if(sequences > 0xffff || q_heads > (int64_t)kMaxHeads * heads || n > 1 << 20) return 0;
  int64_t bytes = 0;   // (enough for any capacity)
  for(const int64_t capacity : {(int64_t)1, (int64_t)1 << 31})
    bytes = std::max(bytes, cache_attention_bytes(cache_attention_plan(sequences, heads, q_heads, capacity, n, dk), heads));
  return (size_t)bytes;
}

int marian_hip_cache_attention_workspace_init(void* workspace, size_t workspace_bytes, void* stream) {
  if(workspace_bytes == 0) return MARIAN_HIP_OK;
  if(!workspace) return MARIAN_HIP_ERR_NULL;
  if(!aligned(workspace, 256)) return MARIAN_HIP_ERR_ALIGN;
  const unsigned words = (unsigned)(std::min<size_t>(workspace_bytes, kCacheCounterBytes) / 4);
  MH_LAUNCH(clear_kernel, dim3((words + 255) / 256), dim3(256), 0, static_cast<hipStream_t>(stream), static_cast<unsigned*>(workspace), words);
  return MARIAN_HIP_OK;
}

int marian_hip_cache_attention(const marian_hip_kv_cache* cache, const marian_hip_drafts* drafts, const void* q, const int64_t* q_strides,
                               int64_t q_heads, int type, float scale, void* out, const int64_t* out_strides, void* workspace,
                               size_t workspace_bytes, void* stream) {
  MH_CHECK(check_cache(cache));
  MH_CHECK(check_drafts(drafts));
  MH_CHECK(check_type(type));
  const int64_t sequences = cache->sequences, n = drafts->n, dk = cache->dk, heads = cache->heads;
  if(q_heads < heads || q_heads % heads != 0 || !(scale > 0.0f) || !std::isfinite(scale)) return MARIAN_HIP_ERR_SHAPE;
  if(q_heads / heads > kMaxHeads || n * (q_heads / heads) > 1 << 26) return MARIAN_HIP_ERR_RANGE;
  if(sequences == 0 || n == 0) return MARIAN_HIP_OK;
  const CacheAttentionPlan p = cache_attention_plan(sequences, heads, q_heads, cache->capacity, n, dk);
  if(p.grid > kMostThreads / (64 * p.waves)) return MARIAN_HIP_ERR_RANGE;
  MH_CHECK(check_cache_memory(cache));
  MH_CHECK(check_drafts_memory(drafts));
  Span qs, os;
  MH_CHECK(check_rows(q, q_strides, type, sequences, q_heads, n, dk, &qs));
  MH_CHECK(check_written(out, out_strides, type, sequences, q_heads, n, dk, &os));
  const int64_t need = cache_attention_bytes(p, heads), rows = cache_rows(cache);
  if(need > 0 && !workspace) return MARIAN_HIP_ERR_NULL;
  if((int64_t)workspace_bytes < need) return MARIAN_HIP_ERR_WORKSPACE;
  if(!aligned(workspace, 256)) return MARIAN_HIP_ERR_ALIGN;
  const Span work{need > 0 ? workspace : nullptr, need};
  MH_CHECK(apart({os, work}, {qs, {cache->k, rows * dk}, {cache->v, rows * dk}, {cache->k_scale, rows * 4}, {cache->v_scale, rows * 4},
                              {drafts->lens, 4 * sequences}, {drafts->counts, 4 * sequences}, {drafts->parents, 4 * sequences * n}}));
  MH_CHECK(apart({os}, {work}));
  CacheAttentionArgs a{};
  a.q = q;
  a.q_s = q_strides[0];
  a.q_h = q_strides[1];
  a.q_n = q_strides[2];
  a.out = out;
  a.o_s = out_strides[0];
  a.o_h = out_strides[1];
  a.o_n = out_strides[2];
  a.k = static_cast<const unsigned char*>(cache->k);
  a.v = static_cast<const unsigned char*>(cache->v);
  a.ks = cache->k_scale;
  a.vs = cache->v_scale;
  a.lens = drafts->lens;
  a.counts = drafts->counts;
  a.parents = drafts->parents;
  a.counters = static_cast<unsigned*>(workspace);
  a.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + kCacheCounterBytes);
  a.S = (int)sequences;
  a.Hk = (int)heads;
  a.G = (int)(q_heads / heads);
  a.n = (int)n;
  a.cap = (int)cache->capacity;
  a.dk = (int)dk;
  a.row_tiles = (int)p.row_tiles;
  a.target = (int)p.target;
  a.least = p.least;
  a.items = (int)p.items;
  a.by_tiles = CacheDivisor((unsigned)p.row_tiles);
  a.by_heads = CacheDivisor((unsigned)heads);
  a.by_group = CacheDivisor((unsigned)a.G);
  a.scale_log2 = (float)((double)scale * 1.4426950408889634);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if(type == MARIAN_HIP_FLOAT32) return launch_cache_attention_float32(a, p, cache->format, st);
  if(type == MARIAN_HIP_FLOAT16) return launch_cache_attention_float16(a, p, cache->format, st);
  return launch_cache_attention_bfloat16(a, p, cache->format, st);
}

int marian_hip_cache_keep(const marian_hip_kv_cache* cache, const int32_t* lens, const int32_t* path, int64_t path_len,
                          const int32_t* accepted, int32_t* new_lens, void* stream) {
  MH_CHECK(check_cache(cache));
  if(path_len < 0 || path_len > MARIAN_HIP_TREE_MAX) return MARIAN_HIP_ERR_SHAPE;
  const int64_t sequences = cache->sequences, rows = cache_rows(cache), dk = cache->dk;
  if(sequences * cache->heads > kMostThreads / 256) return MARIAN_HIP_ERR_RANGE;
  if(sequences == 0) return MARIAN_HIP_OK;
  MH_CHECK(check_cache_memory(cache));
  if(!lens || !accepted || !new_lens || (path_len > 0 && !path)) return MARIAN_HIP_ERR_NULL;
  if(!aligned(lens, 4) || !aligned(accepted, 4) || !aligned(new_lens, 4) || !aligned(path, 4)) return MARIAN_HIP_ERR_ALIGN;
  const Span codes[2] = {{cache->k, rows * dk}, {cache->v, rows * dk}}, scales[2] = {{cache->k_scale, rows * 4}, {cache->v_scale, rows * 4}};
  const Span now{lens, 4 * sequences}, taken{accepted, 4 * sequences}, along{path, 4 * sequences * path_len}, then{new_lens, 4 * sequences};
  MH_CHECK(apart({codes[0], codes[1], scales[0], scales[1], then}, {now, taken, along}));
  MH_CHECK(apart({codes[0]}, {codes[1], scales[0], scales[1], then}));
  MH_CHECK(apart({codes[1]}, {scales[0], scales[1], then}));
  MH_CHECK(apart({scales[0]}, {scales[1], then}));
  MH_CHECK(apart({scales[1]}, {then}));
  MH_LAUNCH(cache_keep_kernel, dim3((unsigned)(sequences * cache->heads), 2), dim3(256), 0, static_cast<hipStream_t>(stream),
            static_cast<unsigned char*>(cache->k), static_cast<unsigned char*>(cache->v), cache->k_scale, cache->v_scale, lens, path,
            (int)path_len, accepted, new_lens, (int)cache->heads, (int)cache->capacity, (int)dk);
  return MARIAN_HIP_OK;
}

}  // extern "C"
