// packed.cpp -- C entries of the rotary variants, the 8-bit K/V cache and the
// attention of packed batches over it (include/slate_hip.h).  Arguments are
// checked before the device is touched.
#include <math.h>

#include <mutex>

#include "packed.h"

namespace slate_hip {
extern std::mutex g_enqueue_mu;
}
using namespace slate_hip;

namespace {

constexpr double TWO_PI = 6.283185307179586;

bool rope_ok(const slate_hip_rope_t* r) {
    if (!r || (r->layout != 0 && r->layout != 1) || r->rot_dim < 2 || r->rot_dim % 2 ||
        r->rot_dim / 2 > ROPE_MAX_PAIRS || r->scaling < 0 || r->scaling > 3)
        return false;
    if (!(r->theta_base > 0) || !isfinite(r->theta_base) || !isfinite(r->magnitude)) return false;
    if (r->scaling >= 1 && (!(r->factor > 0) || !isfinite(r->factor))) return false;
    if (r->scaling >= 2 && (r->orig_ctx < 1 || !(r->low > 0) || !(r->high > r->low) || !isfinite(r->high)))
        return false;
    return r->scaling != 3 || r->theta_base > 1;
}

// False where a frequency or the magnitude is too large for its type (an angle
// of any position has to be a finite double).
bool rope_frequencies(double* w, double* magnitude, const slate_hip_rope_t* r) {
    const int n = r->rot_dim / 2;
    double a = 0, b = 0;
    if (r->scaling == 3) {
        const double per = r->rot_dim / (2 * log(r->theta_base));
        a = fmax(0.0, floor(per * log(r->orig_ctx / (r->high * TWO_PI))));
        b = fmin(r->rot_dim - 1.0, ceil(per * log(r->orig_ctx / (r->low * TWO_PI))));
    }
    bool fine = true;
    const double per_pair = -2.0 * log(r->theta_base) / r->rot_dim;   // exp: a tenth of pow's time, within 2^-48
    for (int i = 0; i < n; ++i) {
        const double f = exp(per_pair * i);
        double slow = 0;                               // the share of f / factor
        if (r->scaling == 1) slow = 1;
        if (r->scaling == 2) slow = 1 - fmin(1.0, fmax(0.0, (r->orig_ctx * f / TWO_PI - r->low) / (r->high - r->low)));
        if (r->scaling == 3) slow = fmin(1.0, fmax(0.0, (i - a) / (b > a ? b - a : 0.001)));
        w[i] = slow == 0 ? f : slow * (f / r->factor) + (1 - slow) * f;
        fine &= isfinite(w[i] * 2147483648.0) != 0;
    }
    *magnitude = r->magnitude != 0 ? r->magnitude
                                   : (r->scaling == 3 && r->factor > 1 ? 0.1 * log(r->factor) + 1 : 1.0);
    return fine && isfinite((float)*magnitude);
}

// Whether the byte ranges [a, a + n) and [b, b + m) share a byte.
bool overlap(const void* a, size_t n, const void* b, size_t m) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return x < y + m && y < x + n;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

int kv8_check(const char* what, const void* kq, const void* ks, const void* vq, const void* vs, const float* k,
              const float* v, int64_t ld, const int32_t* tok_off, const int32_t* pos0, const int64_t* kv_base, int B,
              int T, int n_kv, int hd, int64_t head_stride, int max_seq) {
    SH_REQUIRE(kq && ks && vq && vs && k && v && tok_off && pos0 && kv_base, "%s: null pointer", what);
    SH_REQUIRE(B >= 1 && B <= PK_MAX_SEQ && T >= 1 && n_kv >= 1 && max_seq >= 1, "%s: bad sizes", what);
    SH_REQUIRE(hd >= KV8_BLOCK && hd <= PK_MAX_HD && hd % KV8_BLOCK == 0 && head_stride >= 0 && head_stride % hd == 0,
               "%s: head_dim=%d or head_stride=%lld", what, hd, (long long)head_stride);
    SH_REQUIRE((int64_t)n_kv * hd <= INT32_MAX / 4 && ld >= (int64_t)n_kv * hd && ld % 4 == 0, "%s: ld=%lld", what,
               (long long)ld);
    SH_REQUIRE(aligned16(kq) && aligned16(ks) && aligned16(vq) && aligned16(vs) && aligned16(k) && aligned16(v),
               "%s: pointers are not 16-byte aligned", what);
    return 0;
}

int attention_packed(const char* what, const PackedAttn& a, PackedBatch pb, bool tree, size_t ws_bytes) {
    const bool q8 = a.kf == nullptr && a.vf == nullptr;
    SH_REQUIRE(a.out && a.q && pb.tok_off && pb.pos0 && pb.kv_base && (!tree || a.parent) &&
                   (q8 ? a.kv8.kq && a.kv8.ks && a.kv8.vq && a.kv8.vs : a.kf && a.vf),
               "%s: null pointer", what);
    SH_REQUIRE(pb.B >= 1 && pb.B <= PK_MAX_SEQ && pb.T >= 1 && pb.max_new >= 1 && pb.max_seq >= 1 &&
                   (!tree || pb.max_new <= PK_MAX_DRAFT),
               "%s: bad sizes (B=%d, T=%d, max_new=%d, max_seq=%d)", what, pb.B, pb.T, pb.max_new, pb.max_seq);
    SH_REQUIRE(a.Hkv >= 1 && a.Hq >= a.Hkv && a.Hq % a.Hkv == 0 && a.Hq <= 65535, "%s: %d/%d heads", what, a.Hq, a.Hkv);
    const int unit = q8 ? KV8_BLOCK : 16;
    SH_REQUIRE(a.hd >= unit && a.hd <= PK_MAX_HD && a.hd % unit == 0 && a.head_stride >= 0 &&
                   (!q8 || a.head_stride % a.hd == 0),
               "%s: head_dim=%d or head_stride=%lld", what, a.hd, (long long)a.head_stride);
    SH_REQUIRE(!q8 || (aligned16(a.kv8.kq) && aligned16(a.kv8.ks) && aligned16(a.kv8.vq) && aligned16(a.kv8.vs)),
               "%s: pools are not 16-byte aligned", what);
    if (pb.max_seq > PK_MAX_KEYS) pb.max_seq = PK_MAX_KEYS;
    SH_REQUIRE((int64_t)pb.T * a.Hq <= INT32_MAX - 127 && attention_packed_fits(a, pb),
               "%s: %d tokens over max_seq=%d are too much for one call", what, pb.T, pb.max_seq);
    const size_t bytes = (size_t)pb.T * a.Hq * a.hd * sizeof(float);
    SH_REQUIRE(!overlap(a.out, bytes, a.q, bytes), "%s: out overlaps q", what);
    const size_t need = (size_t)attention_packed_bytes(a.Hq, a.Hkv, a.hd);
    SH_REQUIRE(!a.ws || (aligned16(a.ws) && ws_bytes >= need), "%s: workspace of %zu bytes, %zu are needed (aligned)",
               what, ws_bytes, need);
    if (!device_ok()) return -7;
    std::lock_guard<std::mutex> lk(g_enqueue_mu);
    PackedAttn c = a;
    if (!c.ws) {
        hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
        SH_CHECK_HIP(hipStreamIsCapturing(stream(), &st));
        if (st != hipStreamCaptureStatusNone) {
            set_error(-5, "%s: a captured call needs a workspace of its own", what);
            return -5;
        }
        if (need && !(c.ws = scratch(7, need))) return -2;
    }
    return launch_attention_packed(c, pb, stream());
}

}  // namespace

extern "C" {

int slate_hip_rope_frequencies(double* w, double* magnitude, const slate_hip_rope_t* rope) {
    SH_REQUIRE(w && magnitude && rope_ok(rope), "rope_frequencies: bad arguments");
    SH_REQUIRE(rope_frequencies(w, magnitude, rope), "rope_frequencies: out of range");
    return 0;
}

int slate_hip_rope_scaled(float* y, const float* x, const int32_t* pos, int n_rows, int n_heads, int head_dim,
                          int64_t ld, const slate_hip_rope_t* rope) {
    SH_REQUIRE(y && x && pos && n_rows > 0 && n_heads > 0 && head_dim > 0, "rope_scaled: bad arguments");
    SH_REQUIRE(rope_ok(rope) && rope->rot_dim <= head_dim, "rope_scaled: bad rotation");
    SH_REQUIRE((int64_t)n_heads * head_dim <= INT32_MAX && ld >= (int64_t)n_heads * head_dim, "rope_scaled: ld=%lld",
               (long long)ld);
    const size_t bytes = ((size_t)(n_rows - 1) * ld + (size_t)n_heads * head_dim) * sizeof(float);
    SH_REQUIRE(y == x || !overlap(y, bytes, x, bytes), "rope_scaled: y overlaps x");
    RopeTurns turns = {};
    double magnitude = 1;
    SH_REQUIRE(rope_frequencies(turns.w, &magnitude, rope), "rope_scaled: frequencies out of range");
    if (!device_ok()) return -7;
    for (int i = 0; i < rope->rot_dim / 2; ++i) turns.w[i] /= TWO_PI;
    std::lock_guard<std::mutex> lk(g_enqueue_mu);
    return launch_rope_scaled(y, x, pos, n_rows, n_heads, head_dim, ld, rope->layout, rope->rot_dim, (float)magnitude,
                              turns, stream());
}

int slate_hip_kv_store_q8(int8_t* Kq, uint16_t* Ks, int8_t* Vq, uint16_t* Vs, const float* k, const float* v,
                          int64_t ld, const int32_t* tok_off, const int32_t* pos0, const int64_t* kv_base, int B,
                          int T, int n_kv_heads, int head_dim, int64_t head_stride, int max_seq) {
    const int rc = kv8_check("kv_store_q8", Kq, Ks, Vq, Vs, k, v, ld, tok_off, pos0, kv_base, B, T, n_kv_heads,
                             head_dim, head_stride, max_seq);
    if (rc) return rc;
    if (!device_ok()) return -7;
    std::lock_guard<std::mutex> lk(g_enqueue_mu);
    return launch_kv_store_q8(Kq, (_Float16*)Ks, Vq, (_Float16*)Vs, k, v, ld,
                              PackedBatch{tok_off, pos0, kv_base, B, T, T, max_seq}, n_kv_heads, head_dim, head_stride,
                              stream());
}

int slate_hip_kv_load_q8(float* k, float* v, int64_t ld, const int8_t* Kq, const uint16_t* Ks, const int8_t* Vq,
                         const uint16_t* Vs, const int32_t* tok_off, const int32_t* pos0, const int64_t* kv_base,
                         int B, int T, int n_kv_heads, int head_dim, int64_t head_stride, int max_seq) {
    const int rc = kv8_check("kv_load_q8", Kq, Ks, Vq, Vs, k, v, ld, tok_off, pos0, kv_base, B, T, n_kv_heads,
                             head_dim, head_stride, max_seq);
    if (rc) return rc;
    if (!device_ok()) return -7;
    std::lock_guard<std::mutex> lk(g_enqueue_mu);
    return launch_kv_load_q8(k, v, ld, Kv8{Kq, Vq, (const _Float16*)Ks, (const _Float16*)Vs},
                             PackedBatch{tok_off, pos0, kv_base, B, T, T, max_seq}, n_kv_heads, head_dim, head_stride,
                             stream());
}

int64_t slate_hip_attention_packed_bytes(int n_q_heads, int n_kv_heads, int head_dim) {
    if (n_kv_heads < 1 || n_q_heads < n_kv_heads || n_q_heads % n_kv_heads || n_q_heads > 65535 || head_dim < 16 ||
        head_dim > PK_MAX_HD || head_dim % 16)
        return -1;
    return attention_packed_bytes(n_q_heads, n_kv_heads, head_dim);
}

int slate_hip_attention_ragged_q8(float* out, const float* q, const int8_t* Kq, const uint16_t* Ks,
                                  const int8_t* Vq, const uint16_t* Vs, const int32_t* tok_off, const int32_t* pos0,
                                  const int64_t* kv_base, int B, int T, int max_new, int n_q_heads, int n_kv_heads,
                                  int head_dim, int64_t head_stride, int max_seq, void* ws, size_t ws_bytes) {
    return attention_packed("attention_ragged_q8",
                            PackedAttn{out, q, nullptr, nullptr, {Kq, Vq, (const _Float16*)Ks, (const _Float16*)Vs},
                                       nullptr, n_q_heads, n_kv_heads, head_dim, head_stride, ws},
                            PackedBatch{tok_off, pos0, kv_base, B, T, max_new, max_seq}, false, ws_bytes);
}

int slate_hip_attention_tree(float* out, const float* q, const float* Kpool, const float* Vpool,
                             const int32_t* tok_off, const int32_t* pos0, const int64_t* kv_base,
                             const int32_t* parent, int B, int T, int max_new, int n_q_heads, int n_kv_heads,
                             int head_dim, int64_t head_stride, int max_seq, void* ws, size_t ws_bytes) {
    SH_REQUIRE(Kpool && Vpool, "attention_tree: null pointer");
    return attention_packed("attention_tree",
                            PackedAttn{out, q, Kpool, Vpool, {}, parent, n_q_heads, n_kv_heads, head_dim, head_stride,
                                       ws},
                            PackedBatch{tok_off, pos0, kv_base, B, T, max_new, max_seq}, true, ws_bytes);
}

int slate_hip_attention_tree_q8(float* out, const float* q, const int8_t* Kq, const uint16_t* Ks, const int8_t* Vq,
                                const uint16_t* Vs, const int32_t* tok_off, const int32_t* pos0,
                                const int64_t* kv_base, const int32_t* parent, int B, int T, int max_new,
                                int n_q_heads, int n_kv_heads, int head_dim, int64_t head_stride, int max_seq,
                                void* ws, size_t ws_bytes) {
    return attention_packed("attention_tree_q8",
                            PackedAttn{out, q, nullptr, nullptr, {Kq, Vq, (const _Float16*)Ks, (const _Float16*)Vs},
                                       parent, n_q_heads, n_kv_heads, head_dim, head_stride, ws},
                            PackedBatch{tok_off, pos0, kv_base, B, T, max_new, max_seq}, true, ws_bytes);
}

}  // extern "C"
