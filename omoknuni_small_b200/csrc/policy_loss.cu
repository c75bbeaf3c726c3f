// Entry points of the policy losses over rows of logits: cross entropy with the search's visit distribution, and the
// clipped-ratio loss with a KL term against a reference policy.  Checks of arguments and the choice of a kernel; the
// kernels are in policy_loss_rows.cuh.
#include "policy_loss_rows.cuh"

namespace ob200 {

static std::atomic<uint32_t> g_spin_limit{ptx::kSpinLimit};
uint32_t policy_spin_limit() { return g_spin_limit.load(std::memory_order_relaxed); }

namespace {

using Rows = PolicyRows;

int elem_bytes(int dtype) { return dtype == OB200_DTYPE_F32 ? 4 : 2; }

// Whether rows [n][A] of `es`-byte elements at a (pitch pa) and of eb-byte elements at b (pitch pb) may share a byte.
bool rows_meet(const void* a, long long pa, int ea, const void* b, long long pb, int eb, long long n, long long A) {
    const intptr_t a0 = (intptr_t)a, b0 = (intptr_t)b;
    const intptr_t a1 = a0 + ((n - 1) * pa + A) * ea, b1 = b0 + ((n - 1) * pb + A) * eb;
    if (a1 <= b0 || b1 <= a0) return false;
    if (pa * ea != pb * eb) return true;
    const intptr_t step = pa * ea, off = (((b0 - a0) % step) + step) % step;   // b's rows start here within a's
    return off < A * ea || off + A * eb > step;
}

// A matrix ends within 2^46 elements of its start: beyond any memory, and no offset in bytes leaves 64 bits.
bool pitch_fits(long long pitch, int A, int n) { return pitch >= A && pitch <= 1LL << 31 && (n - 1LL) * pitch + A <= 1LL << 46; }

// What both losses ask of their rows; fills the shared part of r.
int take_rows(const char* who, const ob200_policy_rows* p, Rows* r) {
    if (!p) return set_error(OB200_ERR_INVALID, "%s: null argument", who);
    if (p->dtype != OB200_DTYPE_BF16 && p->dtype != OB200_DTYPE_F16 && p->dtype != OB200_DTYPE_F32)
        return set_error(OB200_ERR_INVALID, "%s: bad dtype %d", who, p->dtype);
    if (p->n < 0 || p->n_actions < 1) return set_error(OB200_ERR_INVALID, "%s: bad size (n %d, n_actions %d)", who, p->n, p->n_actions);
    if (p->n_actions > (1 << 30)) return set_error(OB200_ERR_TOO_LARGE, "%s: over 2^30 actions", who);
    if (p->n == 0) return OB200_OK;
    const int es = elem_bytes(p->dtype);
    if (!p->logits || !p->grad) return set_error(OB200_ERR_INVALID, "%s: null logits or grad", who);
    if (!pitch_fits(p->logits_pitch, p->n_actions, p->n) || !pitch_fits(p->grad_pitch, p->n_actions, p->n))
        return set_error(OB200_ERR_INVALID, "%s: a pitch is below n_actions or above 2^31, or a matrix beyond 2^46 elements", who);
    if (((uintptr_t)p->logits | (uintptr_t)p->grad) % es || ((uintptr_t)p->legal_bits | (uintptr_t)p->row_weight | (uintptr_t)p->loss) % 4 || (uintptr_t)p->stats % 16)
        return set_error(OB200_ERR_INVALID, "%s: a pointer is not aligned", who);
    if (p->legal_bits && p->mask_words < (p->n_actions + 31) / 32)
        return set_error(OB200_ERR_INVALID, "%s: mask_words %d too small for %d actions", who, p->mask_words, p->n_actions);
    if (p->legal_bits && (long long)p->n * p->mask_words > 1LL << 46) return set_error(OB200_ERR_INVALID, "%s: legal_bits beyond 2^46 words", who);
    if (!(p->grad == p->logits && p->grad_pitch == p->logits_pitch) &&
        rows_meet(p->grad, p->grad_pitch, es, p->logits, p->logits_pitch, es, p->n, p->n_actions))
        return set_error(OB200_ERR_INVALID, "%s: grad overlaps logits (it may be logits itself, with the same pitch)", who);
    r->z = p->logits; r->bits = p->legal_bits; r->weight = p->row_weight;
    r->grad = p->grad; r->loss = p->loss; r->stats = (float4*)p->stats;
    r->z_pitch = p->logits_pitch; r->g_pitch = p->grad_pitch;
    r->n = p->n; r->A = p->n_actions; r->mask_words = p->mask_words;
    return OB200_OK;
}

// What a call writes shares no memory with what it reads, or with what else it writes (grad and the matrices it reads: take_rows
// and the entry points).  x: target or reference logits.
int check_vectors(const char* who, const Rows& r, int es, int x_bytes) {
    struct Vector { const char* what; const void* at; long long unit; };
    const Vector v[7] = {{"loss", r.loss, 4}, {"stats", r.stats, 16}, {"row_weight", r.weight, 4}, {"action", r.action, 4},
                         {"old_logp", r.old_logp, 4}, {"advantage", r.advantage, 4}, {"legal_bits", r.bits, 4LL * r.mask_words}};
    const struct Matrix { intptr_t at, step, row; } m[3] = {{(intptr_t)r.grad, (intptr_t)r.g_pitch * es, (intptr_t)r.A * es},
                                                            {(intptr_t)r.z, (intptr_t)r.z_pitch * es, (intptr_t)r.A * es},
                                                            {(intptr_t)r.x, (intptr_t)r.x_pitch * x_bytes, (intptr_t)r.A * x_bytes}};
    intptr_t end[3];
    for (int k = 0; k < 3; ++k) end[k] = m[k].at + (m[k].at ? (r.n - 1) * m[k].step + m[k].row : 0);
    for (int i = 0; i < 7; ++i) {
        const intptr_t a = (intptr_t)v[i].at, b = a + v[i].unit * r.n;
        if (!a) continue;
        for (int k = 0; k < (i < 2 ? 3 : 1); ++k) {
            if (a >= end[k] || b <= m[k].at) continue;
            const intptr_t off = (((a - m[k].at) % m[k].step) + m[k].step) % m[k].step;      // it may lie between two rows
            if (off < m[k].row || off + (b - a) > m[k].step) return set_error(OB200_ERR_INVALID, "%s: %s overlaps %s", who, v[i].what, k ? "a matrix" : "grad");
        }
        for (int j = i + 1; i < 2 && j < 7; ++j)
            if (v[j].at && a < (intptr_t)v[j].at + v[j].unit * r.n && (intptr_t)v[j].at < b)
                return set_error(OB200_ERR_INVALID, "%s: %s overlaps %s", who, v[i].what, v[j].what);
    }
    return OB200_OK;
}

// Whether the rows of all matrices start at the same element of a vector; then that of row 0.
void find_phase(Rows* r, int dtype, int x_bytes) {
    const int es = elem_bytes(dtype), V = 16 / es;
    const uintptr_t z = (uintptr_t)r->z / es % V, g = (uintptr_t)r->grad / es % V;
    const uintptr_t x = r->x ? (uintptr_t)r->x / x_bytes % V : z;
    const long long xp = r->x ? r->x_pitch : r->z_pitch;
    const bool alike = z == g && z == x && (r->n == 1 || (r->z_pitch % V == r->g_pitch % V && r->z_pitch % V == xp % V));
    r->phase = alike ? (int)z : -1;
}

int launch_rows(int kind, const Rows& r, int dtype, cudaStream_t st) {
    if (dtype == OB200_DTYPE_BF16) return launch_policy_rows_bf16(kind, r, st);
    if (dtype == OB200_DTYPE_F16) return launch_policy_rows_f16(kind, r, st);
    return launch_policy_rows_f32(kind, r, st);
}

}  // namespace
}  // namespace ob200

using namespace ob200;

extern "C" {

void ob200_debug_policy_waits(int32_t give_up) { g_spin_limit.store(give_up ? 0u : ptx::kSpinLimit, std::memory_order_relaxed); }

int ob200_launch_policy_loss_search(const ob200_policy_rows* rows, const void* target, int64_t target_pitch, int32_t target_kind,
                                    float entropy_coef, ob200_stream stream) {
    const char* who = "ob200_launch_policy_loss_search";
    Rows r{};
    if (int rc = take_rows(who, rows, &r)) return rc;
    if (target_kind != OB200_TARGET_VISITS && target_kind != OB200_TARGET_PROBS)
        return set_error(OB200_ERR_INVALID, "%s: bad target_kind %d", who, target_kind);
    if (rows->n > 0) {
        if (!target || (uintptr_t)target % 4 || !pitch_fits(target_pitch, r.A, r.n))
            return set_error(OB200_ERR_INVALID, "%s: target is null, not aligned, its pitch is below n_actions, or it goes too far", who);
        if (rows_meet(r.grad, r.g_pitch, elem_bytes(rows->dtype), target, target_pitch, 4, r.n, r.A))
            return set_error(OB200_ERR_INVALID, "%s: grad overlaps target", who);
        r.x = target; r.x_pitch = target_pitch;
        if (int rc = check_vectors(who, r, elem_bytes(rows->dtype), 4)) return rc;
    }
    if (int rc = require_device()) return rc;
    if (rows->n == 0) return OB200_OK;
    r.entropy = entropy_coef;
    r.visits = target_kind == OB200_TARGET_VISITS;
    find_phase(&r, rows->dtype, 4);
    return launch_rows(kSearch, r, rows->dtype, as_stream(stream));
}

int ob200_launch_policy_loss_clipped(const ob200_policy_rows* rows, const int32_t* action, const float* old_logp, const float* advantage,
                                     const void* ref_logits, int64_t ref_pitch, float clip_low, float clip_high, float kl_coef,
                                     float entropy_coef, ob200_stream stream) {
    const char* who = "ob200_launch_policy_loss_clipped";
    Rows r{};
    if (int rc = take_rows(who, rows, &r)) return rc;
    if (!(clip_low >= 0.f) || !(clip_high >= 0.f)) return set_error(OB200_ERR_INVALID, "%s: a clip range is negative", who);
    if (!ref_logits && kl_coef != 0.f) return set_error(OB200_ERR_INVALID, "%s: kl_coef without ref_logits", who);
    if (rows->n > 0) {
        if (!action || !old_logp || !advantage || ((uintptr_t)action | (uintptr_t)old_logp | (uintptr_t)advantage) % 4)
            return set_error(OB200_ERR_INVALID, "%s: action, old_logp or advantage is null or not aligned", who);
        if (ref_logits) {
            const int es = elem_bytes(rows->dtype);
            if ((uintptr_t)ref_logits % es || !pitch_fits(ref_pitch, r.A, r.n))
                return set_error(OB200_ERR_INVALID, "%s: ref_logits is not aligned, its pitch is below n_actions, or it goes too far", who);
            if (rows_meet(r.grad, r.g_pitch, es, ref_logits, ref_pitch, es, r.n, r.A))
                return set_error(OB200_ERR_INVALID, "%s: grad overlaps ref_logits", who);
        }
        r.x = ref_logits; r.x_pitch = ref_pitch;
        r.action = action; r.old_logp = old_logp; r.advantage = advantage;
        if (int rc = check_vectors(who, r, elem_bytes(rows->dtype), elem_bytes(rows->dtype))) return rc;
    }
    if (int rc = require_device()) return rc;
    if (rows->n == 0) return OB200_OK;
    r.lo = 1.f - clip_low; r.hi = 1.f + clip_high; r.kl = kl_coef; r.entropy = entropy_coef;
    find_phase(&r, rows->dtype, elem_bytes(rows->dtype));
    return launch_rows(ref_logits ? kClippedRef : kClipped, r, rows->dtype, as_stream(stream));
}

}  // extern "C"
