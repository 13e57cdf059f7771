// Entry points of the selective state space scan: argument checks, the choice between whole
// utterances and pieces of them, and the division of the caller's workspace (kernels: ssm_scan.h).
#include "ssm_scan.h"

namespace {

// States of a wave: 4 S.
int block_states(int states) { return states <= 4 ? 4 : states <= 8 ? 8 : states <= 16 ? 16 : states <= 32 ? 32 : 64; }

// Channels of a lane, at most (params_for takes one where two leave too few waves).
int most_wide(int states) { return states <= 4 ? 4 : states <= 16 ? 2 : 1; }

int64_t round_up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

int check_scan(srx_handle_t h, const srx_scan_t* s, int64_t utts, int64_t frames, const char* who) {
    SRX_REQUIRE(h != nullptr, "%s: NULL context", who);
    SRX_REQUIRE(s != nullptr, "%s: scan is NULL", who);
    SRX_REQUIRE(s->n_channels >= 1 && s->n_groups >= 1 && s->n_channels % s->n_groups == 0,
                "%s: Shape mismatch (n_channels=%d n_groups=%d)", who, s->n_channels, s->n_groups);
    SRX_REQUIRE(s->n_channels <= kMostColumns, "%s: n_channels %d above 2^24", who, s->n_channels);
    SRX_REQUIRE(s->n_states >= 1 && s->n_states <= 64, "%s: n_states %d outside [1, 64]", who, s->n_states);
    SRX_REQUIRE(s->A != nullptr, "%s: NULL A", who);
    SRX_REQUIRE(utts >= 0 && frames >= 0, "%s: negative size", who);
    return SRX_OK;
}

// A wave reaches its rows with 32-bit offsets from the first: 4 rows of the channels' matrices, 16 of B and C.
bool pitch_fits(int64_t ld, int64_t width, int dtype, int rows) {
    const int64_t size = dtype == SRX_F32 ? 4 : 2;
    return ld < ((int64_t)1 << 32) && ((rows - 1) * ld + width) * size <= 0xffffffffll;
}

int check_inputs(const srx_scan_t* s, const srx_scan_inputs_t* in, int dtype, int64_t frames, const char* who) {
    SRX_REQUIRE(frame_dtype(dtype), "%s: unknown dtype %d", who, dtype);
    SRX_REQUIRE(in != nullptr, "%s: inputs are NULL", who);
    if (frames == 0) return SRX_OK;
    const int64_t c = s->n_channels, bc = (int64_t)s->n_groups * s->n_states;
    SRX_REQUIRE(in->x && in->dt && in->B && in->C, "%s: NULL input", who);
    SRX_REQUIRE(in->ld_x >= c && in->ld_dt >= c && in->ld_B >= bc && in->ld_C >= bc &&
                    (in->gate == nullptr || in->ld_gate >= c),
                "%s: a row pitch is smaller than its row", who);
    SRX_REQUIRE(pitch_fits(in->ld_x, s->n_channels, dtype, 4) && pitch_fits(in->ld_dt, s->n_channels, dtype, 4) && pitch_fits(in->ld_B, bc, dtype, 16) &&
                    pitch_fits(in->ld_C, bc, dtype, 16) && (in->gate == nullptr || pitch_fits(in->ld_gate, s->n_channels, dtype, 4)),
                "%s: a row pitch of about 2^30 bytes (B, C: 2^28) or more", who);
    return SRX_OK;
}

ScanParams params_for(const srx_context* h, const srx_scan_t* s, int64_t utts, int64_t frames) {
    ScanParams p;
    memset(&p, 0, sizeof(p));
    p.A = s->A;
    p.skip = s->skip;
    p.bias = s->dt_bias;
    p.softplus = s->softplus;
    p.channels = s->n_channels;
    p.states = s->n_states;
    p.groups = s->n_groups;
    p.per_group = s->n_channels / s->n_groups;
    p.utts = utts;
    p.frames = frames;
    const int64_t simds = (int64_t)h->n_cu * 4;
    auto blocks_of = [&](int wide) { return (int64_t)s->n_groups * ((p.per_group + 16 * wide - 1) / (16 * wide)); };
    // Two channels a lane, or one where two leave too few waves (the work beside the exponentials is smaller for
    // two) and from 17 states on, whose registers leave no room for more.  Utterances of 200 frames x 1024 channels, 16
    // states, forward and backward: 32 of them 173 us with two and 158 with one, 64 of them 261 and 300.
    p.wide = most_wide(s->n_states);
    if (s->n_states > 8 && utts * blocks_of(2) < 2 * simds) p.wide = 1;
    p.group_blocks = (p.per_group + 16 * p.wide - 1) / (16 * p.wide);
    p.blocks = p.group_blocks * s->n_groups;
    // Whole utterances where they alone give every SIMD a wave; else pieces, whose states are computed twice: shorter ones
    // where even those leave SIMDs without a wave, and only of utterances long enough for it -- the longest of several
    // is taken to have twice the mean.  512 channels, 16 states, one utterance, forward (and with the backward pass): 100
    // frames whole 19 us (67), in pieces 24 (69); 300 frames 43 (158) and 24 (69), in pieces of 64 28 (81).
    // The lengths are the device's: a long utterance among many short ones is not cut (63 of 100 to 300 frames and one of
    // 24,001, 1536 channels, forward: 5.0 ms; the long one alone, in pieces, 0.29).
    p.segment = 0;
    p.units = utts;
    if (utts > 0 && utts * p.blocks < simds) {           // (so never with two channels a lane and 16 states)
        const int64_t even = frames * p.blocks / (4 * simds), least = frames * p.blocks < 64 * simds ? 32 : 64;
        const int64_t segment = round_up(even > least ? even : least, 16);
        if ((utts == 1 ? frames : 2 * (frames / utts)) > 7 * segment / 2) {
            p.segment = segment;
            p.units = frames / segment + utts;
        }
    }
    // By falling length where there are more waves than run at full rate at once (fewer do not wait for one another),
    // utterances to choose from, but not so many that the last ones do not matter, and long enough to be worth it.
    p.ordered = p.segment == 0 && utts >= kScanOrderedLeast && utts <= kScanOrdered && frames >= 32 * utts &&
                utts * p.blocks >= 2 * simds;
    const int64_t round = h->n_cu / ((p.blocks + kScanWaves - 1) / kScanWaves);
    p.round = (int)(round > 1 ? round : 1);
    // backward: a wave sums the parameters' gradients over all its units (every parts-th of them: long and short ones)
    p.parts = p.units;
    const int64_t enough = 8 * simds / p.blocks + 1;
    if (p.segment == 0 && p.parts > enough) p.parts = enough;
    if (p.parts < 1) p.parts = 1;
    return p;
}

int64_t saved_states(const srx_scan_t* s, int64_t utts, int64_t frames) {
    const int64_t ch = 16 * most_wide(s->n_states), per = s->n_channels / s->n_groups;      // (room for every way to cut the channels)
    return (frames / kScanSaveEvery + utts) * ((per + ch - 1) / ch * s->n_groups) * ch * block_states(s->n_states);
}

// Hands out the workspace; with a NULL base it only counts.
struct Carver {
    char* base;
    int64_t used = 0;
    float* floats(int64_t n) {
        float* at = base != nullptr ? (float*)(base + used) : nullptr;
        used += round_up(n * 4, 256);
        return at;
    }
};

int64_t carve(ScanParams& p, bool backward, void* workspace) {
    Carver c{(char*)workspace};
    const int64_t ch = 16 * p.wide, ns = block_states(p.states);
    if (p.segment != 0) {
        p.seg_state = c.floats(p.units * p.blocks * ch * ns);
        p.seg_sum = c.floats(p.units * p.blocks * ch);
    } else if (p.ordered && p.saved == nullptr) {
        p.order = (int*)c.floats(p.utts);
    }
    if (backward) {
        p.part_A = c.floats(p.parts * p.blocks * ch * ns);
        p.part_vec = c.floats(p.parts * p.blocks * 2 * ch);
        p.part_bc = c.floats(p.blocks * p.frames * 2 * ns);
    }
    return c.used;
}

int run(const ScanParams& p, int dtype, bool backward, hipStream_t st) {
    switch (dtype) {
        case SRX_F32: return scan_run<float>(p, backward, st);
        case SRX_BF16: return scan_run<__bf16>(p, backward, st);
        default: return scan_run<_Float16>(p, backward, st);
    }
}

void take_inputs(ScanParams& p, const srx_scan_inputs_t* in) {
    p.x = in->x;
    p.dt = in->dt;
    p.B = in->B;
    p.C = in->C;
    p.gate = in->gate;
    p.ld_x = in->ld_x;
    p.ld_dt = in->ld_dt;
    p.ld_B = in->ld_B;
    p.ld_C = in->ld_C;
    p.ld_gate = in->ld_gate;
}

int64_t workspace_bytes_for(srx_handle_t h, const srx_scan_t* s, int64_t utts, int64_t frames, bool backward,
                            const char* who) {
    if (check_scan(h, s, utts, frames, who)) return -1;
    ScanParams p = params_for(h, s, utts, frames);
    return carve(p, backward, nullptr);
}

}  // namespace

extern "C" {

int64_t srx_selective_scan_saved(const srx_scan_t* s, int64_t n_utts, int64_t n_frames) {
    if (s == nullptr || s->n_channels < 1 || s->n_groups < 1 || s->n_states < 1 || s->n_states > 64 ||
        s->n_channels % s->n_groups != 0 || n_utts < 0 || n_frames < 0) {
        srx_set_error("srx_selective_scan_saved: Shape mismatch");
        return -1;
    }
    const bool order = n_utts >= kScanOrderedLeast && n_utts <= kScanOrdered;      // (room for it behind the states)
    return saved_states(s, n_utts, n_frames) + (order ? n_utts : 0);
}

int64_t srx_selective_scan_workspace(srx_handle_t h, const srx_scan_t* s, int64_t n_utts, int64_t n_frames) {
    return workspace_bytes_for(h, s, n_utts, n_frames, false, "srx_selective_scan_workspace");
}

int64_t srx_selective_scan_backward_workspace(srx_handle_t h, const srx_scan_t* s, int64_t n_utts,
                                              int64_t n_frames) {
    return workspace_bytes_for(h, s, n_utts, n_frames, true, "srx_selective_scan_backward_workspace");
}

int srx_selective_scan(srx_handle_t h, const srx_scan_t* s, const srx_scan_inputs_t* in, int dtype,
                       const int64_t* utt_offsets, int64_t n_utts, int64_t n_frames, const float* state_in,
                       float* state_out, void* y, int64_t ld_y, float* saved, void* workspace,
                       int64_t workspace_bytes, void* stream) {
    const char* who = "srx_selective_scan";
    const bool zero = take_zero_rows(dtype) && n_frames > 0;
    int rc = check_scan(h, s, n_utts, n_frames, who);
    if (rc) return rc;
    if ((rc = check_inputs(s, in, dtype, n_frames, who))) return rc;
    if (n_utts == 0 && !zero) return SRX_OK;
    SRX_REQUIRE(n_utts == 0 || utt_offsets != nullptr, "%s: NULL utterance offsets", who);
    SRX_REQUIRE(n_frames == 0 || y != nullptr, "%s: NULL y", who);
    SRX_REQUIRE(n_frames == 0 || (ld_y >= s->n_channels && pitch_fits(ld_y, s->n_channels, dtype, 4)),
                "%s: a row pitch is smaller than its row, or 2^30 bytes or more", who);
    ScanParams p = params_for(h, s, n_utts, n_frames);
    p.clear = zero ? kClearGroups : 0;
    p.saved = saved;
    if (saved != nullptr && p.ordered) p.order = (int*)(saved + saved_states(s, n_utts, n_frames));
    const int64_t need = carve(p, false, workspace);
    SRX_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need),
                "%s: workspace of %lld bytes, %lld are needed", who, (long long)workspace_bytes, (long long)need);
    take_inputs(p, in);
    p.off = utt_offsets;
    p.state_in = state_in;
    p.state_out = state_out;
    p.y = y;
    p.ld_y = ld_y;
    DeviceGuard guard(h->device);
    if (guard.rc) return guard.rc;
    return run(p, dtype, false, (hipStream_t)stream);
}

int srx_selective_scan_step(srx_handle_t h, const srx_scan_t* s, const srx_scan_inputs_t* in, int dtype,
                            int64_t n_rows, float* state, void* y, int64_t ld_y, void* stream) {
    const char* who = "srx_selective_scan_step";
    int rc = check_scan(h, s, n_rows, n_rows, who);
    if (rc) return rc;
    if ((rc = check_inputs(s, in, dtype, n_rows, who))) return rc;
    if (n_rows == 0) return SRX_OK;
    SRX_REQUIRE(state != nullptr && y != nullptr, "%s: NULL state or y", who);
    SRX_REQUIRE(ld_y >= s->n_channels, "%s: a row pitch is smaller than its row", who);
    ScanParams p = params_for(h, s, n_rows, n_rows);
    take_inputs(p, in);
    p.y = y;
    p.ld_y = ld_y;
    DeviceGuard guard(h->device);
    if (guard.rc) return guard.rc;
    switch (dtype) {
        case SRX_F32: return scan_step_run<float>(p, state, n_rows, (hipStream_t)stream);
        case SRX_BF16: return scan_step_run<__bf16>(p, state, n_rows, (hipStream_t)stream);
        default: return scan_step_run<_Float16>(p, state, n_rows, (hipStream_t)stream);
    }
}

int srx_selective_scan_backward(srx_handle_t h, const srx_scan_t* s, const srx_scan_inputs_t* in, int dtype,
                                const int64_t* utt_offsets, int64_t n_utts, int64_t n_frames,
                                const float* saved, const void* dy, int64_t ld_dy, const float* dstate_out,
                                const srx_scan_gradients_t* grads, float* dA, float* dskip, float* ddt_bias,
                                float* dstate_in, void* workspace, int64_t workspace_bytes, void* stream) {
    const char* who = "srx_selective_scan_backward";
    int rc = check_scan(h, s, n_utts, n_frames, who);
    if (rc) return rc;
    if ((rc = check_inputs(s, in, dtype, n_frames, who))) return rc;
    const int64_t c = s->n_channels, bc = (int64_t)s->n_groups * s->n_states;
    SRX_REQUIRE(grads != nullptr && dA != nullptr, "%s: NULL gradients", who);
    SRX_REQUIRE((dskip != nullptr) == (s->skip != nullptr) && (ddt_bias != nullptr) == (s->dt_bias != nullptr),
                "%s: dskip / ddt_bias must be given exactly where skip / dt_bias are", who);
    SRX_REQUIRE(n_utts == 0 || utt_offsets != nullptr, "%s: NULL utterance offsets", who);
    if (n_frames > 0) {
        SRX_REQUIRE((saved != nullptr || n_utts == 0) && dy != nullptr, "%s: NULL saved or dy", who);
        SRX_REQUIRE(grads->dx && grads->ddt && grads->dB && grads->dC &&
                        (in->gate == nullptr) == (grads->dgate == nullptr),
                    "%s: NULL gradient of an input (dgate must be given exactly where gate is)", who);
        SRX_REQUIRE(ld_dy >= c && grads->ld_dx >= c && grads->ld_ddt >= c && grads->ld_dB >= bc &&
                        grads->ld_dC >= bc && (in->gate == nullptr || grads->ld_dgate >= c),
                    "%s: a row pitch is smaller than its row", who);
        SRX_REQUIRE(pitch_fits(ld_dy, s->n_channels, dtype, 4) && pitch_fits(grads->ld_dx, s->n_channels, dtype, 4) &&
                        pitch_fits(grads->ld_ddt, s->n_channels, dtype, 4) && (in->gate == nullptr || pitch_fits(grads->ld_dgate, s->n_channels, dtype, 4)),
                    "%s: a row pitch of 2^30 bytes or more", who);
    }
    ScanParams p = params_for(h, s, n_utts, n_frames);
    p.clear = n_frames > 0 ? kClearGroups : 0;
    p.saved = const_cast<float*>(saved);     // (the backward kernels only read it)
    if (p.ordered) p.order = (int*)(p.saved + saved_states(s, n_utts, n_frames));
    const int64_t need = carve(p, true, workspace);
    SRX_REQUIRE(workspace != nullptr && workspace_bytes >= need,
                "%s: workspace of %lld bytes, %lld are needed", who, (long long)workspace_bytes, (long long)need);
    take_inputs(p, in);
    p.off = utt_offsets;
    p.dy = dy;
    p.ld_dy = ld_dy;
    p.dx = grads->dx;
    p.ddt = grads->ddt;
    p.dB = grads->dB;
    p.dC = grads->dC;
    p.dgate = grads->dgate;
    p.ld_dx = grads->ld_dx;
    p.ld_ddt = grads->ld_ddt;
    p.ld_dB = grads->ld_dB;
    p.ld_dC = grads->ld_dC;
    p.ld_dgate = grads->ld_dgate;
    p.dA = dA;
    p.dskip = dskip;
    p.dbias = ddt_bias;
    p.dstate_in = dstate_in;
    p.dstate_out = dstate_out;
    DeviceGuard guard(h->device);
    if (guard.rc) return guard.rc;
    return run(p, dtype, true, (hipStream_t)stream);
}

}  // extern "C"
