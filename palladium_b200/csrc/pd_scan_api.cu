// pd_scan_api.cu -- the C-ABI side of the state-space families: parameter
// checks, buffer sizes, launch geometry and scratch of a call (pd_scan_plan) and
// its launch (pd_scan_launch).  Called by pd_api.cu, which owns streams and pools.
#include "../../include/palladium_cuda.h"
#include "pd_scan.h"

#include <math.h>
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

namespace {

int fail(char* err, size_t cap, const char* fmt, ...) {
    if (err && cap) {
        va_list ap;
        va_start(ap, fmt);
        vsnprintf(err, cap, fmt, ap);
        va_end(ap);
    }
    return PD_ERR_INVALID_ARGUMENT;
}

bool is_conv(int family) { return family >= PD_FAMILY_CAUSAL_CONV && family <= PD_FAMILY_CAUSAL_CONV_GRAD; }
size_t element(int64_t type) { return type == PD_TYPE_F32 ? 4 : 2; }
int64_t align256(int64_t v) { return (v + 255) / 256 * 256; }
bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
bool flag(int64_t v) { return v == 0 || v == 1; }

struct Dims {
    int64_t seqs, channels, rows;   // rows of the token arrays
    size_t cells;                   // rows * channels
};

// `what`: the family's name in messages
int dims_of(const char* what, const int64_t grid[3], int64_t length, int64_t packed, bool step, int64_t type, Dims* d,
            char* err, size_t cap) {
    const int64_t kMost = INT32_MAX;
    if (type < PD_TYPE_F32 || type > PD_TYPE_BF16) return fail(err, cap, "%s: type must be 0, 1 or 2", what);
    if (!flag(packed)) return fail(err, cap, "%s: flags must be 0 or 1", what);
    if (grid[2] > 1) return fail(err, cap, "%s: grid must be (sequences, channels)", what);
    if (grid[0] > kMost || grid[1] < 1 || grid[1] > (1 << 20))
        return fail(err, cap, "%s: grid (%lld, %lld) must hold at most 2^31 - 1 sequences and 1 to 2^20 channels", what,
                    (long long)grid[0], (long long)grid[1]);
    if (!step && (length < 0 || length > kMost)) return fail(err, cap, "%s: length must lie in [0, 2^31)", what);
    d->seqs = grid[0];
    d->channels = grid[1];
    d->rows = step ? d->seqs : packed ? length : d->seqs * length;
    if (d->rows > ((int64_t)1 << 40) / d->channels || d->seqs > ((int64_t)1 << 40) / (d->channels * 64))
        return fail(err, cap, "%s: more than 2^40 elements per call", what);
    d->cells = (size_t)d->rows * (size_t)d->channels;
    return PD_OK;
}

// Rows per thread of the convolution.  A run re-reads width - 1 rows of its predecessor (from L2), so long runs
// move less; 1024 threads per SM run at a time, so a call is cut into as few whole waves of them as give runs of
// at most 128 rows.
int conv_run(int64_t rows, int64_t lanes, int sms) {
    const int64_t wave = (int64_t)sms * 1024, each = (rows * lanes + wave - 1) / wave;
    const int64_t waves = (each + 127) / 128;
    const int64_t run = waves ? (rows * lanes + waves * wave - 1) / (waves * wave) : 1;
    return run < 4 ? 4 : (int)run;
}
// Channels per thread of the convolutions: four.  (Eight bf16 channels, 16 bytes, leave registers for two blocks per
// SM instead of four: 8 x 2048 x 4096 took 76 us against 67 before the runs were cut into whole waves, 61 since.)
int conv_vector(int64_t channels) { return channels % 4 == 0 ? 4 : 1; }
// The gradient's blocks: 32 threads across channels, eight runs of rows side by side.  Enough rows of blocks for
// about two blocks per SM, each of which writes one partial sum of dweight, and runs as long as that asks for.
void conv_grad_blocks(int64_t rows, int64_t extra, int64_t lanes, int sms, int* run, int64_t* row_blocks) {
    const int64_t columns = (lanes + 31) / 32;
    int64_t blocks = (int64_t)sms * 2 / columns;
    if (blocks < 1) blocks = 1;
    int64_t n = (rows + 8 * blocks - 1) / (8 * blocks);
    if (n < 8) n = 8;
    *run = (int)(n > (1 << 20) ? 1 << 20 : n);
    const int64_t jobs = (rows + *run - 1) / *run + extra;
    blocks = (jobs + 7) / 8;
    *row_blocks = blocks < 1 ? 1 : blocks > 65535 ? 65535 : blocks;
}
int64_t conv_partial(const Dims& d, int64_t width, int64_t row_blocks) { return row_blocks * d.channels * (width + 1) * 4; }

int64_t scan_chunks(const pd_selective_scan_params* p, const Dims& d) {
    return p->packed ? p->length / PD_SCAN_CHUNK + d.seqs : d.seqs * ((p->length + PD_SCAN_CHUNK - 1) / PD_SCAN_CHUNK);
}
// Channels a warp of the gradient kernel takes one after another (a block is four warps, three blocks an SM where
// shared memory allows).  More of them share one sum over the block's warps and one partial sum of dB and dC in memory,
// worth about one channel's work per chunk, two with more than sixteen states; fewer give more blocks.  The smallest
// product of waves and work per wave wins, where a wave of two blocks an SM takes nine tenths of one of three, and one
// of one block eight tenths (4 x 2048 tokens x 2048 channels, one to six channels a warp: bf16 x 16 states 1060, 794,
// 744, 767, 687, 763 us, of which it takes 687; float32 x 16 states 1031, 765, 716, 751, 810, 908, of which 716).
int grad_per_warp(const pd_selective_scan_params* p, const Dims& d, int sms) {
    const int64_t per = d.channels / p->groups;
    const int most = p->state > 16 ? 4 : 6;    // (more were not measured)
    int best = 1;
    int64_t least = INT64_MAX;
    for (int n = most; n >= 1; --n) {
        const int fit = pd_scan_resident(pd_scan_grad_bytes((int)p->state, n, (int)element(p->type)));
        const int64_t slots = (int64_t)sms * (fit < 3 ? fit : 3), wave = fit >= 3 ? 10 : fit == 2 ? 9 : 8;
        const int64_t blocks = (per + 4 * n - 1) / (4 * n) * p->groups * (d.seqs > 0 ? d.seqs : 1);
        const int64_t cost = (blocks + slots - 1) / slots * (n + (p->state > 16 ? 2 : 1)) * wave;
        if (cost < least) { least = cost; best = n; }
    }
    return best;
}
// How many blocks of a packed call, per tile of channels, clear the rows of no sequence, which only the device knows:
// one for every 128 KB that a token array holds, two per SM at most.
int64_t scan_free_blocks(const pd_selective_scan_params* p, const Dims& d, int64_t tiles, int sms) {
    if (!p->packed) return 0;
    const int64_t most = (int64_t)sms * 2, want = (int64_t)(d.cells * element(p->type) >> 17) + 1;
    return ((want < most ? want : most) + tiles - 1) / tiles;
}
int64_t scan_tiles(const pd_selective_scan_params* p, const Dims& d, int per_lane) {
    const int64_t per = d.channels / p->groups, ch = 2 * 32 / pd_scan_lanes((int)p->state) * per_lane;
    return (per + ch - 1) / ch * p->groups;
}
// The prompt kernel's channels per lane and segments.  Two channels per lane halve the reads of B and C, one gives
// twice the blocks and more of them on an SM (2-byte tokens, 16 states: five instead of three): two from 12 blocks per SM on (16 x 1024 tokens x 4096
// channels x 16 states: 571 against 604 us; 4 x 2048 x 2048: 211 against 182).  Cutting a sequence into segments
// costs a first pass over all but its last, which takes two thirds of the second's time: it pays where a call has
// fewer than two blocks per SM (1 x 8192 x 2048: 16 segments 252 us; 4 x 2048 x 2048: uncut 182 us,
// two segments 236).  A block composes the states of all segments before its own, one after another, so a sequence is
// cut into half the root of its length at most (1 x 131072 x 16 bf16 in 2048, 512, 181, 128, 64 segments: 1106, 188, 136,
// 120, 173 us; 1 x 2^20 x 16 in 2072, 512, 128: 1384, 419, 622).  A packed call is cut at three times an even share, so that one long sequence does not
// outlast all others (17 of them, 8200 x 2560: 249 us, cut at 1024 tokens 298).
void scan_cut(const pd_selective_scan_params* p, const Dims& d, int sms, PdScanPlan* plan) {
    const int64_t seqs = d.seqs > 0 ? d.seqs : 1, rows = d.rows > 0 ? d.rows : 1, mean = (rows + seqs - 1) / seqs;
    const int64_t root = (int64_t)(sqrt((double)mean) / 2), least = mean / 64;
    const int64_t most = least < 1 ? 1 : least < root ? least : root;
    const int per_lane = p->state > 32 || (p->state > 8 && scan_tiles(p, d, 2) * seqs >= (int64_t)sms * 12) ? 2 : 1;
    const int64_t tiles = scan_tiles(p, d, per_lane);
    int64_t cuts = tiles * seqs < sms * 2 ? (int64_t)sms * 14 / (tiles * seqs) : 1, segment = INT32_MAX;
    if (cuts > most) cuts = most;
    if (cuts > 1) {
        segment = (mean + cuts - 1) / cuts;
        const int64_t floor = (int64_t)sqrt((double)rows);
        // (one sequence may have nearly all the rows: 131072 tokens and 63 x 16 beside them, 16 channels, took 601 us
        // without this floor and take 151; 64 x 2048 tokens 62 either way)
        if (p->packed && segment < floor) segment = floor;
    }
    if (cuts <= 1 && p->packed) segment = rows * tiles / ((int64_t)sms * 4) * 3;
    if (segment < 64) segment = 64;
    segment = (segment + PD_SCAN_CHUNK - 1) / PD_SCAN_CHUNK * PD_SCAN_CHUNK;     // (carries are kept at whole chunks)
    plan->items = per_lane;
    plan->segment = segment;
    if (p->packed) plan->segments = d.rows / segment + d.seqs;
    else plan->segments = d.seqs * (p->length > segment ? (p->length + segment - 1) / segment : 1);
}

int64_t scan_partial_bc(const pd_selective_scan_params* p, const Dims& d, int sms) {
    const int64_t per = d.channels / p->groups, ch = 4 * grad_per_warp(p, d, sms);
    return align256((per + ch - 1) / ch * p->groups * d.rows * 2 * pd_scan_pad((int)p->state) * 4);
}

int plan_conv(int family, const pd_causal_conv_params* p, const int64_t grid[3], int sms, PdScanPlan* plan, char* err,
              size_t cap) {
    const bool step = family == PD_FAMILY_CAUSAL_CONV_STEP, grad = family == PD_FAMILY_CAUSAL_CONV_GRAD;
    const char* what = step ? "causal_conv_step" : grad ? "causal_conv_grad" : "causal_conv";
    Dims d;
    int rc = dims_of(what, grid, p->length, p->packed, step, p->type, &d, err, cap);
    if (rc) return rc;
    if (p->width < 2 || p->width > 4) return fail(err, cap, "%s: width must lie in [2, 4], got %lld", what, (long long)p->width);
    if (!flag(p->silu) || !flag(p->bias) || !flag(p->initial) || !flag(p->final))
        return fail(err, cap, "%s: flags must be 0 or 1", what);
    const size_t e = element(p->type), D = (size_t)d.channels, tokens = d.cells * e;
    const size_t edge = (size_t)d.seqs * (size_t)(p->width - 1) * D * e, weight = D * (size_t)p->width * 4, vec = D * 4;
    const size_t offsets = ((size_t)d.seqs + 1) * 4;
    std::vector<size_t>&in = plan->in_bytes, &out = plan->out_bytes;
    const int64_t lanes = d.channels / conv_vector(d.channels);
    if (step) {
        in = {tokens, edge, weight};
        if (p->bias) in.push_back(vec);
        out = {tokens, edge};
        plan->kernel_name = "pd_causal_conv_step_kernel";
        plan->block = 128;
        plan->grid = (lanes + 127) / 128;
        plan->grid_y = d.seqs < 65535 ? d.seqs : 65535;
        return PD_OK;
    }
    in = {tokens, weight};
    if (grad) in.insert(in.begin(), tokens);
    if (p->bias) in.push_back(vec);
    if (p->initial) in.push_back(edge);
    if (grad && p->final) in.push_back(edge);
    if (p->packed) in.push_back(offsets);
    const int run = conv_run(d.rows, lanes, sms);
    const int64_t runs = (d.rows + run - 1) / run;
    plan->items = run;
    plan->block = 256;
    if (!grad) {
        out = {tokens};
        if (p->final) out.push_back(edge);
        plan->kernel_name = "pd_causal_conv_kernel";
        plan->grid = ((runs + (p->final ? d.seqs : 0)) * lanes + 255) / 256;
        return PD_OK;
    }
    out = {tokens, weight};
    if (p->bias) out.push_back(vec);
    if (p->initial) out.push_back(edge);
    plan->kernel_name = "pd_causal_conv_grad_kernel";
    int grad_run;
    conv_grad_blocks(d.rows, p->initial ? d.seqs : 0, lanes, sms, &grad_run, &plan->row_blocks);
    plan->items = grad_run;
    plan->grid = (lanes + 31) / 32;
    plan->grid_y = plan->row_blocks;
    plan->launches = 2;
    plan->scratch_bytes = conv_partial(d, p->width, plan->row_blocks);
    plan->dynamic_smem = 256 * conv_vector(d.channels) * 4;
    return PD_OK;
}

int plan_scan(int family, const pd_selective_scan_params* p, const int64_t grid[3], int sms, PdScanPlan* plan, char* err,
              size_t cap) {
    const bool step = family == PD_FAMILY_SELECTIVE_SCAN_STEP, grad = family == PD_FAMILY_SELECTIVE_SCAN_GRAD;
    const char* what = step ? "selective_scan_step" : grad ? "selective_scan_grad" : "selective_scan";
    Dims d;
    int rc = dims_of(what, grid, p->length, p->packed, step, p->type, &d, err, cap);
    if (rc) return rc;
    if (p->state < 1 || p->state > PD_SCAN_MAX_STATE)
        return fail(err, cap, "%s: state must lie in [1, %d], got %lld", what, PD_SCAN_MAX_STATE, (long long)p->state);
    if (p->groups > 65535) return fail(err, cap, "%s: more than 65535 groups", what);
    if (p->groups < 1 || d.channels % p->groups != 0)
        return fail(err, cap, "%s: %lld channels do not divide into %lld groups", what, (long long)d.channels, (long long)p->groups);
    if (!flag(p->softplus) || !flag(p->bias) || !flag(p->skip) || !flag(p->gate) || !flag(p->initial) || !flag(p->final) ||
        !flag(p->carries))
        return fail(err, cap, "%s: flags must be 0 or 1", what);
    const size_t e = element(p->type), D = (size_t)d.channels, N = (size_t)p->state, tokens = d.cells * e;
    const size_t coupling = (size_t)d.rows * (size_t)p->groups * N * e, rates = D * N * 4, vec = D * 4;
    const size_t edge = (size_t)d.seqs * D * N * 4, offsets = ((size_t)d.seqs + 1) * 4;
    const size_t carries = (size_t)scan_chunks(p, d) * D * N * 4;
    std::vector<size_t>&in = plan->in_bytes, &out = plan->out_bytes;
    in = {tokens, tokens, rates, coupling, coupling};
    if (step) in.insert(in.begin(), edge);
    if (grad) in.insert(in.begin(), tokens);
    if (p->bias) in.push_back(vec);
    if (p->skip) in.push_back(vec);
    if (p->gate) in.push_back(tokens);
    plan->block = 128;
    if (step) {
        out = {tokens, edge};
        plan->kernel_name = "pd_selective_scan_step_kernel";
        plan->grid = pd_step_blocks(d.channels, (int)p->groups, (int)p->state, d.seqs);
        plan->items = pd_step_run(d.channels, (int)p->groups, (int)p->state, d.seqs, sms);
        plan->grid_y = (d.seqs + plan->items - 1) / plan->items;
        plan->block = 32 * pd_step_warps(d.channels, (int)p->groups, (int)p->state, d.seqs);
        return PD_OK;
    }
    if (grad) {
        // one block per tile of channels and sequence
        const int64_t per = d.channels / p->groups;
        plan->items = grad_per_warp(p, d, sms);
        const int64_t tiles = (per + 4 * plan->items - 1) / (4 * plan->items) * p->groups;
        plan->dynamic_smem = pd_scan_grad_bytes((int)p->state, (int)plan->items, (int)e);
        plan->free_blocks = scan_free_blocks(p, d, 1, sms);      // (in the launch that adds up the parameters' sums)
        plan->grid = tiles * d.seqs;
    } else {
        scan_cut(p, d, sms, plan);
        const int64_t tiles = scan_tiles(p, d, (int)plan->items);
        plan->dynamic_smem = PdScanShape(pd_scan_lanes((int)p->state), (int)plan->items, (int)e).bytes;
        plan->free_blocks = scan_free_blocks(p, d, tiles, sms);
        plan->grid = tiles * (plan->segments + plan->free_blocks);
        plan->block = 128;
        if (d.rows > plan->segment) {
            // (a dense call is cut only where a sequence is longer than a segment)
            if (p->packed || p->length > plan->segment) {
                plan->totals_offset = align256(plan->segments * d.channels * p->state * 4);
                plan->scratch_bytes = plan->totals_offset + plan->segments * d.channels * 4;
                plan->launches = 2;
            }
        }
    }
    if (grad) {
        in.push_back(carries);
        if (p->final) in.push_back(edge);
        out = {tokens, tokens, rates, coupling, coupling};
        if (p->bias) out.push_back(vec);
        if (p->skip) out.push_back(vec);
        if (p->gate) out.push_back(tokens);
        if (p->initial) out.push_back(edge);
        plan->kernel_name = "pd_selective_scan_grad_kernel";
        plan->launches = 3;
        plan->params_offset = scan_partial_bc(p, d, sms);
        plan->scratch_bytes = plan->params_offset + d.seqs * d.channels * (p->state + 2) * 4;
    } else {
        if (p->initial) in.push_back(edge);
        out = {tokens};
        if (p->final) out.push_back(edge);
        if (p->carries) out.push_back(carries);
        plan->kernel_name = "pd_selective_scan_kernel";
    }
    if (p->packed) in.push_back(offsets);
    return PD_OK;
}

}  // namespace

bool pd_is_scan_family(int family) { return family >= PD_FAMILY_CAUSAL_CONV && family <= PD_FAMILY_SELECTIVE_SCAN_GRAD; }

int pd_scan_plan(int family, const void* params, size_t params_bytes, const int64_t grid[3], const int64_t block[3],
                 int sms, PdScanPlan* plan, char* err, size_t err_cap) {
    const size_t want = is_conv(family) ? sizeof(pd_causal_conv_params) : sizeof(pd_selective_scan_params);
    if (!params || params_bytes != want)
        return fail(err, err_cap, "state-space family: params block must be %zu bytes, got %zu", want, params ? params_bytes : (size_t)0);
    if (block && (block[0] > 0 || block[1] > 0 || block[2] > 0))
        return fail(err, err_cap, "state-space family: the library chooses the threadgroup; leave it unset");
    int rc = is_conv(family) ? plan_conv(family, static_cast<const pd_causal_conv_params*>(params), grid, sms, plan, err, err_cap)
                             : plan_scan(family, static_cast<const pd_selective_scan_params*>(params), grid, sms, plan, err, err_cap);
    if (rc == PD_OK && plan->grid > INT32_MAX) rc = fail(err, err_cap, "state-space family: the call needs more than 2^31 - 1 blocks");
    return rc;
}

int pd_scan_overlap(int family, int n_in, const void* const* in, const size_t* in_bytes, int n_out, void* const* out,
                    const size_t* out_bytes, char* err, size_t err_cap) {
    // the state of a step: operand 1 of the convolution's, 0 of the scan's; result 1 of both
    const int state = family == PD_FAMILY_CAUSAL_CONV_STEP ? 1 : family == PD_FAMILY_SELECTIVE_SCAN_STEP ? 0 : -1;
    auto meet = [](const void* p, size_t n, const void* q, size_t m) {
        const uintptr_t a = reinterpret_cast<uintptr_t>(p), b = reinterpret_cast<uintptr_t>(q);
        return n && m && a < b + m && b < a + n;
    };
    for (int o = 0; o < n_out; ++o) {
        for (int i = 0; i < n_in; ++i)
            if (meet(out[o], out_bytes[o], in[i], in_bytes[i]) && !(o == 1 && i == state && out[o] == in[i]))
                return fail(err, err_cap, "output %d shares memory with input %d", o, i);
        for (int p = 0; p < o; ++p)
            if (meet(out[o], out_bytes[o], out[p], out_bytes[p]))
                return fail(err, err_cap, "output %d shares memory with output %d", o, p);
    }
    return PD_OK;
}

namespace {
// (report: the kernel is described instead, and no pointer is read)
int scan_launch(int family, const void* params, int math_mode, const int64_t grid[3], const PdScanPlan& plan,
                const void* const* in, void* const* out, void* scratch, cudaStream_t st, PdScanReport* report, char* err,
                size_t err_cap) {
    const PdScanTable* table = math_mode == PD_MATH_SAFE ? pd_scan_table_safe()
                               : math_mode == PD_MATH_RELAXED ? pd_scan_table_relaxed() : pd_scan_table_fast();
    cudaError_t e;
    int i = 0, o = 0;
    if (is_conv(family)) {
        const pd_causal_conv_params* p = static_cast<const pd_causal_conv_params*>(params);
        PdConvArgs a;
        memset(&a, 0, sizeof(a));
        a.report = report;
        const bool step = family == PD_FAMILY_CAUSAL_CONV_STEP, grad = family == PD_FAMILY_CAUSAL_CONV_GRAD;
        a.type = (int)p->type;
        a.width = (int)p->width;
        a.silu = (int)p->silu;
        a.channels = grid[1];
        a.tok.seqs = grid[0];
        a.tok.length = p->length;
        a.tok.rows = step ? grid[0] : p->packed ? p->length : grid[0] * p->length;
        a.run = (int)plan.items;
        if (grad) a.dy = in[i++];
        a.x = in[i++];
        if (step) a.initial = in[i++];
        a.weight = (const float*)in[i++];
        if (p->bias) a.bias = (const float*)in[i++];
        if (!step && p->initial) a.initial = in[i++];
        if (grad && p->final) a.dfinal = in[i++];
        if (!step && p->packed) a.tok.offsets = (const int32_t*)in[i++];
        if (grad) {
            a.dx = out[o++];
            a.dweight = (float*)out[o++];
            if (p->bias) a.dbias = (float*)out[o++];
            if (p->initial) a.dinitial = out[o++];
        } else {
            a.y = out[o++];
            if (step || p->final) a.final_state = out[o++];
        }
        a.vec = conv_vector(a.channels);
        const void* tokens[] = {a.x, a.dy, a.initial, a.dfinal, a.y, a.final_state, a.dx, a.dinitial};
        for (const void* t : tokens) if (reinterpret_cast<uintptr_t>(t) % (a.vec * element(p->type))) a.vec = 1;
        if (!aligned16(a.weight) || !aligned16(a.bias)) a.vec = 1;
        a.row_blocks = plan.row_blocks;
        a.partial = (float*)scratch;
        e = step ? table->conv_step(a, st) : grad ? table->conv_grad(a, st) : table->conv(a, st);
    } else {
        const pd_selective_scan_params* p = static_cast<const pd_selective_scan_params*>(params);
        PdScanArgs a;
        memset(&a, 0, sizeof(a));
        a.report = report;
        const bool step = family == PD_FAMILY_SELECTIVE_SCAN_STEP, grad = family == PD_FAMILY_SELECTIVE_SCAN_GRAD;
        a.type = (int)p->type;
        a.state = (int)p->state;
        a.groups = (int)p->groups;
        a.softplus = (int)p->softplus;
        a.channels = grid[1];
        a.tok.seqs = grid[0];
        a.tok.length = p->length;
        a.tok.rows = step ? grid[0] : p->packed ? p->length : grid[0] * p->length;
        if (step) a.initial = (const float*)in[i++];
        if (grad) a.dy = in[i++];
        a.x = in[i++];
        a.delta = in[i++];
        a.A = (const float*)in[i++];
        a.B = in[i++];
        a.C = in[i++];
        if (p->bias) a.bias = (const float*)in[i++];
        if (p->skip) a.skip = (const float*)in[i++];
        if (p->gate) a.z = in[i++];
        if (grad) {
            a.carries_in = (const float*)in[i++];
            if (p->final) a.dfinal = (const float*)in[i++];
            a.dx = out[o++];
            a.ddelta = out[o++];
            a.dA = (float*)out[o++];
            a.dB = out[o++];
            a.dC = out[o++];
            if (p->bias) a.dbias = (float*)out[o++];
            if (p->skip) a.dskip = (float*)out[o++];
            if (p->gate) a.dz = out[o++];
            if (p->initial) a.dinitial = (float*)out[o++];
            a.partial_bc = (float*)scratch;
            a.partial_params = (float*)((char*)scratch + plan.params_offset);
        } else {
            a.segment = plan.segment;
            a.segments = plan.segments;
            if (!step && plan.scratch_bytes > 0) {
                a.ends = (float*)scratch;
                a.totals = (float*)((char*)scratch + plan.totals_offset);
            }
            if (!step && p->initial) a.initial = (const float*)in[i++];
            a.y = out[o++];
            if (step || p->final) a.final_state = (float*)out[o++];
            if (!step && p->carries) a.carries = (float*)out[o++];
        }
        if (!step && p->packed) a.tok.offsets = (const int32_t*)in[i++];
        const size_t four = 4 * element(p->type);
        a.vec = a.channels / a.groups % 4 == 0;
        const void* tokens[] = {a.x, a.delta, a.z, a.dy, a.y, a.dx, a.ddelta, a.dz};
        for (const void* t : tokens) if (reinterpret_cast<uintptr_t>(t) % four) a.vec = 0;
        a.vec_states = a.state % 4 == 0 && reinterpret_cast<uintptr_t>(a.B) % four == 0 && reinterpret_cast<uintptr_t>(a.C) % four == 0;
        a.per_warp = a.run = (int)plan.items;
        a.free_blocks = plan.free_blocks;
        a.vec_params = a.state % 4 == 0 && aligned16(a.A) && aligned16(a.carries_in) && aligned16(a.initial) && aligned16(a.carries) && aligned16(a.final_state) &&
                       aligned16(a.ends);
        e = step ? table->scan_step(a, st) : grad ? table->scan_grad(a, st) : table->scan(a, st);
    }
    if (e != cudaSuccess) {
        fail(err, err_cap, "%s: launch failed: %s", plan.kernel_name, cudaGetErrorString(e));
        return PD_ERR_CUDA;
    }
    return PD_OK;
}
}  // namespace

int pd_scan_launch(int family, const void* params, int math_mode, const int64_t grid[3], const PdScanPlan& plan,
                   const void* const* in, void* const* out, void* scratch, cudaStream_t st, char* err, size_t err_cap) {
    return scan_launch(family, params, math_mode, grid, plan, in, out, scratch, st, nullptr, err, err_cap);
}

PdScanReport pd_scan_describe(int family, const void* params, int math_mode, const int64_t grid[3], const PdScanPlan& plan) {
    PdScanReport report;
    void* operands[16];       // as many as a call can have; aligned, never read
    for (void*& p : operands) p = reinterpret_cast<void*>((uintptr_t)256);
    char err[64];
    scan_launch(family, params, math_mode, grid, plan, operands, operands, operands[0], nullptr, &report, err, sizeof(err));
    return report;
}
