// pd_scan.h -- argument blocks, geometry and launcher tables of the state-space
// families (causal convolution and selective scan: prompts, gradients, single
// tokens), shared by the C-ABI side (pd_scan_api.cu) and the kernels
// (pd_scan.cu, compiled once per math mode like pd_kernels.cu).
#ifndef PD_SCAN_H_
#define PD_SCAN_H_

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <vector>

#include "../../include/palladium_cuda.h"

// A sequence's tokens are rows of `x`.  Dense calls: sequence s has rows [s * length, (s + 1) * length).
// Packed calls: rows [offsets[s], offsets[s + 1]), every value clamped to [0, rows], a decreasing pair an
// empty sequence; whatever the offsets hold, no kernel leaves its arrays.
struct PdTokens {
    const int32_t* offsets;   // null: dense
    int64_t rows;             // rows of the token arrays
    int64_t length;           // dense: tokens per sequence
    int64_t seqs;
};

// What a launcher says of its kernel instead of launching it.
struct PdScanReport {
    int registers = -1, static_smem = -1, blocks_per_sm = -1;
};

struct PdConvArgs {
    PdScanReport* report;     // non-null: describe, do not launch (no pointer is read)
    PdTokens tok;
    int type, width, silu;
    int64_t channels;
    const void *x, *dy, *initial, *dfinal;
    const float *weight, *bias;
    void *y, *final_state, *dx, *dinitial;
    float *dweight, *dbias;
    float* partial;           // gradient: (row_blocks, channels, width + 1) sums of dweight and dbias
    int64_t row_blocks;
    int vec;                  // channels per thread in one aligned access, or 1
    int run;                  // consecutive rows per thread
};

struct PdScanArgs {
    PdScanReport* report;     // as above
    PdTokens tok;
    int type, state, groups, softplus;
    int vec;                  // tokens can be read four channels at a time
    int vec_states;           // B and C four states at a time
    int vec_params;           // A and the states four at a time
    int run;                  // single tokens: sequences a block takes one after another
    int per_warp;             // gradient: channels a warp takes one after another; prompts: channels per lane
    int64_t channels;
    const void *x, *delta, *B, *C, *z, *dy;
    const float *A, *bias, *skip, *initial, *carries_in, *dfinal;
    void *y, *dx, *ddelta, *dB, *dC, *dz;
    float *final_state, *carries, *dA, *dbias, *dskip, *dinitial;
    // gradient: sums over the channels of one tile, (tiles, rows, 2, states rounded up), and over the tokens of
    // one sequence, (seqs, channels, state + 2)
    float *partial_bc, *partial_params;
    // prompts cut into segments of `segment` tokens (`segments` of them in all): their end states from zero,
    // (segments, channels, state), and total steps, (segments, channels); null where no sequence is cut
    int64_t segment, segments;
    float *ends, *totals;
    int64_t free_blocks;      // packed: blocks that clear the rows of no sequence; prompts: for each tile of channels
};

// Lanes that share one channel: each holds four states.
inline int pd_scan_lanes(int state) { return state <= 4 ? 1 : state <= 8 ? 2 : state <= 16 ? 4 : state <= 32 ? 8 : 16; }
// The same for the prompt and gradient kernels, which take more than sixteen states in slices.
inline int pd_scan_slice_lanes(int state) { return state <= 4 ? 1 : state <= 8 ? 2 : 4; }
inline int pd_scan_pad(int state) { const int w = 4 * pd_scan_slice_lanes(state); return (state + w - 1) / w * w; }

// The step kernel's geometry: warps of 32 / lanes channels, up to eight to a block; a small call takes one to a
// block, so that its warps spread over the SMs.
inline int64_t pd_step_tiles(int64_t channels, int groups, int state) {
    const int64_t per = channels / groups, ch = 32 / pd_scan_lanes(state);
    return (per + ch - 1) / ch * groups;
}
inline int pd_step_warps(int64_t channels, int groups, int state, int64_t seqs) {
    const int64_t tiles = pd_step_tiles(channels, groups, state);
    return tiles * seqs < 1024 ? 1 : tiles < 8 ? (int)tiles : 8;
}
inline int64_t pd_step_blocks(int64_t channels, int groups, int state, int64_t seqs) {
    const int warps = pd_step_warps(channels, groups, state, seqs);
    return (pd_step_tiles(channels, groups, state) + warps - 1) / warps;
}

// Sequences per block: a few where that leaves a full GPU of blocks, and what the second launch dimension asks for.
inline int pd_step_run(int64_t channels, int groups, int state, int64_t seqs, int sms) {
    const int64_t warps = pd_step_tiles(channels, groups, state) * seqs, full = (int64_t)sms * 64;
    int64_t run = warps / full;
    run = run < 1 ? 1 : run > 8 ? 8 : run;
    const int64_t least = (seqs + 65534) / 65535;
    return (int)(run < least ? least : run);
}

// Blocks of that much shared memory on an SM: it has 228 KB, of which each block takes 1 KB more than it asks for.
__host__ __device__ constexpr int pd_scan_resident(int bytes) { return 228 * 1024 / (bytes + 1024); }

// The prompt kernel's block and its shared memory: `ln` lanes a channel, `nch` channels a lane, `element` bytes a value.
constexpr int PD_SCAN_WALKING_WARPS = 2;
struct PdScanShape {
    int lane_channels, warp_channels, channels, pad;    // channels of a lane, of a walking warp, of the block; states rounded up
    int du, B, C, y, raw, bytes;      // offsets in floats, from `raw` on in bytes
    static constexpr int kRow = PD_SCAN_CHUNK;
    __host__ __device__ constexpr PdScanShape(int ln, int nch, int element)
        : lane_channels(nch), warp_channels(32 / ln * nch), channels(PD_SCAN_WALKING_WARPS * warp_channels), pad(4 * ln), du(0),
          // two buffers of each: (tokens, channels) steps and inputs, (tokens, pad) B and C, (tokens, channels) sums
          B(4 * kRow * channels), C(B + 2 * kRow * pad), y(C + 2 * kRow * pad), raw((y + 2 * kRow * channels) * 4),
          // as stored: four buffers of x, delta, z, (3, tokens, channels), and two of B and C, (2, tokens, pad)
          bytes(raw + 12 * kRow * channels * element + 4 * kRow * pad * element) {}
    // the blocks an SM is to hold: what shared memory has room for, five at most (96 registers a thread), four where a
    // lane has two channels (128)
    __host__ __device__ constexpr int resident() const {
        const int most = lane_channels > 1 ? 4 : 5, fit = pd_scan_resident(bytes);
        return fit < most ? fit : most;
    }
};

// The gradient kernel's block: four warps' channels, `per_warp` of them one after another in each, and its shared
// memory.  (ONE: all states in one slice, and with it all but the channels known when compiling)
constexpr int PD_SCAN_GRAD_WARPS = 4;
template <int LN, bool ONE>
struct PdGradShape {
    int channels, slices, pad;    // channels per block, slices of 4 LN states, states rounded up
    // offsets in shared memory: float32 arrays in floats, the chunks as stored behind them in bytes
    int d, u, g, x, s, z, y, du, dd, carry, rate, entry, dA, red, skip, raw, couplings, bytes;
    int pitch;                    // elements between two tokens' couplings
    static constexpr int kRow = PD_SCAN_CHUNK, kWide = 4 * LN;
    __host__ __device__ PdGradShape(int state, int per_warp, int element) {
        channels = PD_SCAN_GRAD_WARPS * per_warp;
        slices = ONE ? 1 : (state + kWide - 1) / kWide;
        pad = slices * kWide;
        pitch = pad + 4;          // (the token groups' rows then lie in different banks)
        const int cells = channels * kRow, more = slices > 1 ? cells : 0;
        d = 0; u = d + 2 * cells; g = u + 2 * cells;     // as pairs of equal halves, which packed operations take
        x = g + 2 * cells; s = x + cells; z = s + cells;
        y = z + cells; du = y + more; dd = du + more;
        carry = dd + more;
        rate = carry + channels * pad;
        entry = rate + channels * pad;           // two buffers
        dA = entry + 2 * channels * pad;
        red = dA + channels * slices * 128;
        // at different times: the warps' sums of dB and dC, the staging threads' of dbias and dskip
        const int warps = PD_SCAN_GRAD_WARPS * kRow * (2 * kWide + 4), staged = 32 * PD_SCAN_GRAD_WARPS * 8;
        skip = red + (warps > staged ? warps : staged);
        raw = (skip + channels) * 4;             // x, delta, dy, z: (4, tokens, channels)
        couplings = raw + 4 * cells * element;   // two buffers of B and C: (2, 2, tokens, pitch)
        bytes = couplings + 4 * kRow * pitch * element;
    }
};
inline int pd_scan_grad_bytes(int state, int per_warp, int element) {
    const int lanes = pd_scan_slice_lanes(state);
    if (lanes == 1) return PdGradShape<1, false>(state, per_warp, element).bytes;
    if (lanes == 2) return PdGradShape<2, false>(state, per_warp, element).bytes;
    return PdGradShape<4, false>(state, per_warp, element).bytes;
}

struct PdScanTable {
    cudaError_t (*conv)(const PdConvArgs&, cudaStream_t);
    cudaError_t (*conv_step)(const PdConvArgs&, cudaStream_t);
    cudaError_t (*conv_grad)(const PdConvArgs&, cudaStream_t);
    cudaError_t (*scan)(const PdScanArgs&, cudaStream_t);
    cudaError_t (*scan_step)(const PdScanArgs&, cudaStream_t);
    cudaError_t (*scan_grad)(const PdScanArgs&, cudaStream_t);
};
const PdScanTable* pd_scan_table_safe();
const PdScanTable* pd_scan_table_relaxed();
const PdScanTable* pd_scan_table_fast();

// What the C ABI needs of a call: its buffers' sizes, its launches and its scratch.
struct PdScanPlan {
    const char* kernel_name = "";
    int64_t grid = 1, grid_y = 1, block = 1, items = 1, launches = 1, scratch_bytes = 0, dynamic_smem = 0;
    int64_t segment = 1, segments = 0, totals_offset = 0;    // prompts: see PdScanArgs
    int64_t free_blocks = 0;      // see PdScanArgs
    int64_t row_blocks = 0;       // gradient of the convolution: blocks along the rows
    int64_t params_offset = 0;    // gradient of the scan: where in the scratch the parameters' sums begin
    std::vector<size_t> in_bytes, out_bytes;
};
bool pd_is_scan_family(int family);
int pd_scan_plan(int family, const void* params, size_t params_bytes, const int64_t grid[3], const int64_t block[3],
                 int sms, PdScanPlan* plan, char* err, size_t err_cap);
// Refuses results that share memory with an operand or with one another; a step's new state may be its old one.
int pd_scan_overlap(int family, int n_in, const void* const* in, const size_t* in_bytes, int n_out, void* const* out,
                    const size_t* out_bytes, char* err, size_t err_cap);
int pd_scan_launch(int family, const void* params, int math_mode, const int64_t grid[3], const PdScanPlan& plan,
                   const void* const* in, void* const* out, void* scratch, cudaStream_t st, char* err, size_t err_cap);
// The kernel that a call on aligned operands gets, on the current device; what cannot be had stays -1.
PdScanReport pd_scan_describe(int family, const void* params, int math_mode, const int64_t grid[3], const PdScanPlan& plan);

#endif  // PD_SCAN_H_
