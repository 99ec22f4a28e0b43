// fake_device.cu -- what the stand-in for the CUDA runtime (fake_device.cpp) needs to know of the library: an
// attention call's arguments, a coded prefix's handle, the older kernels' launches, and the helpers of host.cuh
// that api.cu defines.
#include "../compressed-kv-attention_b200/csrc/attention.cuh"
#include "../compressed-kv-attention_b200/csrc/codec.cuh"
#include "../compressed-kv-attention_b200/csrc/host.cuh"
#include "../compressed-kv-attention_b200/csrc/prefix.cuh"
#include "fake_device.h"

namespace {
thread_local std::string last_error;
}

namespace kvx {
int fail(int code, const std::string &msg) {
    last_error = msg;
    return code;
}
void clear_error() { last_error.clear(); }
int check_device() { return KVX_OK; }
int sm_count() { return 148; }
const char *detail_message(int, int) { return "device error"; }
int read_status(int *s, bool) { return s[0]; }
}  // namespace kvx

extern "C" {

void fake_paged(const void *args, Launch *l) {
    const kvx::PagedArgs &p = *static_cast<const kvx::PagedArgs *>(args);
    l->counter = *p.next_run;
    l->prefix_tiles = p.prefix_tiles, l->n_split = p.n_split, l->split_tiles = p.split_tiles, l->row_groups = p.row_groups;
    l->stream_ctas = p.stream_ctas, l->stream_runs = p.stream_runs, l->shared_runs = p.shared_runs;
    l->rows = p.batch * p.group;
    if (l->kind == STREAM && p.shared_runs) *p.next_run += p.stream_runs;
    if (l->kind == COMBINE && p.shared_runs) *p.next_run = 0;
}

const char *fake_last_error() { return last_error.c_str(); }
void fake_set_error(const char *s) { last_error = s; }

// The decode attention kernel and the encoder's first one (their arguments are not looked at).
int fake_decode_attention(int dim, int bf16, int compact) {
    return kvx::launch_attention(dim, bf16 != 0, compact != 0, kvx::AttnArgs{}, 1, nullptr);
}
int fake_encode(int dim) { return kvx::launch_encode_analyze(nullptr, 1, 100, dim, 128, 0x14, nullptr, nullptr, nullptr); }

// A coded prefix of so many tokens a head on the current device (nothing reads its table here).
kvx_prefix fake_prefix(int heads, int dim, int seq) {
    auto *p = new kvx_prefix_s();
    p->n_kv_heads = heads, p->dim = dim, p->seq = seq;
    cudaGetDevice(&p->device);
    p->dev.tiles = p->dev.head_tiles = (seq + kvx::kPrefixTile - 1) / kvx::kPrefixTile;
    return p;
}
void fake_prefix_free(kvx_prefix p) { delete p; }

}  // extern "C"
