// Host side of the slots' adapters: loading, binding, and their launches in a step (slot_adapters.cuh).  Included by engine.cu.

// the projection matrices a file may address, as check_loras() has them for files blended at load
static bool adapter_base(const std::string& base) {
    static const char* ok[] = {".att.receptance", ".att.key", ".att.value", ".att.gate", ".att.output", ".ffn.key", ".ffn.value", ".ffn.receptance"};
    if (base == "head") return true;
    for (const char* o : ok)
        if (ends_with(base, o)) return true;
    return false;
}

int b200rwkv_engine::adapter_site(const SegDesc& d) {
    if (world != 1 || d.slice >= 0 || d.n0 != 0 || d.k0 != 0 || !ends_with(d.t->name, ".weight")) return -1;
    const std::string base = d.t->name.substr(0, d.t->name.size() - 7);
    if (!adapter_base(base)) return -1;
    sites.push_back({base, (int)d.t->shape[1], (int)d.t->shape[0]});
    return (int)sites.size() - 1;
}

void b200rwkv_engine::adapter_setup() {
    if (d_entries) return;
    const size_t n = sites.size() * ADAPTER_POOL;
    // (allocations that fail leave nothing half made: the table comes last)
    if (!d_slot_adapter) {
        d_slot_adapter = (int*)dalloc((size_t)S * 4, false);
        CK(cudaMemset(d_slot_adapter, 0xFF, (size_t)S * 4));
    }
    if (!d_index_tok) d_index_tok = (int*)dalloc((size_t)(maxT + maxR) * 4);
    if (!adapter_ws) adapter_ws = (uint8_t*)dalloc(2 * adapter_ws_bytes(), false);
    if (!adapter_tmp) adapter_tmp = (float*)dalloc((size_t)maxT * (F + C) * 4, false);
    slot_adapter.assign(S, -1);
    pool.assign(ADAPTER_POOL, LoadedAdapter());
    d_entries = (AdapterEntry*)dalloc(n * sizeof(AdapterEntry));
    adapters_prepare(B200RWKV_TYPE_F16, B200RWKV_TYPE_F32);
    CK(cudaDeviceSynchronize());
}

size_t b200rwkv_engine::adapter_ws_bytes() const { return (adapters_workspace(std::max(maxT, ADP_INLINE + 1), ADAPTER_POOL, GEMM_MAX_SEG, ADP_MAX_RANK) + 255) & ~(size_t)255; }

uint64_t b200rwkv_engine::adapter_load(const StFile& st, float alpha) {
    REQUIRE(!kx && world == 1, B200RWKV_ERR_UNSUPPORTED, "adapters of slots: RWKV models on one GPU");
    REQUIRE(std::isfinite(alpha), B200RWKV_ERR_INVALID, "adapter: alpha must be a number");
    struct Pair { int site; const StTensor *a, *b; int r, rp; size_t at; };
    std::vector<Pair> pairs;
    size_t halves = 0;
    int most = 0;
    for (auto& kv : st.tensors) {
        const std::string& name = kv.first;
        if (ends_with(name, ".lora.1")) {
            REQUIRE(st.find(name.substr(0, name.size() - 1) + "0"), B200RWKV_ERR_INVALID, "adapter file: " + name + " has no .lora.0");
            continue;
        }
        REQUIRE(ends_with(name, ".lora.0"), B200RWKV_ERR_UNSUPPORTED, "adapter file carries " + name + ": only low-rank pairs on projection matrices are served");
        const std::string base = name.substr(0, name.size() - 7);
        int site = -1;
        for (size_t i = 0; i < sites.size(); ++i)
            if (sites[i].base == base) site = (int)i;
        REQUIRE(site >= 0, B200RWKV_ERR_UNSUPPORTED, "adapter on " + base + ": the model has no such projection matrix");
        const StTensor *a = st.find(name), *b = st.find(base + ".lora.1");
        REQUIRE(b, B200RWKV_ERR_INVALID, "adapter file: " + base + ".lora.1 is missing");
        REQUIRE(a->dtype == "F16" && b->dtype == "F16", B200RWKV_ERR_UNSUPPORTED, "adapter tensors must be F16: " + base);
        REQUIRE(a->shape.size() == 2 && b->shape.size() == 2 && a->shape[0] == sites[site].K && b->shape[0] == sites[site].N && a->shape[1] == b->shape[1] && a->shape[1] >= 1,
                B200RWKV_ERR_INVALID, "adapter shapes do not match " + base + " (expected lora.0 [in, r], lora.1 [out, r])");
        REQUIRE(a->shape[1] <= ADP_MAX_RANK, B200RWKV_ERR_UNSUPPORTED, "adapter on " + base + ": ranks above 256 are not served");
        const int r = (int)a->shape[1], rp = rup(r, 8);
        pairs.push_back({site, a, b, r, rp, halves});
        halves += (size_t)rp * (sites[site].K + sites[site].N);
        halves = (halves + 127) & ~(size_t)127;
        most = std::max(most, rp);
    }
    REQUIRE(!pairs.empty(), B200RWKV_ERR_INVALID, "adapter file holds no <name>.lora.0 / <name>.lora.1 pairs");
    adapter_setup();
    int place = -1;
    for (int i = ADAPTER_POOL - 1; i >= 0; --i)
        if (pool[i].id == 0) place = i;
    REQUIRE(place >= 0, B200RWKV_ERR_STATE, "adapters: the model holds " + std::to_string(ADAPTER_POOL) + " already");
    DevTmp buf(halves * 2);
    std::vector<AdapterEntry> col(sites.size(), AdapterEntry{nullptr, nullptr, 0, 0.f});
    for (const Pair& q : pairs) {
        const AdapterSite& s = sites[q.site];
        __half* const a = (__half*)buf.p + q.at;
        __half* const b = a + (size_t)q.rp * s.K;
        DevTmp up(std::max(q.a->nbytes, q.b->nbytes));
        CK(cudaMemcpyAsync(up.p, q.a->data, q.a->nbytes, cudaMemcpyHostToDevice, stream));
        adapter_pack_a_kernel<<<num_sms * 4, 256, 0, stream>>>((const __half*)up.p, a, s.K, q.r, q.rp);
        CK(cudaMemcpyAsync(up.p, q.b->data, q.b->nbytes, cudaMemcpyHostToDevice, stream));
        adapter_pack_b_kernel<<<num_sms * 4, 256, 0, stream>>>((const __half*)up.p, b, s.N, q.r, q.rp);
        CK(cudaGetLastError());
        CK(cudaStreamSynchronize(stream));
        col[q.site] = AdapterEntry{a, b, q.rp, alpha};
    }
    // this adapter's column of the table [site][pool]
    CK(cudaMemcpy2DAsync(d_entries + place, ADAPTER_POOL * sizeof(AdapterEntry), col.data(), sizeof(AdapterEntry), sizeof(AdapterEntry), sites.size(), cudaMemcpyHostToDevice, stream));
    CK(cudaStreamSynchronize(stream));
    pool[place].buf = buf.p;
    buf.p = nullptr;
    adapter_rank = std::max(adapter_rank, most);
    return pool[place].id = next_adapter++;
}

int b200rwkv_engine::adapter_place(uint64_t id) const {
    for (size_t i = 0; id != 0 && i < pool.size(); ++i)
        if (pool[i].id == id) return (int)i;
    return -1;
}

void b200rwkv_engine::adapter_free(uint64_t id) {
    const int place = adapter_place(id);
    REQUIRE(place >= 0, B200RWKV_ERR_STATE, "unknown adapter id");
    for (int s = 0; s < S; ++s)
        REQUIRE(slot_adapter[s] != place, B200RWKV_ERR_STATE, "adapter is in use by slot " + std::to_string(s));
    CK(cudaStreamSynchronize(stream));          // no step that may read it is in flight
    CK(cudaFree(pool[place].buf));
    pool[place] = LoadedAdapter();
}

void b200rwkv_engine::adapter_bind(int slot, uint64_t id) {
    REQUIRE(slot >= 0 && slot < S, B200RWKV_ERR_STATE, "slot out of range");
    const int place = id == 0 ? -1 : adapter_place(id);
    REQUIRE(id == 0 || place >= 0, B200RWKV_ERR_STATE, "unknown adapter id");
    if (slot_adapter.empty() || slot_adapter[slot] == place) return;      // (nothing was ever loaded: the slot has none)
    adapter_slot_kernel<<<1, 1, 0, stream>>>(d_slot_adapter, slot, place);
    CK(cudaGetLastError());
    slot_adapter[slot] = place;
}

// params of this step's tokens (or logits rows); longer steps: with the plan of adapter_begin
AdapterParams b200rwkv_engine::adapter_params(int rows, bool out_rows) const {
    AdapterParams p;
    memset(&p, 0, sizeof(p));
    p.tokens = rows;
    p.adapters = ADAPTER_POOL;
    p.index = out_rows ? d_index_tok + maxT : d_index_tok;
    p.rank = adapter_rank;
    adapters_shape(p, adapter_ws + (out_rows ? adapter_ws_bytes() : 0), B200RWKV_TYPE_F16, B200RWKV_TYPE_F32);
    return p;
}

void b200rwkv_engine::adapter_begin(cudaStream_t s, const MetaView& mv, int rows, int out_rows, Profiler* prof) {
    AdapterIndexParams ip{mv, d_slot_adapter, d_index_tok, d_index_tok + maxT, rows, out_rows};
    launch_k(adapter_index_kernel, dim3(cdiv(std::max(rows, out_rows), 256)), dim3(256), 0, ip, KC_OTHER, s, prof);
    for (int i = 0; i < 2; ++i) {
        const int n = i ? out_rows : rows;
        if (n == 0) continue;
        const AdapterParams p = adapter_params(n, i == 1);
        if (!p.plan.base) continue;
        adapters_plan(s, p);
        ++launches_last_step;
    }
}

// in front of a projection launch: sums that an activation follows go to scratch rows
void b200rwkv_engine::adapter_redirect(const GemmLaunch& g, GemmParams& gp, int rows) {
    float* tmp = adapter_tmp;
    for (int i = 0; i < gp.nseg; ++i) {
        GemmSeg& sg = gp.seg[i];
        if (g.site[i] < 0 || (sg.out_mode == OUT_F32 && sg.act == ACT_NONE)) continue;
        sg.out = tmp;
        sg.out_mode = OUT_F32;
        sg.act = ACT_NONE;
        sg.ldo = sg.N;
        sg.grp = 0;
        tmp += (size_t)rows * sg.N;
    }
}

// behind it: the adapters on its outputs, then the activations.  `was`: the launch before adapter_redirect
void b200rwkv_engine::adapter_add(const GemmLaunch& g, const GemmParams& was, const GemmParams& gp, int rows, int th, bool tiles, bool split, cudaStream_t s,
                                   Profiler* prof) {
    AdapterParams p = adapter_params(rows, &g == &head);
    int n = 0;
    for (int i = 0; i < gp.nseg; ++i) {
        if (g.site[i] < 0) continue;
        const GemmSeg& sg = gp.seg[i];
        const AdapterSite& site = sites[g.site[i]];
        AdapterPart& d = p.part[n++];
        d.x = sg.A;
        d.x_a16 = 1;
        d.x_th = tiles ? th | sg.a_tile << 16 : th;
        d.x_lo = split ? 16 : 0;
        d.table = d_entries + (size_t)g.site[i] * ADAPTER_POOL;
        d.base = d.out = sg.out;
        d.base_stride = d.out_stride = sg.ldo;
        d.K = site.K; d.N = site.N; d.R = adapter_rank;
        d.vec = sg.ldo % 4 == 0 && (uintptr_t)sg.out % 16 == 0;
        const GemmSeg& to = was.seg[i];
        if (p.plan.base || sg.out == to.out) continue;
        const bool a16 = to.out_mode == OUT_A16;
        REQUIRE(to.act == ACT_SIGMOID || to.act == ACT_SILU || to.act == ACT_RELU2, B200RWKV_ERR_INVALID, "internal: activation behind an adapter");
        p.copy = p.finish = 1;
        d.out = to.out;
        d.act = to.act;
        d.fin = a16 ? (split ? ADP_A16_SPLIT : ADP_A16) : ADP_F32;
        if (a16) d.out_th = to.ldo;
        else {
            d.out_stride = to.ldo;
            d.vec = d.vec && to.ldo % 4 == 0 && (uintptr_t)to.out % 16 == 0;
        }
    }
    if (n == 0) return;
    p.nparts = n;
    launches_last_step += adapters_apply(s, p, B200RWKV_TYPE_F16, B200RWKV_TYPE_F32);
    for (int i = 0; i < gp.nseg && !p.finish; ++i) {
        const GemmSeg &sg = gp.seg[i], &to = was.seg[i];
        if (g.site[i] < 0 || sg.out == to.out) continue;
        AdapterFinishParams q{(const float*)sg.out, gp.nrows, to.out, to.N, to.act, to.out_mode == OUT_A16, split, to.ldo};
        launch_k(adapter_finish_kernel, dim3(std::min(4 * num_sms, cdiv(rows * (to.N / 8), 256))), dim3(256), 0, q, KC_OTHER, s, prof);
    }
}

// what the callers of the listed slots' rows have to get right
void b200rwkv_engine::check_rows(const char* call, int nrows, const int* slots) {
    auto need = [&](bool fine, int code, const char* what) { REQUIRE(fine, code, std::string(call) + ": " + what); };
    need(rank == 0, B200RWKV_ERR_INVALID, "only rank 0 holds the gathered logits");
    need(d_keep, B200RWKV_ERR_UNSUPPORTED, "the model keeps no logits rows");
    need(V <= LOGITS_MAX_VOCAB, B200RWKV_ERR_UNSUPPORTED, "vocabularies above 524288 are not supported");
    need(nrows >= 0 && nrows <= 4096 && (nrows == 0 || slots), B200RWKV_ERR_INVALID, "bad argument");
    std::lock_guard<std::mutex> lk(keep_mu);
    for (int i = 0; i < nrows; ++i) {
        need(slots[i] >= 0 && slots[i] < S, B200RWKV_ERR_STATE, "slot out of range");
        REQUIRE(keep_valid[slots[i]], B200RWKV_ERR_STATE, std::string(call) + ": slot " + std::to_string(slots[i]) + " has produced no logits row yet");
    }
}

// copies the pieces, behind the step that wrote the rows; `room` more bytes stand behind them on both sides
void b200rwkv_engine::send_pieces(const RowPieces& x, size_t room) {
    if (x.total + room > tk_cap) {
        if (tk_dev) { CK(cudaFree(tk_dev)); tk_dev = nullptr; }
        if (tk_host) { CK(cudaFreeHost(tk_host)); tk_host = nullptr; }
        tk_cap = 0;
        const size_t want = std::max<size_t>((x.total + room) * 2, 1 << 20);
        CK(cudaMalloc(&tk_dev, want));
        CK(cudaMallocHost(&tk_host, want));
        tk_cap = want;
    }
    for (const auto& q : x.pieces) memcpy(tk_host + q.at, q.src, q.bytes);
    CK(cudaStreamWaitEvent(sm_stream, step_done, 0));
    CK(cudaMemcpyAsync(tk_dev, tk_host, x.total, cudaMemcpyHostToDevice, sm_stream));
}

// the rows' adjustments: checked, and put among the pieces; the call itself once these are on their way (pointers are places until then)
LogitsParams b200rwkv_engine::adjusted_rows(const char* call, int nrows, const b200rwkv_row_controls& q, RowPieces& x) {
    auto need = [&](bool fine, const char* what) { REQUIRE(fine, B200RWKV_ERR_INVALID, std::string(call) + ": " + what); };
    const int nh = q.history_offset ? q.history_offset[nrows] : 0, nb = q.bias_offset ? q.bias_offset[nrows] : 0;
    need(nh >= 0 && nb >= 0 && (nh == 0 || q.history) && (nb == 0 || (q.bias_token && q.bias_value)), "bad lists");
    for (int i = 0; i < nrows; ++i) {
        need(!q.history_offset || (q.history_offset[i] >= 0 && q.history_offset[i] <= q.history_offset[i + 1]), "history offsets must ascend");
        need(!q.bias_offset || (q.bias_offset[i] >= 0 && q.bias_offset[i] <= q.bias_offset[i + 1]), "bias offsets must ascend");
        if (!q.controls) continue;
        const float* c = q.controls + 5 * (size_t)i;
        need(c[0] > 0.f && std::isfinite(c[0]) && std::isfinite(c[1]) && std::isfinite(c[2]) && c[3] >= 0.f && c[3] <= 1.f && c[4] > 0.f && std::isfinite(c[4]) && std::isfinite(1.f / c[4]),
             "repetition and temperature must be positive, decay in [0, 1], presence and frequency numbers");
    }
    const size_t words = (size_t)(V + 31) / 32, row4 = (size_t)nrows * 4;
    LogitsParams p;
    memset(&p, 0, sizeof(p));
    p.in = d_keep; p.in_stride = V;
    p.out_stride = V;
    p.V = V; p.kind = q.kind;
    auto place = [&](auto& to, const void* src, size_t bytes) {           // (one more, so that none is null)
        if (src && bytes) to = (std::remove_reference_t<decltype(to)>)(uintptr_t)(x.add(src, bytes) + 1);
    };
    place(p.in_row, q.slots, row4);
    place(p.controls, q.controls, (size_t)nrows * 20);
    if (nh) {
        place(p.hist_off, q.history_offset, row4 + 4);
        place(p.hist, q.history, (size_t)nh * 4);
        place(p.hist_from, q.history_from, row4);
    }
    if (nb) {
        place(p.bias_off, q.bias_offset, row4 + 4);
        place(p.bias_tok, q.bias_token, (size_t)nb * 4);
        place(p.bias_val, q.bias_value, (size_t)nb * 4);
    }
    if (q.allow_bits) {
        place(p.allow, q.allow_bits, (size_t)nrows * words * 4);
        p.words = (int)words;
        p.allow_rows = nrows;
    }
    return p;
}

// into sr_out
void b200rwkv_engine::adjust_rows(LogitsParams p, int nrows) {
    if (nrows > sr_cap) {
        if (sr_out) { CK(cudaFree(sr_out)); sr_out = nullptr; }
        sr_cap = 0;
        CK(cudaMalloc(&sr_out, (size_t)nrows * V * 4));
        sr_cap = nrows;
    }
    p.out = sr_out;
    auto real = [&](auto& at) {
        if (at) at = (std::remove_reference_t<decltype(at)>)(tk_dev + (uintptr_t)at - 1);
    };
    real(p.in_row); real(p.controls); real(p.hist_off); real(p.hist); real(p.hist_from); real(p.bias_off); real(p.bias_tok); real(p.bias_val); real(p.allow);
    logits_rows(sm_stream, p, nrows, B200RWKV_TYPE_F32);
}

// rows that b200rwkv_sample_rows adjusts (logits.cuh), on the sampling stream: see sample_topk
void b200rwkv_engine::sample_rows(int nrows, const b200rwkv_row_controls& q, float* out) {
    check_rows("sample_rows", nrows, q.slots);
    REQUIRE(nrows == 0 || out, B200RWKV_ERR_INVALID, "sample_rows: bad argument");
    REQUIRE(q.kind >= B200RWKV_LOGITS && q.kind <= B200RWKV_LOG_PROBS, B200RWKV_ERR_INVALID, "sample_rows: kind must be logits, probabilities or log-probabilities");
    if (nrows == 0) return;
    RowPieces x;
    const LogitsParams p = adjusted_rows("sample_rows", nrows, q, x);
    send_pieces(x, 0);
    adjust_rows(p, nrows);
    CK(cudaMemcpyAsync(out, sr_out, (size_t)nrows * V * 4, cudaMemcpyDeviceToHost, sm_stream));
    CK(cudaStreamSynchronize(sm_stream));
}

// a token for each of these rows (sample_tokens.cuh): from the kept rows themselves where nothing is to be adjusted
void b200rwkv_engine::sample_tokens(int nrows, const b200rwkv_row_controls& q, const b200rwkv_draw& d, int* tokens, float* probs) {
    check_rows("sample_tokens", nrows, q.slots);
    REQUIRE(nrows == 0 || (d.uniform && tokens), B200RWKV_ERR_INVALID, "sample_tokens: null uniform or tokens_out");
    if (nrows == 0) return;
    for (int i = 0; i < nrows; ++i) {
        REQUIRE(d.uniform[i] >= 0.f && d.uniform[i] < 1.f, B200RWKV_ERR_INVALID, "sample_tokens: uniform must be in [0, 1)");
        REQUIRE(!d.temperature || (d.temperature[i] >= 0.f && std::isfinite(d.temperature[i])), B200RWKV_ERR_INVALID, "sample_tokens: temperature must not be negative");
        REQUIRE((!d.top_p || !std::isnan(d.top_p[i])) && (!d.min_p || !std::isnan(d.min_p[i])), B200RWKV_ERR_INVALID, "sample_tokens: top_p and min_p must be numbers");
    }
    RowPieces x;
    LogitsParams p = adjusted_rows("sample_tokens", nrows, q, x);
    p.kind = LOGITS_ROWS;
    const size_t row4 = (size_t)nrows * 4;
    const size_t o_u = x.add(d.uniform, row4), o_t = x.add(d.temperature, row4), o_k = x.add(d.top_k, row4), o_p = x.add(d.top_p, row4), o_m = x.add(d.min_p, row4);
    send_pieces(x, 2 * row4);
    const bool as_they_are = !p.controls && !p.hist_off && !p.bias_off && !p.allow;
    if (!as_they_are) adjust_rows(p, nrows);
    DrawParams w;
    memset(&w, 0, sizeof(w));
    w.in = as_they_are ? d_keep : sr_out;
    w.in_stride = V;
    if (as_they_are) w.in_row = (const int*)(tk_dev + (uintptr_t)p.in_row - 1);
    w.uniform = (const float*)(tk_dev + o_u);
    if (d.temperature) w.temperature = (const float*)(tk_dev + o_t);
    if (d.top_k) w.top_k = (const int*)(tk_dev + o_k);
    if (d.top_p) w.top_p = (const float*)(tk_dev + o_p);
    if (d.min_p) w.min_p = (const float*)(tk_dev + o_m);
    w.tokens = (int*)(tk_dev + x.total);
    w.probs = (float*)(tk_dev + x.total + row4);
    w.V = V;
    w.type = B200RWKV_TYPE_F32;
    draw_rows(sm_stream, w, nrows);
    CK(cudaMemcpyAsync(tk_host + x.total, tk_dev + x.total, 2 * row4, cudaMemcpyDeviceToHost, sm_stream));
    CK(cudaStreamSynchronize(sm_stream));
    memcpy(tokens, tk_host + x.total, row4);
    if (probs) memcpy(probs, tk_host + x.total + row4, row4);
}
