// C ABI of libstattn.so: drafted sampling -- gen_sample(stochastic=True) (model_attention.py:863-918) with words drafted by a 4-bit copy of
// the vocabulary projection (ff_logit, :703-705) and checked against the full-precision one, several at a time.
//
// The recurrent part of the decoder needs the words one after the other and is the same for draft and target: behind the same words both
// see the same state, so the states of the drafted positions are kept and nothing of it runs twice.  What a round saves is the
// projection: dim_word x n_words in fp32, read once for draft + 1 positions instead of once a word; the draft reads 17/32 byte an
// element.  (20 000 words: 41 MB against 5.4.)
#include "steps.h"
#include "ops/ops.h"

#include <new>

static int sample_drafted(stattn_handle* h, int nvid, const float* ctxg, const float* ctxg_mask, const float* ctxl, const float* ctxm, int T, int K,
                          int draft, int maxlen, const float* uniforms, int64_t* out_tokens, float* out_scores, int32_t* out_lens,
                          int32_t* out_drafted, int32_t* out_kept) {
    const bool resident = !ctxg && !ctxg_mask && !ctxl && !ctxm;
    if (!h || nvid < 1 || nvid > 16 || (!resident && (!ctxg || !ctxg_mask || !ctxl || !ctxm)) || T <= 0 || K <= 0 || draft < 1 || draft > 8 ||
        maxlen < 1 || maxlen > 65536 || !out_tokens || !out_scores || !out_lens)
        return fail(h, STATTN_EINVAL, "sample_drafted: bad argument (1 <= nvid <= 16, 1 <= draft <= 8, 1 <= maxlen <= 65536)");
    HIPCHK(h, hipSetDevice(h->device));
    if (!resident) CHK(stattn_beam_stage(h, nvid, ctxg, ctxg_mask, ctxl, ctxm, T, K));
    else if (!h->bk_valid || h->bk_n != nvid || h->bk_T != T || h->bk_K != K)
        return fail(h, STATTN_ESTATE, "sample_drafted: no staged videos of this shape (call stattn_beam_stage)");
    const int D = h->D, E = h->E, V = h->V, Vp = h->Vp, M = nvid, P = draft + 1;      // P positions a round
    const Weights& w = h->w;
    hipStream_t s = h->stream;
    HIPCHK(h, hipStreamSynchronize(s));      // (buffers may be reallocated below)

    // --- the videos: projected once (f_init and the context projections)
    CtxPtrs c{};
    float *rawl, *rawm, *mG, *mean, *h0, *c0;
    const size_t nG = (size_t)nvid * T * D, nLd = (size_t)nvid * T * K * D;
    CHK(getbuf_t(h, "bs_G", nG, &c.G)); CHK(getbuf_t(h, "bs_rawl", (size_t)nvid * T * K * h->Fl, &rawl));
    CHK(getbuf_t(h, "bs_rawm", (size_t)nvid * T * h->Fm, &rawm)); CHK(getbuf_t(h, "bs_mG", (size_t)nvid * T, &mG));
    CHK(getbuf_t(h, "bs_L", nLd, &c.L)); CHK(getbuf_t(h, "bs_Mo", nG, &c.Mo)); CHK(getbuf_t(h, "bs_PG", nG, &c.PG));
    CHK(getbuf_t(h, "bs_PL", nLd, &c.PL)); CHK(getbuf_t(h, "bs_PM", nG, &c.PM));
    CHK(getbuf_t(h, "bs_LW", h->opt.lt_mode == 1 ? nLd : 1, &c.LW));
    CHK(getbuf_t(h, "bs_mean", (size_t)nvid * D, &mean)); CHK(getbuf_t(h, "bs_h0", (size_t)nvid * D, &h0));
    CHK(getbuf_t(h, "bs_c0", (size_t)nvid * D, &c0));
    CHK(project_context(h, nvid, T, K, c.G, rawl, rawm, c));
    CHK(init_state(h, nvid, T, c.G, mG, mean, h0, c0));

    // --- buffers of a round
    int* vid; int64_t *xs, *words; int32_t* acc;
    float *hs, *cs, *hd, *emb, *sproj, *preh, *dp, *al, *CL, *eg, *em, *elt, *plt, *ag, *am, *alt, *ctx, *a1, *lq, *q, *lg, *p, *ub;
    uint8_t *hc, *hsc;
    CHK(getbuf_t(h, "dr_vid", (size_t)M, &vid)); CHK(getbuf_t(h, "dr_xs", (size_t)P * M, &xs)); CHK(getbuf_t(h, "dr_words", (size_t)M * P, &words));
    CHK(getbuf_t(h, "dr_acc", (size_t)M, &acc));
    CHK(getbuf_t(h, "dr_hs", (size_t)P * M * D, &hs)); CHK(getbuf_t(h, "dr_cs", (size_t)P * M * D, &cs));
    CHK(getbuf_t(h, "dr_hd", (size_t)M * D, &hd)); CHK(getbuf_t(h, "dr_emb", (size_t)M * E, &emb));
    CHK(getbuf_t(h, "dr_sproj", (size_t)M * 4 * D, &sproj)); CHK(getbuf_t(h, "dr_preh", (size_t)M * 4 * D, &preh));
    CHK(getbuf_t(h, "dr_dp", (size_t)M * 3 * D, &dp));
    CHK(getbuf_t(h, "dr_al", (size_t)M * T * K, &al)); CHK(getbuf_t(h, "dr_CL", (size_t)M * T * D, &CL));
    CHK(getbuf_t(h, "dr_eg", (size_t)M * T, &eg)); CHK(getbuf_t(h, "dr_em", (size_t)M * T, &em)); CHK(getbuf_t(h, "dr_elt", (size_t)M * T, &elt));
    CHK(getbuf_t(h, "dr_plt", h->opt.lt_mode == 0 ? (size_t)M * T * D : 1, &plt));
    CHK(getbuf_t(h, "dr_ag", (size_t)M * T, &ag)); CHK(getbuf_t(h, "dr_am", (size_t)M * T, &am)); CHK(getbuf_t(h, "dr_alt", (size_t)M * T, &alt));
    CHK(getbuf_t(h, "dr_ctx", (size_t)M * D, &ctx)); CHK(getbuf_t(h, "dr_a1", (size_t)P * M * E, &a1));
    CHK(getbuf_t(h, "dr_lq", (size_t)M * Vp, &lq)); CHK(getbuf_t(h, "dr_q", (size_t)draft * M * Vp, &q));
    CHK(getbuf_t(h, "dr_lg", (size_t)P * M * Vp, &lg)); CHK(getbuf_t(h, "dr_p", (size_t)P * M * Vp, &p));
    CHK(getbuf_t(h, "dr_head", (size_t)V * (mx4_kp(E) / 2), &hc)); CHK(getbuf_t(h, "dr_head_scales", (size_t)V * (mx4_kp(E) / 32), &hsc));
    double* vsums;
    CHK(getbuf_t(h, "dr_sums", (size_t)M * 256, &vsums));
    DraftState d{};
    d.M = M; d.D = D; d.k = draft; d.maxlen = maxlen; d.x = xs;
    CHK(getbuf_t(h, "dr_h", (size_t)M * D, &d.h)); CHK(getbuf_t(h, "dr_c", (size_t)M * D, &d.c)); CHK(getbuf_t(h, "dr_info", (size_t)M, &d.info));
    CHK(getbuf_t(h, "dr_tokens", (size_t)M * maxlen, &d.tokens)); CHK(getbuf_t(h, "dr_u", (size_t)(2 * draft + 1) * M, &d.u));
    const size_t nu = (size_t)maxlen * (2 * draft + 1) * M;
    CHK(getbuf_t(h, "dr_uniforms", nu, &ub));
    d.uniforms = ub;

    // On the row-panel kernels the readout launch of a word also leaves the state projections of its h, so the next word starts with its
    // attention; the positions' projections are kept with their states.
    FwdPanels pn{};
    const bool panels = use_panels(h, M, 1) && Vp % 16 == 0;
    float* projs = nullptr;
    if (panels) {
        CHK(pack_fwd_panels(h, &pn, true));
        CHK(getbuf_t(h, "dr_projs", (size_t)P * M * 8 * D, &projs)); CHK(getbuf_t(h, "dr_proj", (size_t)M * 8 * D, &d.proj));
    }

    // --- numbers of this call, the 4-bit head of the current parameters, the captions' beginnings
    std::vector<float> drawn;
    if (!uniforms) {
        auto mix = [](uint64_t z) { z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull; z = (z ^ (z >> 27)) * 0x94D049BB133111EBull; return z ^ (z >> 31); };
        const uint64_t seed = mix(h->seed * 0x9E3779B97F4A7C15ull + 0x632BE59BD9B4E019ull * (++h->draw));
        drawn.resize(nu);
        for (size_t i = 0; i < nu; ++i) drawn[i] = (float)(mix(seed + 0x9E3779B97F4A7C15ull * (i + 1)) >> 40) * (1.0f / 16777216.0f);
        uniforms = drawn.data();
    }
    HIPCHK(h, copy_now(s, ub, uniforms, nu * sizeof(float), hipMemcpyHostToDevice));
    HIPCHK(h, launch_mx4_quantize(s, Mx4QuantArgs{w.Wo, OP_F32, V, E, 1, Vp, hc, hsc}));      // ff_logit_W is (dim_word, n_words)
    HIPCHK(h, launch_iota(s, vid, M, 1));
    HIPCHK(h, launch_fill(s, dp, 0.5f, (size_t)M * 3 * D));                                  // use_noise = 0 (:469-472)
    HIPCHK(h, launch_draft_begin(s, d, h0, c0));

    // state projections of h (M rows) into two segments behind `n` others of a row-panel launch
    auto project = [&](PnArgs& a, int n, const float* hrows, float* to) {
        a.M = M; a.nseg = n + 2;
        for (int i = 0; i < 2; ++i) {
            PnSeg& sp = a.seg[n + i];
            pn_seg_defaults(sp);
            sp.npairs = 1; sp.p[0] = PnPair{hrows, D, i == 0 ? pn.Wd : pn.U, D, 0};
            sp.C = to + (size_t)i * 4 * D; sp.ldc = 8 * D; sp.N = 4 * D;
        }
    };
    if (panels) {
        PnArgs a{};
        project(a, 0, d.h, d.proj);
        HIPCHK(h, launch_panel(s, a));
    }
    auto round = [&]() -> int {
        for (int j = 0; j < P; ++j) {
            // the state behind word j of the round, and the readout's first layer (:817-836) in front of the next word
            if (j == 0) HIPCHK(h, launch_embed(s, xs, w.Wemb, emb, M, E, V, 0));      // (later ones: by the draw)
            StepIO io{};
            io.M = M; io.T = T; io.K = K; io.c = c; io.vid = vid;
            io.h_prev = j ? hs + (size_t)(j - 1) * M * D : d.h; io.c_prev = j ? cs + (size_t)(j - 1) * M * D : d.c;
            io.sproj = sproj; io.preh = preh; io.xproj = nullptr; io.emb = emb; io.dp = dp; io.mask = nullptr; io.d1 = nullptr;
            io.alphal = al; io.CL = CL; io.eg = eg; io.em = em; io.elt = elt; io.plt = plt;
            io.alphag = ag; io.alpham = am; io.alphalt = alt; io.csum = nullptr; io.sel = nullptr; io.ctx = ctx;
            io.h_out = hs + (size_t)j * M * D; io.c_out = cs + (size_t)j * M * D; io.gates = nullptr; io.hd = hd;
            if (panels) {
                io.pn = &pn; io.skip_hproj = true; io.ldproj = 8 * D;
                io.sproj = j ? projs + (size_t)(j - 1) * M * 8 * D : d.proj;
                io.preh = io.sproj + (size_t)4 * D;
            }
            CHK(run_step(h, io));
            float* aj = a1 + (size_t)j * M * E;
            auto readout = [&](auto& sg) {
                if (h->opt.ctx2out) { sg.npairs = 2; sg.bias2 = w.bl2; }
                sg.bias = w.bl1;
                if (h->opt.prev2out) { sg.add = emb; sg.ldadd = E; }
                sg.act = 1; sg.scale = 0.5f; sg.C = aj; sg.ldc = E; sg.N = E;
            };
            if (panels) {
                PnArgs a{};
                pn_seg_defaults(a.seg[0]);
                a.seg[0].npairs = 1; a.seg[0].p[0] = PnPair{hd, D, pn.Wl1, D, 0}; a.seg[0].p[1] = PnPair{ctx, D, pn.Wl2, D, 0};
                readout(a.seg[0]);
                project(a, 1, hs + (size_t)j * M * D, projs + (size_t)j * M * 8 * D);
                HIPCHK(h, launch_panel(s, a));
            } else {
                SkArgs a{};
                a.M = M; a.nseg = 1;
                skinny_seg_defaults(a.seg[0]);
                a.seg[0].npairs = 1; a.seg[0].p[0] = SkPair{hd, w.Wl1, D, E, D, 0}; a.seg[0].p[1] = SkPair{ctx, w.Wl2, D, E, D, 0};
                readout(a.seg[0]);
                HIPCHK(h, launch_skinny(s, a));
            }
            if (j == draft) break;
            // the draft's distribution (4-bit head), a word drawn from it, that word's embedding
            HIPCHK(h, launch_mx4_linear_few(s, Mx4LinearArgs{aj, OP_F32, M, E, Mx4View{hc, hsc, V, E}, w.bo, lq, Vp}));
            HIPCHK(h, launch_softmax_draw(s, DrawArgs{lq, q + (size_t)j * M * Vp, Vp, V, M, d.u + (size_t)j * M, xs + (size_t)(j + 1) * M, w.Wemb, emb, E}));
        }
        // the full-precision distributions of all positions at once (:703-709), the check, the captions
        if (P * M <= 64) {
            SkArgs b{};
            b.M = P * M; b.nseg = 1;
            SkSeg& so = b.seg[0];
            skinny_seg_defaults(so);
            so.npairs = 1; so.p[0] = SkPair{a1, w.Wo, E, Vp, E, 0};
            so.bias = w.bo; so.C = lg; so.ldc = Vp; so.N = Vp;
            HIPCHK(h, launch_skinny(s, b));
        } else {
            GemmArgs g;
            gemm_defaults(g); g.split = h->opt.precision != 0;
            g.A = a1; g.lda = E; g.B = w.Wo; g.ldb = Vp; g.C = lg; g.ldc = Vp; g.M = P * M; g.N = Vp; g.K = E; g.bias = w.bo;
            HIPCHK(h, launch_gemm(s, g, false, false));
        }
        HIPCHK(h, launch_softmax_draw(s, DrawArgs{lg, p, Vp, V, P * M, nullptr, nullptr, nullptr, nullptr, 0}));
        VerifyArgs v{};
        v.split = verify_split(M, V, OP_F32); v.sums = vsums;
        v.draft = xs + M; v.draft_b = 1; v.draft_j = M;
        v.target = p; v.target_b = Vp; v.target_j = (int64_t)M * Vp; v.proposal = q; v.proposal_b = Vp; v.proposal_j = (int64_t)M * Vp;
        v.type = OP_F32; v.accept_u = d.u + (size_t)draft * M; v.accept_b = 1; v.accept_j = M; v.draw_u = d.u + (size_t)2 * draft * M;
        v.b = M; v.j = draft; v.v = V; v.words = words; v.words_ld = P; v.accepted = acc;
        HIPCHK(h, launch_verify_draft(s, v));
        HIPCHK(h, launch_draft_commit(s, d, words, acc, hs, cs, panels ? projs : nullptr, p, Vp));
        return STATTN_OK;
    };

    // The rounds are launched plainly.  (Captured once a shape and replayed, 48 words took 3.8 ms instead of 4.0 with one caption, 5.8 instead of
    // 5.9 with sixteen.  But a copy through the legacy stream or a device synchronization by any thread of the process meanwhile fails, and
    // leaves the capturing stream unusable.)
    std::vector<DraftInfo> info(M);
    for (int r = 0; r < maxlen; ++r) {       // every round adds a word at least to each caption that is not finished
        CHK(round());
        HIPCHK(h, hipMemcpyAsync(info.data(), d.info, (size_t)M * sizeof(DraftInfo), hipMemcpyDeviceToHost, s));
        HIPCHK(h, hipStreamSynchronize(s));
        bool live = false;
        for (const DraftInfo& f : info) live = live || !f.done;
        if (!live) break;
    }
    HIPCHK(h, copy_now(s, out_tokens, d.tokens, (size_t)M * maxlen * sizeof(int64_t), hipMemcpyDeviceToHost));
    for (int m = 0; m < M; ++m) {
        out_scores[m] = info[m].score; out_lens[m] = info[m].len;
        if (out_drafted) out_drafted[m] = info[m].drafted;
        if (out_kept) out_kept[m] = info[m].kept;
    }
    return STATTN_OK;
}

extern "C" int stattn_sample_drafted(stattn_handle* h, int nvid, const float* ctxg, const float* ctxg_mask, const float* ctxl, const float* ctxm,
                                     int T, int K, int draft, int maxlen, const float* uniforms, int64_t* out_tokens, float* out_scores,
                                     int32_t* out_lens, int32_t* out_drafted, int32_t* out_kept) {
    try {
        return sample_drafted(h, nvid, ctxg, ctxg_mask, ctxl, ctxm, T, K, draft, maxlen, uniforms, out_tokens, out_scores, out_lens, out_drafted, out_kept);
    } catch (const std::bad_alloc&) {       // (the numbers of a call, 4 maxlen (2 draft + 1) nvid bytes, when the handle draws them)
        return fail(h, STATTN_EHIP, "sample_drafted: out of host memory");
    }
}
