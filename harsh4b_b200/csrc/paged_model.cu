// One step of the model over a paged cache: a ragged batch in which every
// sequence brings any number of new tokens (a prompt's chunk, one decoded
// token, none). The rows of all sequences go through the batched operations
// of the prefill (prefill.cu) -- RMSNorm + quantisation, the tensor-core int4
// GEMMs, SwiGLU in the quantisation of its rows -- with the append and the
// attention of paged.cu in between; the LM head runs on each sequence's last
// new row. q, k, v and the attended rows are 16-bit here: they are the paged
// operators' tensors, and halve what they move. The attended rows' int8 codes
// (a step is max / 127) mostly do not see the difference, so the logits are those
// of the fp16-cache paths within what the flips of a few codes make of it (2 % of
// a row's norm in the tests, 5 % at most), not their bits. Where those bits matter
// the sessions of one contiguous cache have attention="exact".
//
// With `parents` the new rows are the nodes of drafted trees: they are appended
// and attended as such, and the LM head runs on every row.

namespace h4b {

// 16-bit rows -> fp32, eight values a thread.
template <typename T>
__global__ void __launch_bounds__(256) widen_kernel(const uint4* in, float4* out, long long n) {
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
        const uint4 w = in[i];
        const float2 a = Pair<T>::unpack(w.x), b = Pair<T>::unpack(w.y), c = Pair<T>::unpack(w.z), d = Pair<T>::unpack(w.w);
        out[2 * i] = make_float4(a.x, a.y, b.x, b.y);
        out[2 * i + 1] = make_float4(c.x, c.y, d.x, d.y);
    }
}

// last[b] = x row of sequence b's last new token; zeros where it has none.
__global__ void __launch_bounds__(256) last_rows_kernel(const float* x, const int32_t* q_offsets, int tokens, int H,
                                                        float* last) {
    const int b = blockIdx.x, row = q_offsets[b + 1] - 1;
    const bool any = row >= q_offsets[b] && row >= 0 && row < tokens;
    for (int i = threadIdx.x; i < H; i += 256)
        last[static_cast<long long>(b) * H + i] = any ? x[static_cast<long long>(row) * H + i] : 0.f;
}

int validate_paged_step(const h4b_model* m, const h4b_paged_step* s) {
    if (!m || !s || s->kv.tokens < 1 || s->kv.sequences < 1) return H4B_EINVAL;
    if (m->layers < 1 || m->kv_heads < 1 || m->heads < 1 || m->heads % m->kv_heads) return H4B_EINVAL;
    if (s->kv.kv_heads != m->kv_heads || s->kv.head_dim != m->head_dim || s->layer_bytes < 0) return H4B_EINVAL;
    const int q_size = m->heads * m->head_dim, kv_size = m->kv_heads * m->head_dim;
    const int rows[] = {q_size + 2 * kv_size, m->hidden, 2 * m->intermediate, m->vocab};
    for (int r : rows)
        if (r % kGemmRows) return H4B_EUNSUPPORTED;
    const int widths[] = {m->hidden, q_size, m->intermediate};
    for (int w : widths)
        if (w % kGemmK) return H4B_EUNSUPPORTED;
    if (m->intermediate % kSwigluBlock) return H4B_EUNSUPPORTED;
    const void* required[] = {m->w_qkv, m->s_qkv, m->w_o, m->s_o, m->w_gate_up, m->s_gate_up, m->w_down, m->s_down,
                              m->w_embed, m->s_embed, m->norm_in, m->norm_post, m->norm_q, m->norm_k, m->norm_final,
                              m->rope_cos, m->rope_sin, s->tokens, s->x, s->x8, s->act_scale, s->act_sum, s->qkv, s->q,
                              s->attended16, s->attended, s->gate_up, s->act, s->last, s->logits, s->next_tokens,
                              s->workspace};
    for (const void* p : required)
        if (!p || (reinterpret_cast<uintptr_t>(p) & 15)) return H4B_EINVAL;
    return 0;
}

int forward_paged(const h4b_model* m, const h4b_paged_step* s, const int32_t* parents, cudaStream_t stream) {
    int rc = validate_paged_step(m, s);
    if (rc) return rc;
    const int M = s->kv.tokens, B = s->kv.sequences, H = m->hidden, I = m->intermediate, d = m->head_dim;
    const int q_size = m->heads * d, qkv_rows = q_size + 2 * m->kv_heads * d;
    const float scale = 1.0f / sqrtf(static_cast<float>(d));
    auto gemm = [&](const uint8_t* w, const float* ws, float* out, int tokens, int rows, int width, bool residual) {
        GemmArgs g{s->x8, s->act_scale, s->act_sum, w, ws, out, tokens, rows, width};
        g.residual = residual;
        return launch_int4_gemm(g, stream);
    };
    auto norm_quant = [&](float* x, const float* gamma, int tokens) {
        return launch_rmsnorm_quant(x, gamma, m->eps, H, tokens, s->x8, s->act_scale, s->act_sum, stream);
    };
    batch_embed_kernel<<<M, 256, 0, stream>>>(s->tokens, m->w_embed, m->s_embed, m->vocab, H, s->x);
    H4B_CUDA_TRY(cudaGetLastError());
    for (int l = 0; l < m->layers; ++l) {
        h4b_paged_kv kv = s->kv;
        kv.k_pages = static_cast<char*>(s->kv.k_pages) + l * s->layer_bytes;
        kv.v_pages = static_cast<char*>(s->kv.v_pages) + l * s->layer_bytes;
        if ((rc = norm_quant(s->x, m->norm_in + static_cast<size_t>(l) * H, M))) return rc;
        if ((rc = gemm(m->w_qkv + static_cast<size_t>(l) * qkv_rows * (H / 2),
                       m->s_qkv + static_cast<size_t>(l) * qkv_rows, s->qkv, M, qkv_rows, H, false)))
            return rc;
        if ((rc = paged_append(&kv, parents, s->qkv, H4B_FP32, qkv_rows, m->heads, m->norm_q + static_cast<size_t>(l) * d,
                               m->norm_k + static_cast<size_t>(l) * d, m->eps, m->rope_cos, m->rope_sin, m->max_pos, s->q,
                               q_size, stream)))
            return rc;
        if ((rc = paged_attention(&kv, parents, s->q, q_size, m->heads, scale, s->window, s->sinks, s->max_query,
                                  s->attended16, q_size, nullptr, s->workspace, s->workspace_bytes, stream)))
            return rc;
        const long long eights = static_cast<long long>(M) * q_size / 8;
        const int grid = static_cast<int>(std::min((eights + 255) / 256, 148ll * 8));
        if (s->kv.dtype == H4B_FP16)
            widen_kernel<__half><<<grid, 256, 0, stream>>>(static_cast<const uint4*>(s->attended16),
                                                           reinterpret_cast<float4*>(s->attended), eights);
        else
            widen_kernel<__nv_bfloat16><<<grid, 256, 0, stream>>>(static_cast<const uint4*>(s->attended16),
                                                                  reinterpret_cast<float4*>(s->attended), eights);
        H4B_CUDA_TRY(cudaGetLastError());
        if ((rc = launch_quantize_rows<false>(s->attended, q_size, M, s->x8, s->act_scale, s->act_sum, nullptr, stream)))
            return rc;
        if ((rc = gemm(m->w_o + static_cast<size_t>(l) * H * (q_size / 2), m->s_o + static_cast<size_t>(l) * H, s->x, M,
                       H, q_size, true)))
            return rc;
        if ((rc = norm_quant(s->x, m->norm_post + static_cast<size_t>(l) * H, M))) return rc;
        if ((rc = gemm(m->w_gate_up + static_cast<size_t>(l) * 2 * I * (H / 2),
                       m->s_gate_up + static_cast<size_t>(l) * 2 * I, s->gate_up, M, 2 * I, H, false)))
            return rc;
        if ((rc = launch_quantize_rows<true>(s->gate_up, I, M, s->x8, s->act_scale, s->act_sum, s->act, stream)))
            return rc;
        if ((rc = gemm(m->w_down + static_cast<size_t>(l) * H * (I / 2), m->s_down + static_cast<size_t>(l) * H, s->x, M,
                       H, I, true)))
            return rc;
    }
    if (parents != nullptr) {
        if ((rc = norm_quant(s->x, m->norm_final, M))) return rc;
        return gemm(m->w_embed, m->s_embed, s->logits, M, m->vocab, H, false);
    }
    last_rows_kernel<<<B, 256, 0, stream>>>(s->x, s->kv.q_offsets, M, H, s->last);
    H4B_CUDA_TRY(cudaGetLastError());
    if ((rc = norm_quant(s->last, m->norm_final, B))) return rc;
    if ((rc = gemm(m->w_embed, m->s_embed, s->logits, B, m->vocab, H, false))) return rc;
    batch_argmax_kernel<<<B, 1024, 0, stream>>>(s->logits, m->vocab, s->next_tokens);
    H4B_CUDA_TRY(cudaGetLastError());
    return 0;
}

}  // namespace h4b

extern "C" int h4b_forward_paged(const h4b_model* model, const h4b_paged_step* step, void* stream) {
    return h4b::forward_paged(model, step, nullptr, static_cast<cudaStream_t>(stream));
}

extern "C" int h4b_forward_paged_tree(const h4b_model* model, const h4b_paged_step* step, const int32_t* parents,
                                      void* stream) {
    if (parents == nullptr) return H4B_EINVAL;
    return h4b::forward_paged(model, step, parents, static_cast<cudaStream_t>(stream));
}
