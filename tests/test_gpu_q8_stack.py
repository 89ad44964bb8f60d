"""GPU: the hybrid stack with its feed-forward in 8-bit integers (int8_weights 2).

With the attention layers' output projections at zero the residual stream changes through the feed-forwards alone, so that the public operators, called one
after the other on the same rows, have to give it bit for bit."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

LAYERS, INTER, VOCAB, WIDTH = 4, 192, 640, 1024


def make(synth, seed, zero_attention):
    from oracle import cpu_stack
    w = cpu_stack.make_stack_weights(synth, seed, LAYERS, INTER, VOCAB, int8=False, norm_std=0.1)
    for lw in w["layers"]:
        if zero_attention:
            lw.update({k: dict(lw[k], **{n: np.zeros_like(lw[k][n])}) for k, n in (("fa", "wo"), ("la", "w_out")) if lw.get(k) is not None})
    return w


def build(ops, w, seqs, tokens, chunk, int8=2):
    st = ops.HybridStack(num_layers=LAYERS, intermediate_size=INTER, vocab_size=VOCAB, max_seqs=seqs, max_seq_len=tokens, prefill_chunk_seqs=chunk, kv_dtype=1,
                         int8_weights=int8)
    for i, lw in enumerate(w["layers"]):
        st.set_layer_weights(i, lw, lw["ffn"], fa=lw.get("fa"), la=lw.get("la"))
    st.set_embedding(w["embed"], w["final_norm"])
    return st


def embedding(torch, w):
    """Rows as the stack holds them: codes per row (ties away from zero), times the scale, in fp16."""
    e = torch.from_numpy(w["embed"]).float()
    s = e.abs().amax(1, keepdim=True) / torch.tensor(127.0)
    s = torch.where(s > 1e-8, s, torch.ones_like(s))
    q = (e / s).double()
    return ((torch.sign(q) * torch.floor(q.abs() + 0.5)).clamp(-127, 127).float() * s).half().cuda()


class Reference:
    def __init__(self, torch, ops, w):
        self.torch, self.ops = torch, ops
        self.embed, self.final = embedding(torch, w), torch.from_numpy(w["final_norm"]).float().cuda()
        dev = lambda a: torch.from_numpy(np.ascontiguousarray(a, dtype=np.float32)).cuda()      # noqa: E731
        self.layers = [(1 + dev(lw["post_norm"]), ops.Int8GatedLinear(dev(lw["ffn"]["gate"]), dev(lw["ffn"]["up"])), ops.Int8Linear(dev(lw["ffn"]["down"])))
                       for lw in w["layers"]]

    def hidden(self, tokens):
        """Final normalised rows, all of them in one pass; fp64."""
        torch, h = self.torch, self.embed[tokens.reshape(-1).long()].float()
        for pre, gated, down in self.layers:
            _, codes, scales = self.ops.norm_block(h, pre_w=pre)
            down.forward(gated.forward_codes(codes, scales, out_dtype=torch.float16), out=h, accumulate=True)
        h = h.double()
        return h / torch.sqrt(h.square().mean(1, keepdim=True) + 1e-6) * (1 + self.final.double())

    def check_tokens(self, tokens, picked):
        """The head multiplies fp16 rows: a logit is off by at most 2^-10 of the sum of its terms, and the one picked is the largest but for that."""
        x, e = self.hidden(tokens), self.embed.double()
        logits, slack = x @ e.T, (x.abs() @ e.abs().T) * 2.0 ** -10
        at = picked.reshape(-1, 1).long()
        assert (logits.gather(1, at) + slack.gather(1, at) >= (logits - slack).amax(1, keepdim=True)).all()


@pytest.mark.parametrize("seqs,tokens,chunk", [(1, 1, 1), (1, 9, 1), (3, 5, 3), (1, 16, 1), (1, 17, 1), (4, 32, 4), (5, 77, 5), (5, 77, 2), (3, 430, 3)])
def test_prompts(ops, cuda, synth, seqs, tokens, chunk):
    torch = cuda
    w = make(synth, 60 + tokens, True)
    st, ref = build(ops, w, seqs, tokens, chunk), Reference(cuda, ops, w)
    toks = torch.from_numpy(synth.rng(5, "q8.tokens").integers(0, VOCAB, (seqs, tokens)).astype(np.int32)).cuda()
    _, hid = st.forward_batch_prefill(toks, want_hidden=True)
    assert st.device_status() == 0
    for s0 in range(0, seqs, chunk):
        part = toks[s0:s0 + chunk]
        want = ref.hidden(part).reshape(len(part), tokens, WIDTH)[:, -1]
        err = (hid[s0:s0 + chunk].double() - want).abs()
        # the same bits in front of the final norm; its sum of 1024 squares, root and quotient are off by less than 16 steps of fp32
        assert (err <= 16 * 2.0 ** -23 * want.abs()).all(), (err / want.abs()).max()


@pytest.mark.parametrize("rows,gemm", [(1, ""), (4, ""), (16, ""), (17, ""), (40, ""), (130, ""), (3, "tc"), (20, "tc"), (3, "cublas"), (20, "cublas")])
def test_decode_steps(ops, cuda, synth, monkeypatch, rows, gemm):
    """Eager and captured steps, few rows (up to 16) and more, under every choice of the other projections' kernels."""
    torch = cuda
    if gemm:
        monkeypatch.setenv("B200ATTN_DECODE_GEMM", gemm)
    w = make(synth, 90 + rows, True)
    st, ref = build(ops, w, rows, 16, 1), Reference(cuda, ops, w)
    toks = torch.from_numpy(synth.rng(6, "q8.tokens").integers(0, VOCAB, (rows,)).astype(np.int32)).cuda()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        out = st.forward_batch_decode(toks)
        s.synchronize()
        ref.check_tokens(toks, out)
        st.capture_decode(rows)
        st.set_tokens(out)
        st.launch_decode(1)
        again = st.get_tokens(rows)
        s.synchronize()
    ref.check_tokens(out, again)
    assert st.device_status() == 0


def test_single_tokens_give_the_logits_of_the_rows(ops, cuda, synth):
    torch = cuda
    w = make(synth, 33, True)
    st, ref = build(ops, w, 2, 64, 1), Reference(cuda, ops, w)
    toks = torch.from_numpy(synth.rng(7, "q8.tokens").integers(0, VOCAB, (5,)).astype(np.int32)).cuda()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        st.begin_batching()
        row = st.open(16)
        for t in toks:
            logits = st.extend(row, t.reshape(1), want=(0,))
            s.synchronize()
            x, e = ref.hidden(t), ref.embed.double()
            assert ((logits.double() - x @ e.T).abs() <= (x.abs() @ e.abs().T) * 2.0 ** -10).all()
    assert st.device_status() == 0


@pytest.mark.parametrize("seqs,tokens", [(2, 40), (3, 200)])
def test_against_the_stack_with_16_bit_products(ops, cuda, synth, seqs, tokens):
    """The whole stack, attention included: the two differ by the quantised activations alone.  Half a code is a / 254 of a row's largest value a.  A normalised
    row of 1024 values has a below 4.5 of its root mean square but for one row in a hundred, the product of gate and up below 12; errors of half a code that
    are spread evenly have a third of that as their root mean square in the square, so a feed-forward's input is off by 4.5 / 254 / sqrt(3) = 1.0 % and the
    input of its down projection by 2.8 %, 3 % together, doubled for the gate's slope and rows beyond these bounds.  Every layer adds one such part to
    the residual stream, no part is larger than the stream, and the parts' errors do not depend on one another: sqrt(4) * 6 %."""
    torch = cuda
    w = make(synth, 44, False)
    toks = torch.from_numpy(synth.rng(8, "q8.tokens").integers(0, VOCAB, (seqs, tokens)).astype(np.int32)).cuda()
    hid = []
    for int8 in (1, 2):
        st = build(ops, w, seqs, tokens, seqs, int8)
        hid.append(st.forward_batch_prefill(toks, want_hidden=True)[1])
        assert st.device_status() == 0
    rel = (hid[1] - hid[0]).norm() / hid[0].norm()
    assert 0 < rel <= 0.12, rel


def test_model_folder_key(ops, cuda):
    import importlib
    import __graft_entry__ as entry
    models = importlib.import_module(entry.PKG_NAME + ".models")
    cfg = dict(architecture="Qwen3_5Hybrid", num_layers=1, intermediate_size=64, vocab_size=64)
    for given, want in ((None, 0), (False, 0), (True, 1), (2, 2)):
        st = models.build_model(dict(cfg, **({} if given is None else dict(int8_weights=given))), models.Limits(max_seqs=1, max_seq_len=64))
        assert st.cfg.int8_weights == want
