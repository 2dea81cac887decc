"""`-m gpu`: the low-bit operators together, as GraphDecoder's captured decode step runs them: penalties and masks against transformers'
generate(), the e4m3 cache and 4-bit weights against the same step written out in plain torch."""
import copy

import pytest
import torch

from test_gpu_lowbit import attention_reference, quantise, rotate

pytestmark = pytest.mark.gpu
BF, F64 = torch.bfloat16, torch.float64


@pytest.fixture(scope="module")
def model():
    """a random Qwen2.5-VL text encoder of the real widths with 3 layers and a small vocabulary"""
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from transformers import Qwen2_5_VLConfig, Qwen2_5_VLForConditionalGeneration
    from diffsynth.pipelines import prompt_prologue as PP
    cfg = copy.deepcopy(PP.TEXT_ENCODER_CONFIG)
    cfg["text_config"].update(num_hidden_layers=3, vocab_size=4001, bos_token_id=1, eos_token_id=2, pad_token_id=0)
    cfg["vision_config"].update(depth=1, fullatt_block_indexes=[0])
    cfg.update(image_token_id=10, video_token_id=11, vision_start_token_id=12, vision_end_token_id=13, bos_token_id=1, eos_token_id=2)
    old = torch.get_default_dtype()
    torch.set_default_dtype(BF)
    try:
        with torch.device("cuda"):
            m = Qwen2_5_VLForConditionalGeneration(Qwen2_5_VLConfig(**cfg))
    finally:
        torch.set_default_dtype(old)
    g = torch.Generator(device="cuda").manual_seed(11)
    with torch.no_grad():
        for name, p in m.named_parameters():
            if p.dim() >= 2:
                p.normal_(0.0, 0.03, generator=g)
            elif "norm" in name:
                p.normal_(1.0, 0.1, generator=g)
            else:
                p.normal_(0.0, 0.02, generator=g)
    m.eval()
    m.generation_config.do_sample = False
    m.generation_config.pad_token_id, m.generation_config.eos_token_id = 0, None
    assert PP.accelerate_decode(m) > 0
    return m


@pytest.fixture
def config(model):
    """the model's generation config, put back afterwards"""
    old = copy.deepcopy(model.generation_config)
    yield model.generation_config
    model.generation_config = old


def prompt(n, seed=3):
    ids = torch.randint(20, 3900, (1, n), generator=torch.Generator().manual_seed(seed)).cuda()
    return {"input_ids": ids, "attention_mask": torch.ones_like(ids)}


def decoder(model, **kw):
    from diffsynth.pipelines import prompt_prologue as PP
    return PP.GraphDecoder(model, chunk=8, **kw)


def test_penalties_and_masks_match_generate(model, config):
    """the same kernels decode both ways and both choices are made in fp32 on the same logits: identical tokens"""
    dec = decoder(model)
    inputs = prompt(37)
    plain = dec.generate(max_new_tokens=24, **inputs)
    config.repetition_penalty = 1.3
    with torch.no_grad():
        want = model.generate(**inputs, max_new_tokens=24, min_new_tokens=24)
    got = dec.generate(max_new_tokens=24, **inputs)
    assert torch.equal(got, want)
    config.suppress_tokens = sorted(set(want[0, 37:45].tolist())) + [4001, 99999]  # what it liked best is taken away; ids outside are nobody's
    with torch.no_grad():
        want2 = model.generate(**inputs, max_new_tokens=24, min_new_tokens=24)
    got2 = dec.generate(max_new_tokens=24, **inputs)
    assert torch.equal(got2, want2) and not set(config.suppress_tokens) & set(got2[0, 37:].tolist())
    assert dec.captures == 2                                                      # one plain step, one that selects
    # a grammar: even and odd ids in turn, from a window that moves with the last token
    def grammar(batch, ids):
        last = int(ids[-1])
        return [i for i in range(max(20, last - 900), min(4000, last + 900)) if (i - last) % 2 == 1]
    config.suppress_tokens = None
    with torch.no_grad():
        want3 = model.generate(**inputs, max_new_tokens=12, min_new_tokens=12, prefix_allowed_tokens_fn=grammar)
    got3 = dec.generate(max_new_tokens=12, prefix_allowed_tokens_fn=grammar, **inputs)
    assert torch.equal(got3, want3)
    toks = got3[0, 36:].tolist()
    assert all((b - a) % 2 for a, b in zip(toks, toks[1:])) and dec.captures == 2
    with pytest.raises(RuntimeError, match="no token is allowed"):
        dec.generate(max_new_tokens=4, prefix_allowed_tokens_fn=lambda b, i: [] if i.numel() > 38 else [500], **inputs)
    for outside in (-1, 4001):
        with pytest.raises(ValueError, match="outside"):
            dec.generate(max_new_tokens=4, prefix_allowed_tokens_fn=lambda b, i: [5, outside], **inputs)
    config.repetition_penalty = 1.0
    assert torch.equal(dec.generate(max_new_tokens=24, **inputs), plain)          # and back to the plain arg-max


def dequantised(w4):
    """the weight that a W4Weight stands for, from the layout's definition (include/physicedit_amd.h, pe_w4_weight), exactly"""
    words = w4.codes.contiguous().view(torch.int32).view(*w4.codes.shape[:2], 4, 16, 4)              # tile, chunk, lane / 16, lane % 16, step
    codes = torch.stack([(words >> (4 * (e // 2 + 4 * (e % 2)))) & 15 for e in range(8)], -1)
    codes = codes.permute(0, 3, 1, 4, 2, 5).reshape(words.shape[0] * 16, -1)[:w4.N, :w4.K].to(F64)
    scale, zero = w4.scale[..., 0].to(F64), -128 - w4.scale[..., 1].to(F64)
    per_input = lambda t: t.transpose(1, 2).reshape(words.shape[0] * 16, -1).repeat_interleave(w4.group, 1)[:w4.N, :w4.K]
    return per_input(scale) * (codes - per_input(zero))


@torch.no_grad()
def plain_step(dec, st):
    """one step of the low-bit decode in plain torch: 64-bit products, each operator's result rounded to bf16 once -> logits, and the caches' new rows"""
    model, lm, pos = dec.model, dec.lm, int(st["step"])
    r = lambda t: t.to(BF).to(F64)
    x = lm.embed_tokens.weight[int(st["token"])].to(F64)
    rows = []
    for l, ly in enumerate(dec.layers):
        at, mlp = ly.self_attn, ly.mlp
        norm = lambda t, n: t / (t.square().mean() + n.variance_epsilon).sqrt()
        if dec.weights == "w4":
            qkv_w, qkv_b, o_w, gu_w, down_w = st["w4"][1][l]
            qkv = r(dequantised(qkv_w) @ norm(x, ly.input_layernorm) + qkv_b.to(F64))
        else:
            n1 = r(r(norm(x, ly.input_layernorm)) * ly.input_layernorm.weight.to(F64))
            qkv = r(torch.cat([p.weight.to(F64) @ n1 + p.bias.to(F64) for p in (at.q_proj, at.k_proj, at.v_proj)]))
        q, k, v = qkv.view(-1, 128).split([28, 4, 4])
        cos, sin = st["cos"][pos].to(F64), st["sin"][pos].to(F64)
        q = rotate(q, cos, sin).to(BF)
        rows.append((*quantise(rotate(k, cos, sin).float()), *quantise(v.float())))
        a = r(attention_reference(q.view(1, 1, 28, 128), st["cache"][l], st["step"], scale=float(at.scaling))[0].view(-1))
        if dec.weights == "w4":
            h = r(x + dequantised(o_w) @ a)
            gate, up = (dequantised(gu_w) @ norm(h, ly.post_attention_layernorm)).chunk(2)
            x = r(h + dequantised(down_w) @ r(gate * torch.sigmoid(gate) * up))
        else:
            h = r(x + r(at.o_proj.weight.to(F64) @ a))
            n2 = r(r(norm(h, ly.post_attention_layernorm)) * ly.post_attention_layernorm.weight.to(F64))
            gate, up = r(mlp.gate_proj.weight.to(F64) @ n2), r(mlp.up_proj.weight.to(F64) @ n2)
            x = r(h + r(mlp.down_proj.weight.to(F64) @ r(r(gate * torch.sigmoid(gate)) * up)))
    if dec.weights == "w4":
        return r(dequantised(st["w4"][2]) @ norm(x, lm.norm)), rows
    return r(model.lm_head.weight.to(F64) @ r(r(norm(x, lm.norm)) * lm.norm.weight.to(F64))), rows


@pytest.mark.parametrize("weights", ["bf16", "w4"])
def test_low_bit_step(model, weights):
    """the step's logits against the plain form.  Both round at the same points, so they differ where a sum of another order falls on the other side
    of a rounding: one step of bf16, 2^-7 of the value, where it does.  A layer has five such points in a row (qkv, attention, h, the gated product,
    x), the head one more; errors of a layer pass through the next with a gain of about one (the residual stream is normed): 16 * 2^-7 at the very
    worst, were every value of every point to fall apart; flips are rare and independent, a hundredth of them: 16 * 2^-7 / 10 for the norm."""
    dec = decoder(model, weights=weights, kv_cache="e4m3")
    inputs = prompt(150, seed=8)
    dec.generate(max_new_tokens=3, **inputs)
    st = next(iter(dec._static.values()))
    for step, token in ((150, 77), (152, 1234)):
        st["step"].fill_(step), st["token"].fill_(token)
        got = dec._step_low_bit(st).to(F64)
        want, rows = plain_step(dec, st)
        err = float((got - want).norm() / want.norm())
        print(f"[parity] low-bit step ({weights}): logits off by {err:.2e}")
        assert err <= 16 * 2.0 ** -7 / 10
        for l, (kq, ks, vq, vs) in enumerate(rows):          # the rows that the step wrote: the same up to the flips of their inputs
            c = st["cache"][l]
            k, v = (t[0, :, step].to(F64) * s[0, :, step, None].to(F64) for t, s in
                    ((c.k, c.k_scale), (c.v.reshape(1, 4, -1, 128), c.v_scale)))
            for a, b in ((k, kq.to(F64) * ks[:, None].to(F64)), (v, vq.to(F64) * vs[:, None].to(F64))):
                assert (a - b).norm() <= 2.0 ** -5 * b.norm()        # e4m3's own half step is 2^-4; a flip of it here and there


@pytest.mark.parametrize("weights", ["bf16", "w4"])
def test_low_bit_decode_is_its_own_steps(model, config, weights):
    """the captured step, replayed, gives the tokens of the same step run eagerly; another prompt and a repetition penalty reuse and re-capture it"""
    dec = decoder(model, weights=weights, kv_cache="e4m3")

    def eager(n, Lp, first):
        st = next(iter(dec._static.values()))
        st["step"].fill_(Lp), st["token"].fill_(first)
        for _ in range(n - 1):
            dec._step(st)
        return [first] + st["out_ids"][Lp:Lp + n - 1].tolist()
    for Lp, seed in ((61, 1), (64, 2), (130, 5)):
        inputs = prompt(Lp, seed)
        toks = dec.generate(max_new_tokens=20, **inputs)[0, Lp:].tolist()
        assert toks == eager(20, Lp, toks[0])
    assert dec.captures == 1
    config.repetition_penalty = 1.2
    inputs = prompt(70, 6)
    toks = dec.generate(max_new_tokens=20, **inputs)[0, 70:].tolist()
    assert len(set(toks)) > 1 and dec.captures == 2
    assert toks == dec.generate(max_new_tokens=20, **inputs)[0, 70:].tolist() and dec.captures == 2


def test_four_bit_copies_follow_the_weights(model):
    """a weight changed in place, moved, or changed through .data with reset(): new copies and a new capture; nothing otherwise"""
    dec = decoder(model, weights="w4", kv_cache="e4m3")
    inputs = prompt(40, 9)
    a = dec.generate(max_new_tokens=10, **inputs)
    copies = dec._w4
    assert torch.equal(dec.generate(max_new_tokens=10, **inputs), a) and dec._w4 is copies
    head = model.lm_head.weight
    kept = head.detach().clone()
    try:
        with torch.no_grad():
            head.copy_(kept.roll(7, 0))
        b = dec.generate(max_new_tokens=10, **inputs)
        assert dec._w4 is not copies and int(b[0, 40]) == (int(a[0, 40]) + 7) % 4001
        head.data.copy_(kept)
        dec.reset()
        assert torch.equal(dec.generate(max_new_tokens=10, **inputs), a)
    finally:
        with torch.no_grad():
            head.copy_(kept)


def test_low_bit_choices_are_checked(model):
    for kw in (dict(weights="w4", kv_cache="bf16"), dict(weights="int8"), dict(kv_cache="fp8"), dict(weights="w4", kv_cache="e4m3", w4_group=1024)):
        with pytest.raises(ValueError):
            decoder(model, **kw)


def test_a_tree_of_drafts_equals_its_branches(model):
    """the operators in a speculative step: four drafted tokens as a tree over a cache give each branch what decoding it token by token gives"""
    from physicedit_amd import ops
    g = torch.Generator(device="cuda").manual_seed(31)
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda").to(BF)
    n, cos = 100, torch.rand((256, 128), generator=g, device="cuda").to(BF)
    sin = torch.rand((256, 128), generator=g, device="cuda").to(BF)
    ctx = rnd(1, n, 4, 128), rnd(1, n, 4, 128)
    q, k, v = rnd(1, 4, 28, 128), rnd(1, 4, 4, 128), rnd(1, 4, 4, 128)
    parent, depth = [None, 0, 0, 1], [0, 1, 1, 2]                    # 0 -> (1 -> 3, 2)
    start, zero = torch.tensor([n], dtype=torch.int32, device="cuda"), torch.zeros((1,), dtype=torch.int32, device="cuda")
    cache = ops.KVCacheE4M3(1, 4, 192, 128)
    ops.kv_append_e4m3(cache, *ctx, zero)
    pos = torch.tensor([[n + d for d in depth]], dtype=torch.int32, device="cuda")
    words = [1, 3, 5, 11]
    qr = ops.kv_append_e4m3(cache, k, v, start, q=q, cos=cos, sin=sin, positions=pos)
    got = ops.kv_attention_e4m3(qr, cache, start, tree=torch.tensor([words], device="cuda"))
    for leaf in (2, 3):
        path = []
        i = leaf
        while i is not None:
            path.insert(0, i)
            i = parent[i]
        line = ops.KVCacheE4M3(1, 4, 192, 128)
        ops.kv_append_e4m3(line, *ctx, zero)
        for t, i in enumerate(path):
            at = start + t
            one = ops.kv_append_e4m3(line, k[:, i:i + 1], v[:, i:i + 1], at, q=q[:, i:i + 1], cos=cos, sin=sin)
            alone = ops.kv_attention_e4m3(one, line, at)
            assert torch.equal(one[0, 0], qr[0, i])
            # the same numbers in another order of sums, each rounded once: half a step apart on either side
            assert ((got[0, i].float() - alone[0, 0].float()).abs() <= 2.0 ** -7 * alone[0, 0].float().abs() + 2.0 ** -14).all()


@pytest.mark.parametrize("penalty", [1.0, 1.3])
def test_no_eos_before_the_least_number_of_tokens(model, config, penalty):
    """min_new_tokens and min_length keep EOS out of the first tokens and out of the cache, as transformers does; it ends the answer after them"""
    dec = decoder(model)
    inputs = prompt(37)
    config.repetition_penalty = penalty
    free = dec.generate(max_new_tokens=24, **inputs)[0, 37:].tolist()
    stops = 0
    for least in (dict(min_new_tokens=1), dict(min_new_tokens=5), dict(min_new_tokens=11), dict(min_length=37 + 3), dict(min_length=30), dict(min_new_tokens=2, min_length=50),
                  dict(min_new_tokens=0, min_length=50), dict(min_new_tokens=24)):
        for eos in ([free[0]], [free[2], free[6]], [free[0], free[1], free[12]]):
            config.eos_token_id, config.min_new_tokens, config.min_length = eos, least.get("min_new_tokens"), least.get("min_length")
            with torch.no_grad():
                want = model.generate(**inputs, max_new_tokens=24)
            got = dec.generate(max_new_tokens=24, **inputs)
            assert torch.equal(got, want), (least, eos)
            early = least.get("min_new_tokens", max(least.get("min_length", 0) - 37, 0))
            assert not set(got[0, 37:37 + early].tolist()) & set(eos)
            stops += got.shape[1] < 37 + 24
    assert stops > 0
    # with a grammar in force too
    config.eos_token_id, config.min_new_tokens, config.min_length = [500], 4, None
    with torch.no_grad():
        want = model.generate(**inputs, max_new_tokens=8, prefix_allowed_tokens_fn=lambda b, i: [500, 501 + i.numel()])
    assert torch.equal(dec.generate(max_new_tokens=8, prefix_allowed_tokens_fn=lambda b, i: [500, 501 + i.numel()], **inputs), want)
    config.eos_token_id, config.min_new_tokens = None, 5                     # no EOS: nothing to keep out
    assert dec.generate(max_new_tokens=24, **inputs)[0, 37:].tolist() == free


def test_the_e4m3_cache_takes_long_answers(model, config):
    """more rows than the bf16 cache's 15360: the captured step still decodes, and its tokens are those of the same step run eagerly"""
    from diffsynth.pipelines import prompt_prologue as PP
    pp = PP.PromptPrologue.__new__(PP.PromptPrologue)
    pp.text_encoder, pp.graph_decoder, pp.tokenizer = model, decoder(model, kv_cache="e4m3"), None
    dec, inputs, Lp = pp.graph_decoder, prompt(15400, 4), 15400
    got = pp.generate_ids(inputs, 30)
    assert dec.captures == 1 and got.shape == (1, Lp + 30) and torch.equal(got[:, :Lp], inputs["input_ids"])
    toks = got[0, Lp:].tolist()
    st = next(iter(dec._static.values()))
    assert st["cap"] == 16384
    st["step"].fill_(Lp), st["token"].fill_(toks[0])
    for _ in range(29):
        dec._step(st)
    assert toks[1:] == st["out_ids"][Lp:Lp + 29].tolist()
    plain = decoder(model)
    with pytest.raises(ValueError, match="15360"):
        plain.generate(max_new_tokens=30, **inputs)


@pytest.mark.parametrize("weights,kv_cache", [("bf16", "bf16"), ("bf16", "e4m3"), ("w4", "e4m3")])
def test_old_copies_go_before_new_ones_come(model, config, weights, kv_cache):
    """after a change of the weights or of the capacity the memory of the old step is free before the new one's is taken: the peak of a call that builds the
    step again stays at that of the call that built it first"""
    dec = decoder(model, weights=weights, kv_cache=kv_cache)
    config.eos_token_id = list(range(4001))                                    # the first token ends the answer

    def peak(n, **inputs):
        torch.cuda.synchronize(), torch.cuda.empty_cache(), torch.cuda.reset_peak_memory_stats()
        dec.generate(max_new_tokens=n, **inputs)
        torch.cuda.synchronize()
        return torch.cuda.max_memory_allocated() - base
    inputs = prompt(40, 9)
    dec.generate(max_new_tokens=2, **inputs)                                   # the libraries' own workspaces
    dec.reset()
    base = torch.cuda.memory_allocated()
    first = peak(8000, **inputs) if kv_cache == "bf16" else peak(60000, **inputs)
    held = torch.cuda.memory_allocated() - base
    assert held > 2 ** 25                                                      # planes (and copies) of a size that would show
    head = model.lm_head.weight
    try:
        if kv_cache == "bf16":
            head.data = head.data.clone()
        else:
            with torch.no_grad():
                head.mul_(1.0)                                                 # a change that counts and changes nothing
        again = peak(8000, **inputs) if kv_cache == "bf16" else peak(60000, **inputs)
        assert again <= first + held // 8
        other = peak(6000, **inputs) if kv_cache == "bf16" else peak(50000, **inputs)       # another capacity
        assert other <= first + held // 8
    finally:
        dec.reset()


def test_nothing_behind_eos_counts(model, config):
    """the steps that a chunk runs past EOS may find no token at all (scores of NaN here): the answer ended before them"""
    dec = decoder(model)
    inputs = prompt(37)
    config.repetition_penalty = 1.3
    free = dec.generate(max_new_tokens=12, **inputs)
    config.eos_token_id = int(free[0, 37 + 3])
    table = model.model.language_model.embed_tokens.weight
    kept = table[config.eos_token_id].clone()
    try:
        with torch.no_grad():
            table[config.eos_token_id] = float("nan")
        assert torch.equal(dec.generate(max_new_tokens=12, **inputs), free[:, :37 + 4])
        config.eos_token_id = None
        with pytest.raises(RuntimeError, match="no token is allowed"):
            dec.generate(max_new_tokens=12, **inputs)
    finally:
        with torch.no_grad():
            table[int(free[0, 37 + 3])] = kept


@torch.no_grad()
def test_four_bit_copies_stand_for_the_model(model):
    """each 4-bit copy of the step against the model's own tensors: the right matrices in the right order with the right norm's weight in the columns.
    Elementwise: half a step, a scale rounded to bf16 (15 steps / 256) and a zero point rounded to a whole number (half a step), as quantize_w4's own test
    has it.  By column, over N outputs: the copy regressed on the model's weight gives the norm's weight, 1 +- 0.1, up to the quantisation's noise, below
    0.4 of a weight's deviation in each output (a step of (max - min) / 15 of 128 normal values, 0.4, over sqrt 12, the roundings above added), divided by
    sqrt N; six times that."""
    dec = decoder(model, weights="w4", kv_cache="e4m3")
    dec.generate(max_new_tokens=2, **prompt(20, 1))
    _, layers, head = dec._w4
    norms = [ly.input_layernorm.weight for ly in dec.layers] + [ly.post_attention_layernorm.weight for ly in dec.layers] + [dec.lm.norm.weight]
    assert all((a.float() - b.float()).std() > 0.1 for i, a in enumerate(norms) for b in norms[:i])          # told apart below

    def check(copy, weight, norm):
        got, w = dequantised(copy), weight.to(F64)
        n = torch.ones(w.shape[1], dtype=F64, device="cuda") if norm is None else norm.to(F64)
        assert got.shape == w.shape
        exact = w * n
        parts = exact.view(exact.shape[0], -1, copy.group)
        step = ((parts.amax(-1).clamp_min(0) - parts.amin(-1).clamp_max(0)) / 15).repeat_interleave(copy.group, 1)
        assert ((got - exact).abs() <= step * (1.0 + 15 / 256) + 1e-12).all()
        column = (got * w).sum(0) / w.square().sum(0)
        assert ((column - n).abs() <= 6 * 0.4 / w.shape[0] ** 0.5).all()
    for (qkv, bias, o, gate_up, down), ly in zip(layers, dec.layers):
        at, mlp = ly.self_attn, ly.mlp
        check(qkv, torch.cat([at.q_proj.weight, at.k_proj.weight, at.v_proj.weight]), ly.input_layernorm.weight)
        assert torch.equal(bias, torch.cat([at.q_proj.bias, at.k_proj.bias, at.v_proj.bias]))
        check(o, at.o_proj.weight, None)
        check(gate_up, torch.cat([mlp.gate_proj.weight, mlp.up_proj.weight]), ly.post_attention_layernorm.weight)
        check(down, mlp.down_proj.weight, None)
    check(head, model.lm_head.weight, dec.lm.norm.weight)


@torch.no_grad()
@pytest.mark.parametrize("weights", ["bf16", "w4"])
def test_the_prefill_reaches_the_cache(model, weights):
    """the cache's rows after the prefill against the keys and values of the model's own pass: e4m3's half step of each value (2^-4 of it, 2^-10 of the row's
    scale below the smallest normal code) and one of bf16 for a pass whose sums ran in another order"""
    n = 150
    inputs = prompt(n, 8)
    dec = decoder(model, weights=weights, kv_cache="e4m3")
    dec.generate(max_new_tokens=1, **inputs)
    past = model(**inputs, use_cache=True, logits_to_keep=1).past_key_values
    caches = next(iter(dec._static.values()))["cache"]
    assert len(caches) == 3
    for layer, c in zip(past.layers, caches):
        for want, codes, scale in ((layer.keys, c.k, c.k_scale), (layer.values, c.v.reshape(1, 4, -1, 128), c.v_scale)):
            s = scale[0, :, :n, None].to(F64)
            got, want = codes[0, :, :n].to(F64) * s, want[0].to(F64)
            assert ((got - want).abs() <= (2.0 ** -4 + 2.0 ** -7) * want.abs() + (2.0 ** -10 + 448 * 2.0 ** -7 / 64) * s).all()
            assert (got - want).norm() <= 2.0 ** -4 * want.norm() and not codes[0, :, n:].to(F64).any()


def test_a_group_that_no_kernel_takes_is_refused_at_once(model):
    for group in (16, 256, 512, 0):
        with pytest.raises(ValueError, match="groups of"):
            decoder(model, weights="w4", kv_cache="e4m3", w4_group=group)
    assert decoder(model, weights="w4", kv_cache="e4m3", w4_group=32).w4_group == 32
