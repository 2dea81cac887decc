"""CPU checks of which path PromptPrologue decodes on: the captured step only for what it applies itself, transformers for the rest."""
import types

import pytest
import torch
from transformers import GenerationConfig

from diffsynth.pipelines import prompt_prologue as PP


class Recorder:
    """stands for the captured decoder and for the text encoder: notes which of them was asked, and how"""
    max_rows, low_bit = PP.GraphDecoder.MAX_CACHE_ROWS, False

    def __init__(self, calls, name):
        self.calls, self.name = calls, name

    def generate(self, **kw):
        self.calls.append((self.name, kw))
        return kw["input_ids"]


def prologue(**config):
    calls = []
    pp = PP.PromptPrologue.__new__(PP.PromptPrologue)
    pp.text_encoder, pp.graph_decoder, pp.tokenizer = Recorder(calls, "transformers"), Recorder(calls, "captured"), "the tokenizer"
    pp.text_encoder.generation_config = GenerationConfig(eos_token_id=2, pad_token_id=0, **config)
    return pp, calls


INPUTS = dict(input_ids=torch.zeros((1, 5), dtype=torch.long))
OTHERS = [dict(do_sample=True), dict(num_beams=2), dict(no_repeat_ngram_size=2), dict(bad_words_ids=[[3]]), dict(forced_eos_token_id=2), dict(forced_eos_token_id=0),
          dict(begin_suppress_tokens=[4]), dict(sequence_bias=[[[4], 1.0]]), dict(encoder_repetition_penalty=1.2), dict(encoder_no_repeat_ngram_size=2),
          dict(forced_bos_token_id=0), dict(exponential_decay_length_penalty=(3, 1.1)), dict(remove_invalid_values=True), dict(guidance_scale=1.5),
          dict(max_time=1.0), dict(prompt_lookup_num_tokens=3)]


@pytest.mark.parametrize("more", OTHERS, ids=lambda d: next(iter(d)))
@pytest.mark.parametrize("penalty", [dict(), dict(repetition_penalty=1.3), dict(suppress_tokens=[7])], ids=["plain", "penalty", "suppressed"])
def test_what_the_captured_step_does_not_apply_goes_to_transformers(more, penalty):
    pp, calls = prologue(**more, **penalty)
    pp.generate_ids(INPUTS, 9)
    assert [c[0] for c in calls] == ["transformers"] and calls[0][1]["max_new_tokens"] == 9


@pytest.mark.parametrize("config", [dict(), dict(repetition_penalty=1.3), dict(suppress_tokens=[7, 8]), dict(min_new_tokens=4), dict(min_length=9, repetition_penalty=0.8),
                                    dict(temperature=0.1, top_k=1, top_p=0.5, do_sample=False, num_beams=1, guidance_scale=1.0, no_repeat_ngram_size=0)])
def test_what_the_captured_step_applies_stays_there(config):
    pp, calls = prologue(**config)
    grammar = lambda b, ids: [3]
    pp.generate_ids(INPUTS, 9)
    pp.generate_ids(INPUTS, 9, prefix_allowed_tokens_fn=grammar)
    assert [(c[0], c[1]["prefix_allowed_tokens_fn"]) for c in calls] == [("captured", None), ("captured", grammar)]


def test_stop_strings_come_with_the_tokenizer():
    pp, calls = prologue(stop_strings=["."])
    pp.generate_ids(INPUTS, 9)
    assert calls[0][0] == "transformers" and calls[0][1]["tokenizer"] == "the tokenizer" and "prefix_allowed_tokens_fn" not in calls[0][1]


def test_a_penalty_that_is_none_at_all_is_refused_by_transformers():
    pp, calls = prologue()
    pp.text_encoder.generation_config = types.SimpleNamespace(repetition_penalty=0.0)
    pp.generate_ids(INPUTS, 9)
    assert calls[0][0] == "transformers"


class Processor:
    class tokenizer:
        convert_tokens_to_ids = staticmethod(lambda t: 5)


def build(monkeypatch, fail=None, device="cuda", **kw):
    """a PromptPrologue whose captured decoder is a stand-in (or fails); -> what the decoder was asked for"""
    asked = []

    class Decoder(PP.GraphDecoder):
        def __init__(self, model, weights=None, kv_cache=None):
            asked.append(self.choice(weights, kv_cache))
            if fail:
                raise ValueError(fail)
    monkeypatch.setattr(PP, "GraphDecoder", Decoder)
    monkeypatch.setattr(PP, "accelerate_decode", lambda m: 1)
    pp = PP.PromptPrologue(object(), Processor(), device=device, **kw)
    return asked, pp


LOW = [("w4", "e4m3"), (None, "e4m3"), ("w4", None), ("int8", None)]


@pytest.mark.parametrize("weights,cache", LOW)
@pytest.mark.parametrize("where", ["arguments", "environment"])
def test_a_low_bit_choice_is_used_or_refused(monkeypatch, weights, cache, where):
    kw = {}
    for name, var, value in (("decode_weights", "PE_DECODE_WEIGHTS", weights), ("decode_kv_cache", "PE_DECODE_KV_CACHE", cache)):
        monkeypatch.delenv(var, raising=False)
        if value is not None:
            monkeypatch.setenv(var, value) if where == "environment" else kw.update({name: value})
    asked, pp = build(monkeypatch, **kw)
    assert asked == [(weights or "bf16", cache or "bf16")] and pp.graph_decoder is not None
    with pytest.raises(ValueError, match="does not fit"):
        build(monkeypatch, fail="does not fit", **kw)
    for off in (dict(decode_graph=False), dict(decode_gemv=False), dict(device="cpu")):
        with pytest.raises(ValueError, match="captured decode step"):
            build(monkeypatch, **kw, **off)


def test_bf16_falls_back(monkeypatch, capsys):
    for var in ("PE_DECODE_WEIGHTS", "PE_DECODE_KV_CACHE"):
        monkeypatch.delenv(var, raising=False)
    assert build(monkeypatch, fail="another architecture")[1].graph_decoder is None and "another architecture" in capsys.readouterr().out
    assert build(monkeypatch, decode_graph=False)[1].graph_decoder is None and build(monkeypatch, device="cpu")[1].graph_decoder is None
    monkeypatch.setenv("PE_DECODE_WEIGHTS", "w4"), monkeypatch.setenv("PE_DECODE_KV_CACHE", "e4m3")
    assert build(monkeypatch, decode_weights="bf16", decode_kv_cache="bf16", device="cpu")[1].graph_decoder is None       # the arguments come first
    assert PP.PromptPrologue(None, Processor(), device="cpu").graph_decoder is None                                       # nothing to decode with


def test_the_caches_have_limits_of_their_own():
    """beyond the bf16 cache's rows only the bf16 decoder leaves the captured step"""
    long = dict(input_ids=torch.zeros((1, 15000), dtype=torch.long))
    for kv_cache, path in (("bf16", "transformers"), ("e4m3", "captured")):
        pp, calls = prologue()
        pp.graph_decoder.max_rows = PP.GraphDecoder.max_rows.fget(types.SimpleNamespace(kv_cache=kv_cache, MAX_CACHE_ROWS=PP.GraphDecoder.MAX_CACHE_ROWS,
                                                                                        MAX_CACHE_ROWS_E4M3=PP.GraphDecoder.MAX_CACHE_ROWS_E4M3))
        pp.generate_ids(long, 1000)
        pp.generate_ids(long, 360)
        assert [c[0] for c in calls] == [path, "captured"]


def test_a_low_bit_decoder_that_is_passed_over_says_so(capsys):
    for weights, kv_cache, told in (("bf16", "bf16", False), ("bf16", "e4m3", True), ("w4", "e4m3", True)):
        for config, inputs, path in ((dict(no_repeat_ngram_size=2), INPUTS, "transformers"), (dict(), dict(input_ids=torch.zeros((2, 5), dtype=torch.long)), "transformers"),
                                     (dict(), INPUTS, "captured")):
            pp, calls = prologue(**config)
            pp.graph_decoder.low_bit = PP.GraphDecoder.low_bit.fget(types.SimpleNamespace(weights=weights, kv_cache=kv_cache))
            pp.generate_ids(inputs, 9)
            assert calls[0][0] == path and ("bf16 weights" in capsys.readouterr().out) == (told and path == "transformers")
