"""Many requests at once: modules with a delta for every row's own fine-tuned model, and the decoder on a paged cache, against one
model per fine-tune run by transformers."""
from __future__ import annotations

import copy

import pytest
import torch
import torch.nn.functional as F

from ade_b200 import batch_serving, kernels, synth
from ade_b200._lib import AdeKernelError
from ade_b200.batch_serving import BatchDecoder, DeltaRoute, MultiDeltaLinear, attach_multi_deltas
from ade_b200.decode_ops import enable_fused_decode_ops
from ade_b200.serving import LINEAR_MODULE_NAMES, attach_kernel_linears, fuse_kernel_linears

pytestmark = pytest.mark.gpu
DEV = "cuda"
VOCAB = 320


def _llama(kv_heads=2):
    from transformers import LlamaConfig, LlamaForCausalLM

    cfg = LlamaConfig(hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=kv_heads, vocab_size=VOCAB,
                      max_position_embeddings=512)
    torch.manual_seed(0)
    model = LlamaForCausalLM(cfg).to(torch.bfloat16).eval()
    with torch.no_grad():
        model.lm_head.weight.mul_(20.0)                  # logits that tell tokens apart
    return model


def _deltas(sd, seed, skip=()):
    per = {}
    for li in range(2):
        for i, n in enumerate(LINEAR_MODULE_NAMES):
            if (li, n) in skip:
                continue
            d_o, d_i = sd[f"model.layers.{li}.{n}.weight"].shape
            p = synth.random_packed(d_o, d_i, 128 * (1 + (i + seed) % 2), seed=100 * seed + 10 * li + i)
            for k in ("U_scale", "Vt_scale"):
                p[k] = p[k] * 4.0                         # fine-tunes that differ visibly from the base
            per[f"model.layers.{li}.{n}"] = p
    return per


@pytest.fixture(scope="module")
def served():
    """(base model, [one model per fine-tune], the model that serves all of them)."""
    base = _llama()
    sd = {k: v.clone() for k, v in base.state_dict().items()}
    # the second fine-tune has no delta on two modules, the third none but on one
    every = [(li, n) for li in range(2) for n in LINEAR_MODULE_NAMES]
    deltas = [_deltas(sd, 1), _deltas(sd, 2, skip=every[3:5]), _deltas(sd, 3, skip=every[1:])]
    single = []
    for per in deltas:
        m = copy.deepcopy(base)
        attach_kernel_linears(m, sd, per, device=DEV)
        single.append(m.to(DEV))
    many = copy.deepcopy(base)
    n = attach_multi_deltas(many, sd, deltas, device=DEV)
    assert n == 14
    return base.to(DEV), single, many.to(DEV)


def test_modules_route_rows_to_their_models():
    forms = [kernels.pack_int4(synth.random_packed(192, 256, r, seed=r, device=DEV)) for r in (128, 256)]
    W = synth.base_weight(192, 256, 1).to(DEV)
    route = DeltaRoute(3)
    lin = MultiDeltaLinear(W, [forms[0], None, forms[1]], route)
    g = torch.Generator(device=DEV).manual_seed(1)
    for T in (1, 5, 128, 129, 300):                       # above 128 rows in several launches
        x = torch.randn(T, 256, generator=g, device=DEV).to(torch.bfloat16)
        route.ids = None
        y = lin(x)
        assert torch.equal(y, F.linear(x, W))
        ids = torch.randint(-1, 3, (T,), generator=g, device=DEV, dtype=torch.int32)
        route.ids = ids
        got = lin(x.view(1, T, 256))
        assert got.shape == (1, T, 192)
        for lo in range(0, T, 128):
            part = slice(lo, min(T, lo + 128))
            want = kernels.multi_delta_forward(x[part], y[part], lin.bank(), ids[part])
            assert torch.equal(got[0, part], want)
        rows = (ids < 0) | (ids == 1)
        assert torch.equal(got[0][rows], y[rows])
        route.ids = ids[:-1]
        if T > 1:
            with pytest.raises(ValueError, match="route"):
                lin(x)
    assert lin(x[:0]).shape == (0, 192)
    with pytest.raises(ValueError):
        MultiDeltaLinear(W[:64], forms, route)


# Each of the about thirteen tensors that a layer rounds to bfloat16 (projections, rotated queries and keys, attention, products, sums, norms) is off
# by 2^-8 of its values at most on either side; two layers, the final norm and the logits: 2 * 28 * 2^-8 = 0.22 of the logits' own scale if all
# errors pointed the same way.  They do not: as a random walk sqrt(2 * 28) * 2^-8 / sqrt(3) = 0.017.  Four times that is asked for.
WALK = 4 * 0.017


def _check_answer(model, tokens, logprobs, prompt_len):
    """The answer's log probabilities are the model's, and every token is the model's likeliest to within that."""
    with torch.no_grad():
        logits = model(input_ids=tokens[None]).logits[0].float()
    ref = torch.log_softmax(logits, -1)[prompt_len - 1:-1]
    chosen = ref.gather(1, tokens[prompt_len:, None])[:, 0]
    tol = WALK * float(logits.std())
    assert logprobs.shape == chosen.shape
    assert float((chosen - logprobs).abs().max()) <= 2 * tol, float((chosen - logprobs).abs().max())
    assert bool((ref.amax(-1) - chosen <= 2 * tol).all())


def test_a_ragged_batch_of_many_models_answers_as_each_model_alone(served):
    base, single, many = served
    g = torch.Generator().manual_seed(4)
    prompts = [torch.randint(0, VOCAB, (n,), generator=g) for n in (5, 1, 64, 130, 17, 33)]
    models = [0, 1, 2, 0, -1, 1]
    dec = BatchDecoder(many, max_requests=8, max_len=160, page_size=16)
    free = int(dec.free_count)
    answers = dec.generate(prompts, 20, models)
    assert int(dec.free_count) == free and int(dec.lengths.abs().sum()) == 0
    for (tokens, logprobs), p, d in zip(answers, prompts, models):
        assert torch.equal(tokens[:p.numel()].cpu(), p) and tokens.numel() == p.numel() + 20
        _check_answer(base if d < 0 else single[d], tokens, logprobs, p.numel())
    again = dec.generate(prompts, 20, models)             # the captured step, pages and histories are used again
    for a, b in zip(answers, again):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    # the same requests in another order and company: what a request gets does not depend on the others
    order = [3, 0, 5, 1]
    other = dec.generate([prompts[i] for i in order], 20, [models[i] for i in order])
    for i, (tokens, _) in zip(order, other):
        _check_answer(base if models[i] < 0 else single[models[i]], tokens, other[order.index(i)][1], prompts[i].numel())
    # the serving model itself still runs as its base
    ids = prompts[2][None].to(DEV)
    with torch.no_grad():
        assert torch.equal(many(input_ids=ids).logits, base(input_ids=ids).logits)


def test_requests_enter_and_leave_between_steps(served):
    base, single, many = served
    g = torch.Generator().manual_seed(5)
    prompts = [torch.randint(0, VOCAB, (n,), generator=g) for n in (9, 30, 3)]
    dec = BatchDecoder(many, max_requests=2, max_len=64, page_size=8)
    a = dec.add(prompts[0], 0)
    for _ in range(5):
        dec.step()
    b = dec.add(prompts[1], 1)
    for _ in range(7):
        dec.step()
    assert (a, b) == (0, 1) and dec.lengths.tolist() == [9 + 12, 30 + 7]
    _check_answer(single[0], dec.tokens[a, :22].clone(), dec.logprobs[a, 9:22].clone(), 9)
    dec.finish(a)
    c = dec.add(prompts[2], 2)
    assert c == a
    for _ in range(10):
        dec.step()
    _check_answer(single[1], dec.tokens[b, :48].clone(), dec.logprobs[b, 30:48].clone(), 30)
    _check_answer(single[2], dec.tokens[c, :14].clone(), dec.logprobs[c, 3:14].clone(), 3)
    dec.check_status()
    dec.finish(b)
    dec.finish(c)
    assert int(dec.free_count) == 2 * 8
    for bad in (lambda: dec.finish(c), lambda: dec.finish(7), lambda: dec.add(prompts[0], 3), lambda: dec.add(torch.zeros(64, dtype=torch.long)),
                lambda: dec.add(torch.zeros(0, dtype=torch.long)), lambda: dec.generate(prompts, 4), lambda: dec.generate(prompts[:1], 60),
                lambda: dec.generate(prompts[:2], 3, [0])):
        with pytest.raises(ValueError):
            bad()


def test_a_request_that_cannot_grow_is_reported_and_hurts_no_other(served):
    _, single, many = served
    g = torch.Generator().manual_seed(6)
    prompts = [torch.randint(0, VOCAB, (n,), generator=g) for n in (15, 14, 40)]
    dec = BatchDecoder(many, max_requests=3, max_len=64, pages=3, page_size=16)
    a, b = dec.add(prompts[0], 0), dec.add(prompts[1], 1)
    with pytest.raises(AdeKernelError, match="NO_PAGE"):  # 40 tokens on one free page
        dec.add(prompts[2], 2)
    for _ in range(8):                                    # one of the two gets the third page, the other waits at 16 tokens
        dec.step()
    with pytest.raises(AdeKernelError, match="NO_PAGE"):
        dec.check_status()
    first, second = (a, b) if int(dec.lengths[a]) > 16 else (b, a)
    assert int(dec.lengths[second]) == 16
    n = 15 if first == a else 14
    _check_answer(single[0 if first == a else 1], dec.tokens[first, :n + 9].clone(), dec.logprobs[first, n:n + 9].clone(), n)
    dec.finish(first)                                     # its pages let the other go on
    for _ in range(6):
        dec.step()
    m = 15 if second == a else 14
    _check_answer(single[0 if second == a else 1], dec.tokens[second, :23].clone(), dec.logprobs[second, m:23].clone(), m)


def test_an_end_token_stops_its_request_alone(served):
    _, _, many = served
    g = torch.Generator().manual_seed(7)
    prompts = [torch.randint(0, VOCAB, (n,), generator=g) for n in (6, 11, 4)]
    dec = BatchDecoder(many, max_requests=3, max_len=64)
    plain = dec.generate(prompts, 12, [0, 1, 2])
    eos = int(plain[1][0][11 + 4])
    stopped = dec.generate(prompts, 12, [0, 1, 2], eos_token_id=eos)
    for (t, lp), (s, sp), p in zip(plain, stopped, prompts):
        answer = t[p.numel():].tolist()
        n = answer.index(eos) + 1 if eos in answer else 12
        assert s.tolist() == t[:p.numel() + n].tolist() and torch.equal(sp, lp[:n])


def test_plain_and_single_delta_models_are_served_too(served):
    base, single, _ = served
    g = torch.Generator().manual_seed(8)
    prompts = [torch.randint(0, VOCAB, (n,), generator=g) for n in (7, 21)]
    for model in (base, single[0]):
        for tokens, logprobs in BatchDecoder(model, 4, 48, page_size=32).generate(prompts, 9):
            _check_answer(model, tokens, logprobs, tokens.numel() - 9)
    for bad in (lambda: BatchDecoder(torch.nn.Linear(2, 2), 1, 8), lambda: BatchDecoder(_llama(), 1, 8), lambda: BatchDecoder(base, 0, 8), lambda: BatchDecoder(base, 5000, 8)):
        with pytest.raises(ValueError):
            bad()


def test_a_finished_request_leaves_no_report_behind(served):
    _, single, many = served
    g = torch.Generator().manual_seed(9)
    prompts = [torch.randint(0, VOCAB, (n,), generator=g) for n in (16, 16, 5)]
    dec = BatchDecoder(many, max_requests=3, max_len=64, pages=3, page_size=16)
    with pytest.raises(AdeKernelError, match="NO_PAGE"):  # three pages hold the prompts, none is left to grow
        dec.generate(prompts, 4, [0, 1, 2])
    (tokens, logprobs), = dec.generate(prompts[2:], 6, [2])
    _check_answer(single[2], tokens, logprobs, 5)


def test_each_request_has_its_own_end_token(served):
    """A request beside an answer with an end token goes on through that token, and one entered with an end token stops there."""
    _, _, many = served
    g = torch.Generator().manual_seed(10)
    prompts = [torch.randint(0, VOCAB, (n,), generator=g) for n in (12, 8)]

    def run(eos):
        dec = BatchDecoder(many, max_requests=3, max_len=64)
        a, b = dec.add(prompts[0], 0), dec.add(prompts[0], 0, eos_token_id=eos)
        dec.generate(prompts[1:], 8, [1], eos_token_id=eos)
        for _ in range(10):
            dec.step()
        return dec, a, b, dec.tokens[a, 12:int(dec.lengths[a]) + 1].tolist()

    plain = run(None)[3]
    eos = next(t for i, t in enumerate(plain) if 3 <= i < 9 and t not in plain[:i])
    dec, a, b, through = run(eos)
    assert len(through) == len(plain) and int(dec.new_tokens[a]) == 1
    stopped = dec.tokens[b, 12:int(dec.lengths[b]) + 1].tolist()
    assert stopped == plain[:plain.index(eos) + 1] and int(dec.new_tokens[b]) == 0
    dec.check_status()
    # a number's former end token is forgotten; an answer's first token may be its last
    dec.finish(b)
    c = dec.add(prompts[1], 1)
    begin = int(dec.tokens[c, 8])
    assert c == b and int(dec._eos[c]) == -1
    dec.finish(c)
    c = dec.add(prompts[1], 1, eos_token_id=begin)
    dec.step()
    assert int(dec.new_tokens[c]) == 0 and int(dec.lengths[c]) == 8


def test_requests_that_run_already_rest_while_an_answer_is_generated(served):
    """Lengths, histories and reports of requests that were entered before are what they would be without the answer, in the same company."""
    base, single, many = served
    g = torch.Generator().manual_seed(11)
    prompts = [torch.randint(0, VOCAB, (n,), generator=g) for n in (10, 16, 6)]

    def run(answer):
        dec = BatchDecoder(many, max_requests=4, max_len=48, pages=5, page_size=16)
        a, b = dec.add(prompts[0], 0), dec.add(prompts[1], 1)
        for _ in range(3):
            dec.step()
        if answer:
            (tokens, logprobs), = dec.generate(prompts[2:], 9, [2], eos_token_id=int(dec.tokens[a, 12]))
            assert tokens.numel() <= 15
            _check_answer(single[2], tokens, logprobs, 6)
        assert dec.lengths[:2].tolist() == [13, 19]
        for _ in range(3):
            dec.step()
        assert dec.lengths[:2].tolist() == [16, 22]
        return [t[[a, b]][:, 6:23].clone() for t in (dec.tokens, dec.logprobs)]

    for without, beside in zip(run(False), run(True)):
        assert torch.equal(without[0, :11], beside[0, :11]) and torch.equal(without[1], beside[1])
    # a request that waits for a page does not spoil the answers of others, and is still reported afterwards
    dec = BatchDecoder(many, max_requests=4, max_len=64, pages=3, page_size=16)
    a, b = dec.add(prompts[1], 0), dec.add(prompts[1], 1)
    for _ in range(17):
        dec.step()                                        # one has the third page and has filled it by now
    dec.finish(a if int(dec.lengths[a]) == 16 else b)
    waits = b if a in dec._free_slots else a
    assert int(dec.lengths[waits]) == 32
    dec.add(prompts[2], -1)                               # takes the page that was handed back
    dec.step()
    with pytest.raises(AdeKernelError, match="NO_PAGE"):
        dec.check_status()
    c = next(r for r in range(4) if r not in dec._free_slots and r != waits)
    dec.finish(c)
    (tokens, logprobs), = dec.generate(prompts[2:], 5)
    _check_answer(base, tokens, logprobs, 6)
    with pytest.raises(AdeKernelError, match="NO_PAGE"):
        dec.check_status()
    # an answer that fails leaves the others as they were
    with pytest.raises(AdeKernelError, match="NO_PAGE"):
        dec.generate([torch.cat(prompts)[:30]], 5)
    assert int(dec.new_tokens[waits]) == 1 and int(dec.new_tokens.sum()) == 1 and sorted(dec._free_slots) == [r for r in range(4) if r != waits]


def test_a_request_that_found_its_page_after_all_is_well(served):
    _, single, many = served
    g = torch.Generator().manual_seed(12)
    prompts = [torch.randint(0, VOCAB, (n,), generator=g) for n in (16, 16, 4)]
    dec = BatchDecoder(many, max_requests=3, max_len=64, pages=3, page_size=16)
    a, b = dec.add(prompts[0], 0), dec.add(prompts[1], 1)
    for _ in range(3):
        dec.step()
    with pytest.raises(AdeKernelError, match="NO_PAGE"):
        dec.check_status()
    first, second = (a, b) if int(dec.lengths[a]) > 16 else (b, a)
    dec.finish(first)
    dec.new_tokens[second] = 0                            # resting: its last attempt failed, and that stays
    dec.step()
    with pytest.raises(AdeKernelError, match=f"request {second}: ADE_PAGED_NO_PAGE"):
        dec.check_status()
    dec.new_tokens[second] = 1
    dec.step()
    dec.check_status()
    (tokens, logprobs), = dec.generate(prompts[2:], 5, [2])
    _check_answer(single[2], tokens, logprobs, 4)
    dec.check_status()
    assert int(dec.lengths[second]) == 17


@pytest.mark.parametrize("fails", ["paged_write", "token_logprobs", "model"])
def test_a_request_that_fails_on_its_way_in_leaves_nothing_behind(served, monkeypatch, fails):
    """Whatever raises behind the allocation of its pages: number, pages, length and the rows' models are as before."""
    _, single, many = served
    g = torch.Generator().manual_seed(13)
    prompts = [torch.randint(0, VOCAB, (n,), generator=g) for n in (20, 7)]
    dec = BatchDecoder(many, max_requests=2, max_len=64, page_size=8)
    a = dec.add(prompts[1], 0)
    before = [t.clone() for t in (dec.lengths, dec.new_tokens, dec.status, dec.free_count, dec._model_of)]
    taken = sorted(dec.free_pages[:int(dec.free_count)].tolist())

    def broken(*args, **kw):
        raise RuntimeError("planted")

    with monkeypatch.context() as m:
        if fails == "model":
            m.setattr(many, "forward", broken)
        else:
            m.setattr(batch_serving, fails, broken)
        for _ in range(3):
            with pytest.raises(RuntimeError, match="planted"):
                dec.add(prompts[0], 1)
    assert many._ade_route.ids is None and dec._free_slots == [1]
    for t, kept in zip((dec.lengths, dec.new_tokens, dec.status, dec.free_count, dec._model_of), before):
        assert torch.equal(t, kept)
    assert sorted(dec.free_pages[:int(dec.free_count)].tolist()) == taken
    b = dec.add(prompts[0], 1)
    for _ in range(6):
        dec.step()
    _check_answer(single[0], dec.tokens[a, :14].clone(), dec.logprobs[a, 7:14].clone(), 7)
    _check_answer(single[1], dec.tokens[b, :27].clone(), dec.logprobs[b, 20:27].clone(), 20)


def test_hooks_are_looked_for_again_before_the_step_is_captured(served):
    """A hook on a module that a step does not call is refused, whenever it came; the framework's and transformers' own changes are not."""
    base, _, _ = served
    g = torch.Generator().manual_seed(14)
    prompt = torch.randint(0, VOCAB, (9,), generator=g)
    model = copy.deepcopy(base)
    dec = BatchDecoder(model, 2, 48)
    a = dec.add(prompt)
    handle = model.model.layers[1].register_forward_hook(lambda mod, args, out: out * 2)
    for _ in range(2):
        with pytest.raises(ValueError, match=r"model\.layers\.1 has hooks"):
            dec.step()
    assert int(dec.lengths[a]) == 9 and int(dec.new_tokens[a]) == 1
    handle.remove()
    enable_fused_decode_ops(model)
    with torch.no_grad():
        assert len(model(input_ids=prompt[None].to(DEV), output_hidden_states=True).hidden_states) == 3
    for _ in range(5):
        dec.step()
    _check_answer(base, dec.tokens[a, :15].clone(), dec.logprobs[a, 9:15].clone(), 9)
    dec.finish(a)
    for tokens, logprobs in BatchDecoder(model, 2, 48).generate([prompt, prompt[:3]], 7):
        _check_answer(base, tokens, logprobs, tokens.numel() - 7)


@pytest.mark.parametrize("where", ["model.layers.0.self_attn.o_proj", "model.layers.1.mlp.gate_proj", "model.layers.1.mlp.up_proj", "model.layers.0.mlp.down_proj", "model.embed_tokens"])
def test_modules_that_return_another_type_are_refused(served, where):
    """The launches of a step take what modules return by its address; a type that they do not have is refused before the first of them."""
    _, _, many = served
    model = copy.deepcopy(many)
    model.get_submodule(where).register_forward_hook(lambda mod, args, out: out.float())
    dec = BatchDecoder(model, 2, 48)
    with pytest.raises(ValueError, match="return bfloat16"):
        dec.step()
    assert dec._graph is None and int(dec.lengths.sum()) == 0


@pytest.mark.parametrize("configured, kept", [(1, 2), (2, 1)])
def test_a_model_of_fewer_layers_than_it_has_or_says(configured, kept):
    """transformers runs the first num_hidden_layers of a model's layers, and the final norm behind the last of those."""
    model = _llama()
    model.config.num_hidden_layers = configured
    model.model.layers = model.model.layers[:kept]
    g = torch.Generator().manual_seed(15)
    with torch.no_grad():
        for n, p in model.named_parameters():
            if "norm" in n:
                p.copy_(1 + 0.5 * torch.randn(p.shape, generator=g))
    model = model.to(DEV)
    prompts = [torch.randint(0, VOCAB, (n,), generator=g) for n in (6, 19)]
    dec = BatchDecoder(model, 2, 48)
    assert len(dec.k_pages) == 1
    for tokens, logprobs in dec.generate(prompts, 9):
        _check_answer(model, tokens, logprobs, tokens.numel() - 9)


def test_more_requests_than_one_launch_of_the_deltas_takes(served):
    """A captured step of 150 rows: the deltas in two launches a module, pages and rows by one CTA of 512 threads; a few rest, a few have left."""
    base, single, many = served
    g = torch.Generator().manual_seed(16)
    R = 150
    dec = BatchDecoder(many, max_requests=R, max_len=32, page_size=4)
    free = int(dec.free_count)
    prompts = [torch.randint(0, VOCAB, (1 + i % 6,), generator=g) for i in range(R)]
    models = [i % 4 - 1 for i in range(R)]
    assert [dec.add(p, d) for p, d in zip(prompts, models)] == list(range(R))
    for i in (0, 40, 127):
        dec.finish(i)
    dec.new_tokens[60:63] = 0
    for _ in range(11):
        dec.step()
    dec.check_status()
    gone, rest = {0, 40, 127}, {60, 61, 62}
    assert dec.lengths.tolist() == [0 if i in gone else prompts[i].numel() + (0 if i in rest else 11) for i in range(R)]
    for i in (1, 2, 3, 60, 126, 128, 129, 130, R - 1):
        n, more = prompts[i].numel(), 0 if i in rest else 11
        _check_answer(base if models[i] < 0 else single[models[i]], dec.tokens[i, :n + more + 1].clone(), dec.logprobs[i, n:n + more + 1].clone(), n)
    for i in set(range(R)) - gone:
        dec.finish(i)
    assert int(dec.free_count) == free


def test_fused_groups_of_a_single_model_are_served_too(served):
    """q/k/v and gate/up of a layer as one launch each, next to the other fused operations: prompts through their forwards, steps past them."""
    _, single, _ = served
    model = copy.deepcopy(single[1])
    g = torch.Generator().manual_seed(17)
    prompts = [torch.randint(0, VOCAB, (n,), generator=g) for n in (7, 40, 1)]
    assert fuse_kernel_linears(model) > 0
    enable_fused_decode_ops(model)
    for tokens, logprobs in BatchDecoder(model, 4, 64, page_size=8).generate(prompts, 10):
        _check_answer(single[1], tokens, logprobs, tokens.numel() - 10)


def test_a_decoder_serves_the_deltas_it_was_made_for(served):
    """Deltas attached anew have a route of their own, which the decoder would not set: requests of fine-tuned models would get the base's answers."""
    base, single, many = served
    model = copy.deepcopy(many)
    g = torch.Generator().manual_seed(18)
    prompt = torch.randint(0, VOCAB, (9,), generator=g)
    early, used, plain = BatchDecoder(model, 2, 48), BatchDecoder(model, 2, 48), BatchDecoder(copy.deepcopy(base), 2, 48)
    a = used.add(prompt, 0)
    used.step()
    sd = {k: v.clone() for k, v in base.state_dict().items()}
    attach_multi_deltas(model, sd, [_deltas(sd, 2), _deltas(sd, 1)], device=DEV)
    attach_multi_deltas(plain.model, sd, [_deltas(sd, 2)], device=DEV)
    for call in (lambda: early.add(prompt, 0), early.step, lambda: used.add(prompt, 0), used.step, lambda: plain.add(prompt), plain.step, lambda: early.generate([prompt], 3, [0])):
        with pytest.raises(ValueError, match="other deltas"):
            call()
    used.finish(a)
    (tokens, logprobs), = BatchDecoder(model, 2, 48).generate([prompt], 8, [1])
    _check_answer(single[0], tokens, logprobs, 9)


@pytest.mark.parametrize("where", ["cpu", DEV])
def test_token_ids_that_the_embedding_does_not_have_are_refused(served, where):
    """On the host: the embedding's own look-up would end the process's CUDA context."""
    base, _, _ = served
    dec = BatchDecoder(base, 2, 48)
    free = int(dec.free_count)
    for bad in ([0, VOCAB], [-1, 3], [2 ** 40], [5, -2 ** 31, 7]):
        with pytest.raises(ValueError, match=f"0 to {VOCAB - 1}"):
            dec.add(torch.tensor(bad, device=where))
    assert int(dec.free_count) == free and dec._free_slots == [1, 0]
    a = dec.add(torch.tensor([0, VOCAB - 1], device=where))
    dec.step()
    _check_answer(base, dec.tokens[a, :4].clone(), dec.logprobs[a, 2:4].clone(), 2)
