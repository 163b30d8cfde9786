"""Operators of a serving step over independent requests: what needs no GPU.  Refusals of the C ABI come before any launch, so they can be
looked at on a machine without one; pointers are never read here."""
from __future__ import annotations

import ctypes

import pytest
import torch

from ade_b200 import _lib, decode_ops, kernels, paged, synth

NULL, SHAPE, ALIGN, SCRATCH = -1, -2, -3, -4
P = 4096                                          # an aligned address that nothing reads


def _extend(**kw):
    a = dict(lengths=P, new=P, table=P, free=P, count=P, len_out=P, count_out=P, status=P, slots=P, positions=P, requests=P, work=P, work_bytes=1 << 20, B=4, width=8, stride=8,
             pages=32, page=16, total=4)
    a.update(kw)
    return _lib.load().ade_b200_paged_extend(*a.values(), None)


def _write(**kw):
    a = dict(k=P, v=P, cos=P, sin=P, slots=P, kp=P, vp=P, T=2, heads=2, dim=64, pages=4, page=16, k_row=128, k_head=64, v_row=128, v_head=64, cs_row=64)
    a.update(kw)
    return _lib.load().ade_b200_paged_write(*a.values(), None)


def _attn(**kw):
    a = dict(q=P, cos=P, sin=P, table=P, requests=P, positions=P, kp=P, vp=P, out=P, work=P, work_bytes=1 << 30, T=2, B=2, width=4, stride=4, hq=4, hk=2, dim=64,
             pages=8, page=16, q_row=256, q_head=64, cs_row=64, scale=1.0)
    a.update(kw)
    return _lib.load().ade_b200_paged_attn(*a.values(), None)


def _bank(**kw):
    return _lib.AdeDeltaBank(**{**dict(uq=P, us=P, uz=P, vt=P, vs=P, vz=P, start=P, M=64, N=128, groups=2, deltas=2), **kw})


def _delta(bank=None, **kw):
    a = dict(x=P, y=P, bank=ctypes.byref(bank or _bank()), ids=P, out=P, work=P, work_bytes=1 << 30, T=2)
    a.update(kw)
    return _lib.load().ade_b200_multi_delta(*a.values(), None)


def _logprobs(**kw):
    a = dict(x=P, dtype=1, tokens=P, logp=P, entropy=P, top_logp=P, top_tok=P, rows=2, vocab=100, stride=100, top=5)
    a.update(kw)
    return _lib.load().ade_b200_token_logprobs(*a.values(), None)


@pytest.mark.parametrize("call, code", [
    (lambda: _extend(lengths=None), NULL), (lambda: _extend(slots=None), NULL), (lambda: _extend(status=None), NULL),
    (lambda: _extend(B=0), SHAPE), (lambda: _extend(B=4097), SHAPE), (lambda: _extend(width=0), SHAPE), (lambda: _extend(stride=7), SHAPE),
    (lambda: _extend(pages=0), SHAPE), (lambda: _extend(page=0), SHAPE), (lambda: _extend(total=-1), SHAPE),
    (lambda: _extend(width=1 << 20, stride=1 << 20, page=2048), SHAPE), (lambda: _extend(total=(1 << 30) + 1), SHAPE),
    (lambda: _extend(work=None, total=5000), NULL), (lambda: _extend(work=P + 4), ALIGN), (lambda: _extend(work_bytes=16, total=5000), SCRATCH),
    (lambda: _write(k=None), NULL), (lambda: _write(cos=None), NULL), (lambda: _write(slots=None), NULL), (lambda: _write(T=0), SHAPE),
    (lambda: _write(heads=0), SHAPE), (lambda: _write(dim=48), SHAPE), (lambda: _write(dim=288), SHAPE), (lambda: _write(dim=0), SHAPE),
    (lambda: _write(page=0), SHAPE), (lambda: _write(k_row=-128), SHAPE), (lambda: _write(kp=P + 8), ALIGN), (lambda: _write(vp=P + 2), ALIGN),
    (lambda: _attn(q=None), NULL), (lambda: _attn(sin=None), NULL), (lambda: _attn(work=None), NULL), (lambda: _attn(T=0), SHAPE),
    (lambda: _attn(hq=3), SHAPE), (lambda: _attn(hk=0), SHAPE), (lambda: _attn(dim=100), SHAPE), (lambda: _attn(stride=3), SHAPE),
    (lambda: _attn(kp=P + 8), ALIGN), (lambda: _attn(out=P + 2), ALIGN), (lambda: _attn(work_bytes=0), SCRATCH),
    (lambda: _delta(x=None), NULL), (lambda: _delta(_bank(vt=None)), NULL), (lambda: _delta(T=0), SHAPE), (lambda: _delta(T=129), SHAPE),
    (lambda: _delta(_bank(N=192)), SHAPE), (lambda: _delta(_bank(M=(1 << 21) + 1)), SHAPE), (lambda: _delta(_bank(N=1 << 22)), SHAPE),
    (lambda: _delta(_bank(M=1 << 21, groups=1 << 12)), SHAPE), (lambda: _delta(_bank(groups=0)), SHAPE), (lambda: _delta(_bank(deltas=0)), SHAPE),
    (lambda: _delta(_bank(uq=P + 4)), ALIGN), (lambda: _delta(y=P + 2), ALIGN), (lambda: _delta(work_bytes=16), SCRATCH),
    (lambda: _logprobs(x=None), NULL), (lambda: _logprobs(logp=None), NULL), (lambda: _logprobs(tokens=None), NULL), (lambda: _logprobs(top_tok=None), NULL),
    (lambda: _logprobs(rows=0), SHAPE), (lambda: _logprobs(vocab=0), SHAPE), (lambda: _logprobs(top=33), SHAPE), (lambda: _logprobs(top=-1), SHAPE),
    (lambda: _logprobs(vocab=4, top=5), SHAPE), (lambda: _logprobs(dtype=3), SHAPE),
])
def test_the_c_abi_refuses(call, code):
    assert call() == code


def test_workspace_sizes():
    lib = _lib.load()
    assert lib.ade_b200_paged_attn_workspace_bytes(4, 32, 8, 128) > 0
    for bad in [(0, 32, 8, 128), (4, 32, 5, 128), (4, 32, 8, 100), (4, 0, 8, 128)]:
        assert lib.ade_b200_paged_attn_workspace_bytes(*bad) == 0
    assert lib.ade_b200_multi_delta_workspace_bytes(1, 4096) > 0
    assert lib.ade_b200_multi_delta_workspace_bytes(129, 4096) == lib.ade_b200_multi_delta_workspace_bytes(0, 4096) == 0


def test_cpu_tensors_are_refused():
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)
    i64 = lambda *s: torch.zeros(*s, dtype=torch.int64)
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)
    bank = kernels.bank_deltas([kernels.pack_int4(synth.random_packed(16, 128, 128, s)) for s in (1, 2)])
    for call in (lambda: paged.paged_extend(i32(2), i32(2), i32(2, 3), i32(6), i32(1), 2, 16),
                 lambda: paged.paged_write(bf(2, 2, 32), bf(2, 2, 32), i64(2), bf(4, 2, 8, 32), bf(4, 2, 8, 32)),
                 lambda: paged.paged_attn_decode(bf(2, 2, 32), i32(2, 3), i32(2), i64(2), bf(4, 2, 8, 32), bf(4, 2, 8, 32), 1.0),
                 lambda: kernels.multi_delta_forward(bf(2, 128), bf(2, 16), bank, i32(2)),
                 lambda: decode_ops.token_logprobs(torch.zeros(2, 9))):
        with pytest.raises(ValueError, match="CUDA device"):
            call()


def test_the_bank_holds_the_deltas_group_by_group():
    packed = [synth.random_packed(24, 256, r, seed=r) for r in (256, 128, 384)]
    forms = [kernels.pack_int4(p) for p in packed]
    bank = kernels.bank_deltas(forms)
    assert bank["start"].tolist() == [0, 2, 3, 6] and (bank["M"], bank["N"]) == (24, 256)
    g = 0
    for p, f in zip(packed, forms):
        for j in range(f["r"] // 128):
            ranks = slice(128 * j, 128 * j + 128)
            assert torch.equal(kernels.unpack_nibbles(bank["uq"][g]), p["U_codes"][:, ranks])
            assert torch.equal(kernels.unpack_nibbles(bank["vt"][g]), p["Vt_codes"][ranks])
            assert torch.equal(bank["us"][g], p["U_scale"][:, j]) and torch.equal(bank["vs"][g], p["Vt_scale"][j])
            assert torch.equal(bank["uz"][g].float(), p["U_zero"][:, j].float()) and torch.equal(bank["vz"][g].float(), p["Vt_zero"][j].float())
            g += 1
    for bad in ([], [forms[0], kernels.pack_int4(synth.random_packed(32, 256, 128, 1))], [{**forms[0], "r": 2176}]):
        with pytest.raises(ValueError):
            kernels.bank_deltas(bad)


def test_status_table_follows_the_header():
    import os
    import re

    header = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "ade_b200.h")).read()
    codes = {int(v): k for k, v in re.findall(r"#define (ADE_PAGED_\w+) (\d+)", header) if int(v)}
    assert set(codes) == set(_lib.PAGED_STATUS) and all(_lib.PAGED_STATUS[c].startswith(n + ":") for c, n in codes.items())
    assert f"ADE_B200_MAX_REQUESTS {paged.MAX_REQUESTS}" in header


@pytest.mark.parametrize("change, why", [({"hidden_act": "gelu"}, "SiLU"),
                                         ({"rope_parameters": {"rope_type": "dynamic", "factor": 2.0, "rope_theta": 10000.0}}, "rotary")])
def test_models_that_a_step_would_answer_differently_are_refused(change, why):
    from transformers import LlamaConfig, LlamaForCausalLM

    from ade_b200.batch_serving import BatchDecoder

    cfg = LlamaConfig(hidden_size=64, intermediate_size=64, num_hidden_layers=1, num_attention_heads=2, vocab_size=50, **change)
    with pytest.raises(ValueError, match=why):
        BatchDecoder(LlamaForCausalLM(cfg).to(torch.bfloat16), 2, 16)


@pytest.mark.parametrize("B, most", [(1, 512), (4, 512), (128, 512), (129, 2048), (1024, 2048), (1025, 4096), (4096, 4096)])
def test_page_allocation_needs_a_workspace_where_it_says_so(B, most):
    """The header names the function and no number of rows: the number depends on the requests."""
    import os

    size = _lib.load().ade_b200_paged_extend_workspace_bytes
    assert size(B, 0) == size(B, most) == 0 and size(B, most + 1) >= 16 * B
    assert _extend(B=B, total=most + 1, work=None, work_bytes=0) == NULL
    assert _extend(B=B, total=most + 1, work_bytes=size(B, most + 1) - 1) == SCRATCH
    assert size(0, 5000) == size(4097, 5000) == 0
    header = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "ade_b200.h")).read()
    assert "may be NULL where that function returns 0" in header and "rows: work may be NULL" not in header
