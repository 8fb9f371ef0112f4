"""The sequence operators' argument blocks, frequencies and refusals, without a
GPU: what is wrong with a call is said before the device is asked for."""
import itertools
import math
import os
import re

import pytest
import torch

from catfuse_amd import _hip, kernels, sequence

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = open(os.path.join(ROOT, "include", "catfuse_amd.h")).read()
INVALID = 1


@pytest.mark.parametrize("cname,block", [("CfDecayAttentionArgs", _hip.DECAY_ATTENTION_ARGS),
                                         ("CfDecayStepArgs", _hip.DECAY_STEP_ARGS),
                                         ("CfRotaryArgs", _hip.ROTARY_ARGS)])
def test_blocks_mirror_the_header(cname, block):
    body = re.search(r"typedef struct " + cname + r" \{(.*?)\} " + cname + ";", HEADER,
                     re.S).group(1)
    kinds = ""
    for line in body.split(";"):
        if line.strip():
            kind = "Q" if "*" in line else "q" if "int64_t" in line else "d"
            assert kind != "d" or "double" in line
            kinds += kind * (line.count(",") + 1)
    want = "".join(f"{n}{c}" if n > 1 else c
                   for c, n in ((c, len(list(g))) for c, g in itertools.groupby(kinds)))
    assert block[0].format + block[1].format[1:] == "=" + want
    assert block[0].size + block[1].size == 8 * len(kinds)


def test_limits_mirror_the_header():
    def limit(name):
        return int(re.search(rf"#define {name} (\d+)", HEADER).group(1))
    assert sequence.MAX_HEADS == limit("CF_SEQ_MAX_HEADS")
    assert sequence.MAX_KEY_DIM == limit("CF_DECAY_MAX_DK")
    assert sequence.MAX_VALUE_DIM == limit("CF_DECAY_MAX_DV")
    assert sequence.MAX_SEQUENCES == limit("CF_DECAY_MAX_SEQS")
    assert sequence.MAX_ROTARY_DIM == limit("CF_ROTARY_MAX_DIM")
    assert sequence.MAX_TOKENS == limit("CF_DECAY_MAX_TOKENS")
    assert sequence.SPAN_BYTES == limit("CF_DECAY_SPAN_BYTES")
    assert sequence.CHUNK == limit("CF_DECAY_CHUNK")
    assert sequence.MAX_TOKEN_STRIDE == limit("CF_DECAY_MAX_TOKEN_STRIDE")
    assert sequence.MAX_AXES == limit("CF_ROTARY_MAX_AXES")


def _fields(cname):
    body = re.search(r"typedef struct " + cname + r" \{(.*?)\} " + cname + ";", HEADER,
                     re.S).group(1)
    return [re.findall(r"\w+", part)[-1] for line in body.split(";") if line.strip()
            for part in line.split(",")]


def _block(cname, block, **fields):
    """A block whose every field is 1 (a pointer that is never read) or as given."""
    names = _fields(cname)
    assert set(fields) <= set(names)
    values = [fields.get(n, 1.0 if n in ("scale", "eps") else 1) for n in names]
    pointers = block[0].size // 8
    return block[0].pack(*values[:pointers]) + block[1].pack(*values[pointers:])


def test_c_entries_refuse():
    L = _hip.lib()
    for fn in (L.cf_decay_attention, L.cf_decay_attention_step, L.cf_rotary):
        assert fn(None) == INVALID

    def attention(**f):
        return L.cf_decay_attention(_block("CfDecayAttentionArgs", _hip.DECAY_ATTENTION_ARGS,
                                           **f))
    for bad in (dict(seqs=-1), dict(seqs=65536), dict(tokens=-1), dict(heads=0), dict(kv_heads=0),
                dict(heads=3, kv_heads=2), dict(heads=4097), dict(dk=0), dict(dk=257), dict(dv=0),
                dict(dv=1025), dict(dtype=3), dict(dtype=-1), dict(q=0), dict(v=0), dict(out=0),
                dict(log_decay=0), dict(segment=100), dict(segment=-64), dict(q_token=-1),
                dict(out_token=8000001), dict(segment=64, tokens=65, workspace=0),
                # 65 tokens of a packed sequence in segments of 64: up to two states of 1 x 1
                dict(segment=64, tokens=65, workspace=64, workspace_bytes=2 * 52 - 1),
                dict(segment=64, tokens=65, workspace=8, workspace_bytes=2 * 52)):
        assert attention(**dict(dict(segment=0), **bad)) == INVALID, bad
    assert attention(seqs=0, segment=0) == 0          # nothing to do, nothing launched

    def step(**f):
        return L.cf_decay_attention_step(_block("CfDecayStepArgs", _hip.DECAY_STEP_ARGS, **f))
    for bad in (dict(rows=-1), dict(rows=65536), dict(pool=-1), dict(heads=3, kv_heads=2),
                dict(dk=257), dict(dv=1025), dict(dtype=3), dict(state=0), dict(k=0),
                dict(slots=0, rows=2)):
        assert step(**bad) == INVALID, bad
    assert step(rows=0) == 0

    def turn(**f):
        f = dict(dict(d=8, pairs=4), **f)
        return L.cf_rotary(_block("CfRotaryArgs", _hip.ROTARY_ARGS, **f))
    for bad in (dict(d=513), dict(pairs=5), dict(pairs=-1), dict(axes=0), dict(axes=4),
                dict(axes=3, section1=3, section2=2), dict(axes=2, section1=5),
                dict(axes=2, section1=-1), dict(pos_kind=3), dict(dtype=3), dict(x_heads=0),
                dict(k_heads=-1), dict(outer=-1), dict(outer=2 ** 40, inner=2 ** 40),
                dict(eps=-1.0), dict(eps=math.nan), dict(k=0), dict(freqs=0), dict(x=0)):
        assert turn(**bad) == INVALID, bad
    assert turn(outer=0) == 0 and turn(inner=0) == 0


def _attn(**change):
    a = dict(q=torch.zeros(2, 5, 4, 8), k=torch.zeros(2, 5, 2, 8), v=torch.zeros(2, 5, 2, 6),
             log_decay=torch.zeros(4))
    a.update(change)
    return kernels.decay_attention(**a)


@pytest.mark.parametrize("error,match,change", [
    (RuntimeError, "GPU tensor", {}),
    (TypeError, "torch.Tensor", dict(q=None)),
    (TypeError, "q must be", dict(q=torch.zeros(2, 5, 4, 8, dtype=torch.float64))),
    (TypeError, "k must be", dict(k=torch.zeros(2, 5, 2, 8, dtype=torch.float16))),
    (TypeError, "log_decay must be", dict(log_decay=torch.zeros(4, dtype=torch.float64))),
    (ValueError, "contiguous tensor of 4", dict(log_decay=torch.zeros(3))),
    (ValueError, "dimensions", dict(q=torch.zeros(5, 4, 8))),
    (ValueError, "belong together", dict(k=torch.zeros(2, 5, 2, 9))),
    (ValueError, "belong together", dict(v=torch.zeros(2, 4, 2, 6))),
    (ValueError, "query heads", dict(k=torch.zeros(2, 5, 3, 8), v=torch.zeros(2, 5, 3, 6))),
    (ValueError, "head sizes", dict(q=torch.zeros(2, 5, 4, 257), k=torch.zeros(2, 5, 2, 257))),
    (ValueError, "head sizes", dict(v=torch.zeros(2, 5, 2, 0))),
    (ValueError, "last dimension of v",
     dict(v=torch.zeros(2, 5, 6, 2).transpose(2, 3))),
    (TypeError, "state must be", dict(state=torch.zeros(2, 4, 8, 6, dtype=torch.float16))),
    (ValueError, "state must be", dict(state=torch.zeros(2, 4, 6, 8))),
    (ValueError, "state must be", dict(state=torch.zeros(2, 4, 6, 8).transpose(2, 3))),
    (ValueError, "out has shape", dict(out=torch.zeros(2, 5, 4, 8))),
    (TypeError, "out must be", dict(out=torch.zeros(2, 5, 4, 6, dtype=torch.float16))),
    (ValueError, "overlap each other", dict(out=torch.zeros(1, 5, 4, 6).expand(2, 5, 4, 6))),
    (RuntimeError, "gradient", dict(q=torch.zeros(2, 5, 4, 8, requires_grad=True))),
])
def test_attention_refuses(error, match, change):
    with pytest.raises(error, match=match):
        _attn(**change)


def test_attention_refuses_far_tokens():
    q = torch.empty(8000009).as_strided((1, 2, 1, 8), (0, 8000001, 8, 1))
    with pytest.raises(ValueError, match="elements apart"):
        _attn(q=q, k=torch.zeros(1, 2, 1, 8), v=torch.zeros(1, 2, 1, 6), log_decay=torch.zeros(1))


def test_attention_refuses_packed():
    p = dict(q=torch.zeros(10, 4, 8), k=torch.zeros(10, 2, 8), v=torch.zeros(10, 2, 6))
    cu = torch.tensor([0, 4, 10], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        _attn(cu_seqlens=cu, **p)
    with pytest.raises(ValueError, match="dimensions"):
        _attn(cu_seqlens=cu)
    for bad in (cu[:0], cu[None], 3):
        with pytest.raises(ValueError, match="cu_seqlens must be"):
            _attn(cu_seqlens=bad, **p)
    with pytest.raises(TypeError, match="cu_seqlens must be"):
        _attn(cu_seqlens=cu.float(), **p)
    with pytest.raises(ValueError, match="contiguous tensor of 2"):
        _attn(cu_seqlens=torch.zeros(4, dtype=torch.int32)[::2], **p)
    with pytest.raises(ValueError, match="state must be"):
        _attn(cu_seqlens=cu, state=torch.zeros(3, 4, 8, 6), **p)
    with pytest.raises(ValueError, match="overlaps"):
        _attn(cu_seqlens=cu, q=p["q"][..., :6], k=p["k"][..., :6], v=p["v"],
              out=p["q"][..., :6])


def test_gradients_pass_under_no_grad():
    with torch.no_grad(), pytest.raises(RuntimeError, match="GPU tensor"):
        _attn(q=torch.zeros(2, 5, 4, 8, requires_grad=True))


def _step(**change):
    a = dict(q=torch.zeros(3, 4, 8), k=torch.zeros(3, 2, 8), v=torch.zeros(3, 2, 6),
             log_decay=torch.zeros(4), state=torch.zeros(3, 4, 8, 6))
    a.update(change)
    return kernels.decay_attention_step(**a)


@pytest.mark.parametrize("error,match,change", [
    (RuntimeError, "GPU tensor", {}),
    (RuntimeError, "GPU tensor", dict(state=torch.zeros(9, 5, 4, 8, 6)[:3, 1])),
    (ValueError, "dimensions", dict(q=torch.zeros(1, 3, 4, 8))),
    (ValueError, "slots are needed", dict(state=torch.zeros(4, 4, 8, 6))),
    (ValueError, "each slot contiguous", dict(state=torch.zeros(3, 4, 6, 8).transpose(2, 3))),
    (ValueError, "state must be", dict(state=torch.zeros(3, 4, 8, 5))),
    (ValueError, "overlap each other", dict(state=torch.zeros(1, 4, 8, 6).expand(3, 4, 8, 6))),
    (TypeError, "state must be", dict(state=torch.zeros(3, 4, 8, 6, dtype=torch.bfloat16))),
    (TypeError, "slots must be", dict(slots=torch.zeros(3))),
    (ValueError, "contiguous tensor of 3", dict(slots=torch.zeros(4, dtype=torch.int32))),
    (RuntimeError, "gradient", dict(state=torch.zeros(3, 4, 8, 6, requires_grad=True))),
])
def test_step_refuses(error, match, change):
    with pytest.raises(error, match=match):
        _step(**change)


def _turn(**change):
    a = dict(x=torch.zeros(5, 2, 8), positions=torch.arange(5), freqs=kernels.rotary_freqs(4))
    a.update(change)
    return kernels.rotary(**a)


@pytest.mark.parametrize("error,match,change", [
    (RuntimeError, "GPU tensor", {}),
    (RuntimeError, "GPU tensor", dict(positions=torch.zeros(2, 5), sections=(1, 3))),
    (TypeError, "x must be", dict(x=torch.zeros(5, 2, 8, dtype=torch.int32))),
    (ValueError, "tokens.., heads, d", dict(x=torch.zeros(5, 8))),
    (TypeError, "freqs must be", dict(freqs=torch.zeros(4))),
    (ValueError, "pairs in heads", dict(freqs=kernels.rotary_freqs(5))),
    (ValueError, "pairs in heads", dict(freqs=kernels.rotary_freqs(0))),
    (ValueError, "pairs in heads", dict(x=torch.zeros(5, 2, 514))),
    (ValueError, "sections", dict(sections=(1, 2))),
    (ValueError, "sections", dict(sections=(1, 1, 1, 1))),
    (ValueError, "sections", dict(sections=(5, -1))),
    (TypeError, "positions must be", dict(positions=torch.zeros(5, dtype=torch.float64))),
    (ValueError, "do not fit", dict(positions=torch.arange(4))),
    (ValueError, "do not fit", dict(positions=torch.zeros(3, 5), sections=(1, 3))),
    (ValueError, "positions must be", dict(positions=torch.zeros(1, 1, 5))),
    (ValueError, "last dimension", dict(x=torch.zeros(5, 8, 2).transpose(1, 2))),
    (RuntimeError, "gradient", dict(x=torch.zeros(5, 2, 8, requires_grad=True))),
])
def test_rotary_refuses(error, match, change):
    with pytest.raises(error, match=match):
        _turn(**change)


def test_rotary_in_place_and_overlaps():
    """In place is an output; another view of the input is refused, and heads
    that lie beside each other in fused rows are told apart from it."""
    buf = torch.zeros(6, 2, 8)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        _turn(x=buf[:5], out=buf[:5])
    with pytest.raises(ValueError, match="overlaps"):
        _turn(x=buf[:5], out=buf[1:])
    rows = torch.zeros(5, 40)
    q, k = rows[:, :16].unflatten(1, (2, 8)), rows[:, 16:24].unflatten(1, (1, 8))
    args = (torch.arange(5), kernels.rotary_freqs(4))
    with pytest.raises(RuntimeError, match="GPU tensor"):
        kernels.qk_norm_rotary(q, k, *args, out=(q, k))
    with pytest.raises(ValueError, match="overlaps"):
        kernels.qk_norm_rotary(q, k, *args, out=(rows[:, 8:24].unflatten(1, (2, 8)), None))
    with pytest.raises(ValueError, match="overlaps"):
        kernels.qk_norm_rotary(q, k, *args, out=(rows[:, 24:].unflatten(1, (2, 8)),
                                                 rows[:, 32:].unflatten(1, (1, 8))))
    with pytest.raises(ValueError, match="overlaps"):      # one tensor as both, one in place
        kernels.qk_norm_rotary(q, q, *args, out=(q, None))
    with pytest.raises(ValueError, match="overlaps"):
        kernels.qk_norm_rotary(k, k, *args, out=(k, k))
    with pytest.raises(ValueError, match="two strides"):
        _turn(x=torch.zeros(2, 2, 2, 2, 8).transpose(0, 2), positions=torch.zeros(2, 2, 2))


@pytest.mark.parametrize("error,match,change", [
    (TypeError, "k must be", dict(k=None)),
    (ValueError, "belong together", dict(k=torch.zeros(5, 2, 6))),
    (ValueError, "contiguous \\[8\\]", dict(q_weight=torch.ones(7))),
    (TypeError, "k_weight must be", dict(k_weight=torch.ones(8, dtype=torch.float16))),
    (ValueError, "negative", dict(eps=-1e-6)),
    (ValueError, "pair", dict(out=(None,))),
])
def test_qk_norm_rotary_refuses(error, match, change):
    a = dict(q=torch.zeros(5, 4, 8), k=torch.zeros(5, 2, 8), positions=torch.arange(5),
             freqs=kernels.rotary_freqs(4))
    a.update(change)
    with pytest.raises(error, match=match):
        kernels.qk_norm_rotary(**a)


def test_rotary_freqs():
    f = kernels.rotary_freqs(4, base=16.0)
    assert f.dtype == torch.float64 and f.tolist() == [1.0, 0.5, 0.25, 0.125]
    f = kernels.rotary_freqs(6, base=16.0, sections=(2, 4))
    assert f.tolist() == [1.0, 0.25, 1.0, 0.5, 0.25, 0.125]
    with pytest.raises(ValueError, match="do not make"):
        kernels.rotary_freqs(6, sections=(2, 3))


def test_token_dimensions_reduce_to_two_strides():
    s = sequence._split_tokens
    assert s((7,), [(80,)]) == (1, 7, [(0, 80)])
    assert s((3, 7), [(70, 10), (7, 1)]) == (1, 21, [(0, 10), (0, 1)])
    assert s((3, 7), [(70, 10), (0, 1)]) == (3, 7, [(70, 10), (0, 1)])       # broadcast
    assert s((1, 7, 1), [(5, 3, 9)]) == (1, 7, [(0, 3)])
    with pytest.raises(ValueError, match="two strides"):
        s((2, 3, 4), [(1, 100, 7)])


def _calls():
    """One call of each operator that takes real values, by its inputs' names."""
    q, k, v = torch.zeros(1, 3, 4, 8), torch.zeros(1, 3, 2, 8), torch.zeros(1, 3, 2, 6)
    beta, f, state = torch.zeros(1, 3, 4), torch.zeros(1, 3, 4), torch.zeros(1, 4, 8, 6)
    pos, freqs, w = torch.arange(3), kernels.rotary_freqs(4), torch.zeros(6, 8)
    return [
        (kernels.decay_attention, dict(q=q, k=k, v=v, log_decay=torch.zeros(4), state=state)),
        (kernels.decay_attention_step, dict(q=q[0], k=k[0], v=v[0], log_decay=torch.zeros(4),
                                            state=torch.zeros(3, 4, 8, 6))),
        (kernels.rotary, dict(x=q[0], positions=pos, freqs=freqs)),
        (kernels.qk_norm_rotary, dict(q=q[0], k=k[0], positions=pos, freqs=freqs,
                                      q_weight=torch.ones(8))),
        (kernels.delta_attention, dict(q=q, k=k, v=v, beta=beta, log_decay=f, state=state)),
        (kernels.delta_attention_step, dict(q=q[0], k=k[0], v=v[0], beta=beta[0], log_decay=f[0],
                                            state=torch.zeros(3, 4, 8, 6))),
        (kernels.linear, dict(x=q, w=w, bias=torch.zeros(6), residual=torch.zeros(1, 3, 4, 6))),
        (kernels.gated_linear, dict(x=q, w_gate=w, w_up=w + 1, bias_gate=torch.zeros(6)))]


@pytest.mark.parametrize("i", range(8))
def test_tangents_are_refused(i):
    """By every input of every operator, also after a call of the same shapes that
    passed the checks, and where no gradients are recorded."""
    from torch.autograd import forward_ad
    call, inputs = _calls()[i]
    with pytest.raises(RuntimeError, match="GPU tensor"):
        call(**inputs)
    with forward_ad.dual_level(), torch.no_grad():
        for name, t in inputs.items():
            if t.is_floating_point():
                dual = forward_ad.make_dual(t.clone(), torch.ones_like(t))
                with pytest.raises(RuntimeError, match="tangent"):
                    call(**dict(inputs, **{name: dual}))
                plain = forward_ad.unpack_dual(dual).primal
                with pytest.raises(RuntimeError, match="GPU tensor"):
                    call(**dict(inputs, **{name: plain}))
    with pytest.raises(RuntimeError, match="GPU tensor"):
        call(**inputs)
