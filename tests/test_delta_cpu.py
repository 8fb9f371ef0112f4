"""The delta rule's argument blocks and refusals, without a GPU: what is wrong
with a call is said before the device is asked for."""
import itertools
import math
import os
import re

import pytest
import torch

from catfuse_amd import _hip, delta, kernels

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = open(os.path.join(ROOT, "include", "catfuse_amd.h")).read()
INVALID = 1


def _body(cname):
    return re.search(r"typedef struct " + cname + r" \{(.*?)\} " + cname + ";", HEADER, re.S).group(1)


@pytest.mark.parametrize("cname,block", [("CfDeltaAttentionArgs", _hip.DELTA_ATTENTION_ARGS),
                                         ("CfDeltaStepArgs", _hip.DELTA_STEP_ARGS)])
def test_blocks_mirror_the_header(cname, block):
    kinds = ""
    for line in _body(cname).split(";"):
        if line.strip():
            kind = "Q" if "*" in line else "q" if "int64_t" in line else "d"
            assert kind != "d" or "double" in line
            kinds += kind * (line.count(",") + 1)
    want = "".join(f"{n}{c}" if n > 1 else c
                   for c, n in ((c, len(list(g))) for c, g in itertools.groupby(kinds)))
    assert block[0].format + block[1].format[1:] == "=" + want
    assert block[0].size + block[1].size == 8 * len(kinds)


def _block(cname, block, **fields):
    """A block whose every field is 1 (a pointer that is never read) or as given."""
    names = [re.findall(r"\w+", part)[-1] for line in _body(cname).split(";") if line.strip()
             for part in line.split(",")]
    assert set(fields) <= set(names)
    values = [fields.get(n, 1.0 if n == "scale" else 1) for n in names]
    pointers = block[0].size // 8
    return block[0].pack(*values[:pointers]) + block[1].pack(*values[pointers:])


def _attention(**f):
    return _block("CfDeltaAttentionArgs", _hip.DELTA_ATTENTION_ARGS, **f)


def test_c_entries_refuse():
    L = _hip.lib()
    assert L.cf_delta_attention(None) == INVALID and L.cf_delta_attention_step(None) == INVALID
    assert L.cf_delta_workspace(None) == -1
    for bad in (dict(seqs=-1), dict(seqs=65536), dict(tokens=-1), dict(tokens=2 * 10 ** 9 + 1),
                dict(heads=0), dict(k_heads=0), dict(heads=3, k_heads=2), dict(heads=3, q_heads=2),
                dict(heads=3, v_heads=2), dict(q_heads=2), dict(heads=4097), dict(dk=0), dict(dk=257),
                dict(dv=0), dict(dv=1025), dict(dtype=3), dict(dtype=-1), dict(q=0), dict(k=0),
                dict(v=0), dict(beta=0), dict(out=0), dict(segment=100), dict(segment=-64),
                dict(q_token=-1), dict(out_token=8000001), dict(workspace=0), dict(workspace=128)):
        f = dict(dict(segment=0, workspace=256, workspace_bytes=1 << 40), **bad)
        assert L.cf_delta_attention(_attention(**f)) == INVALID, bad
    need = L.cf_delta_workspace(_attention(segment=0, tokens=65))
    assert L.cf_delta_attention(_attention(segment=0, tokens=65, workspace=256,
                                           workspace_bytes=need - 1)) == INVALID
    # more segments than the launch that joins them takes
    assert L.cf_delta_attention(_attention(segment=64, tokens=64 * 65536, workspace=256,
                                           workspace_bytes=1 << 50)) == INVALID
    assert L.cf_delta_attention(_attention(seqs=0, segment=0)) == 0         # nothing to do, nothing launched
    for bad in (dict(rows=-1), dict(rows=65536), dict(pool=-1), dict(heads=3, k_heads=2),
                dict(heads=3, q_heads=2), dict(heads=3, v_heads=2), dict(dk=257), dict(dv=1025),
                dict(dtype=3), dict(state=0), dict(k=0), dict(beta=0), dict(slots=0, rows=2)):
        assert L.cf_delta_attention_step(_block("CfDeltaStepArgs", _hip.DELTA_STEP_ARGS,
                                                **bad)) == INVALID, bad
    assert L.cf_delta_attention_step(_block("CfDeltaStepArgs", _hip.DELTA_STEP_ARGS, rows=0)) == 0


@pytest.mark.parametrize("dtype,dk", [(0, 128), (1, 32), (2, 64), (2, 128), (2, 65), (2, 256)])
@pytest.mark.parametrize("seqs,tokens,cu", [(1, 1, 0), (3, 200, 0), (5, 1000, 256), (7, 0, 0), (7, 0, 256)])
def test_workspace(dtype, dk, seqs, tokens, cu):
    """T, the sums and betas of every chunk and head; N and M of every segment and
    head; the rows that packed sequences begin at."""
    H, dv, C = 6, 40, 64 if dtype == 2 and 64 < dk <= 128 else 32
    def count(unit):
        return tokens // unit + seqs if cu else seqs * max(1, -(-tokens // unit))
    begins = (8 * (seqs + 1) + 255) // 256 * 256 if cu else 0
    chunks = count(C) * H * ((18432 if C == 64 else 6144) + 12 * C) if tokens else 0
    for segment in (0, 64, 128, 1024):
        own = count(segment) * H * 4 * dk * (dv + dk) if 0 < segment < tokens else 0
        f = dict(dtype=dtype, dk=dk, dv=dv, heads=H, seqs=seqs, tokens=tokens, cu_seqlens=cu,
                 segment=segment)
        assert _hip.lib().cf_delta_workspace(_attention(**f)) == begins + chunks + own


def test_segments_stay_within_limits():
    for seqs, tokens, packed in ((1, 10 ** 9, True), (1, 10 ** 9, False), (65535, 10 ** 9, True),
                                 (3, 100, False), (200, 70000, True)):
        for heads, d in ((1, 32), (32, 128), (1, 256), (4096, 16)):
            s = delta._segment(seqs, tokens, packed, heads, d, d)
            assert s >= 0 and s % 64 == 0
            if s:
                n = tokens // s + seqs if packed else seqs * -(-tokens // s)
                assert s < tokens and n <= delta.MAX_SEGMENTS


def _attn(**change):
    a = dict(q=torch.zeros(2, 5, 4, 8), k=torch.zeros(2, 5, 2, 8), v=torch.zeros(2, 5, 1, 6),
             beta=torch.zeros(2, 5, 4), log_decay=torch.zeros(2, 5, 4))
    a.update(change)
    return kernels.delta_attention(**a)


@pytest.mark.parametrize("error,match,change", [
    (RuntimeError, "GPU tensor", {}),
    (RuntimeError, "GPU tensor", dict(log_decay=None)),
    (TypeError, "torch.Tensor", dict(q=None)),
    (TypeError, "torch.Tensor", dict(beta=None)),
    (TypeError, "q must be", dict(q=torch.zeros(2, 5, 4, 8, dtype=torch.float64))),
    (TypeError, "k must be", dict(k=torch.zeros(2, 5, 2, 8, dtype=torch.float16))),
    (TypeError, "beta must be", dict(beta=torch.zeros(2, 5, 4, dtype=torch.float64))),
    (TypeError, "log_decay must be", dict(log_decay=torch.zeros(2, 5, 4, dtype=torch.bfloat16))),
    (ValueError, "beta must be", dict(beta=torch.zeros(2, 4))),
    (ValueError, "beta must be", dict(beta=torch.zeros(2, 4, 4))),
    (ValueError, "beta's shape", dict(log_decay=torch.zeros(4))),
    (ValueError, "beta's shape", dict(log_decay=torch.zeros(2, 5, 8))),
    (ValueError, "dimensions", dict(q=torch.zeros(5, 4, 8))),
    (ValueError, "belong together", dict(k=torch.zeros(2, 5, 2, 9))),
    (ValueError, "belong together", dict(v=torch.zeros(2, 4, 2, 6))),
    (ValueError, "has to divide", dict(k=torch.zeros(2, 5, 3, 8))),
    (ValueError, "has to divide", dict(v=torch.zeros(2, 5, 8, 6))),
    (ValueError, "has to divide", dict(q=torch.zeros(2, 5, 0, 8))),
    (ValueError, "head sizes", dict(q=torch.zeros(2, 5, 4, 257), k=torch.zeros(2, 5, 2, 257))),
    (ValueError, "head sizes", dict(v=torch.zeros(2, 5, 2, 0))),
    (ValueError, "last dimension of v", dict(v=torch.zeros(2, 5, 6, 2).transpose(2, 3))),
    (TypeError, "state must be", dict(state=torch.zeros(2, 4, 8, 6, dtype=torch.float16))),
    (ValueError, "state must be", dict(state=torch.zeros(2, 4, 6, 8))),
    (ValueError, "state must be", dict(state=torch.zeros(2, 4, 6, 8).transpose(2, 3))),
    (ValueError, "out has shape", dict(out=torch.zeros(2, 5, 4, 8))),
    (TypeError, "out must be", dict(out=torch.zeros(2, 5, 4, 6, dtype=torch.float16))),
    (ValueError, "overlap each other", dict(out=torch.zeros(1, 5, 4, 6).expand(2, 5, 4, 6))),
    (RuntimeError, "gradient", dict(q=torch.zeros(2, 5, 4, 8, requires_grad=True))),
    (RuntimeError, "gradient", dict(beta=torch.zeros(2, 5, 4, requires_grad=True))),
])
def test_attention_refuses(error, match, change):
    with pytest.raises(error, match=match):
        _attn(**change)


def test_attention_refuses_overlaps_and_far_tokens():
    v = torch.zeros(2, 5, 4, 6)
    with pytest.raises(ValueError, match="overlaps the memory"):
        _attn(v=v, out=v)
    q = torch.empty(8000009).as_strided((1, 2, 1, 8), (0, 8000001, 8, 1))
    one = torch.zeros(1, 2, 1)
    with pytest.raises(ValueError, match="elements apart"):
        _attn(q=q, k=torch.zeros(1, 2, 1, 8), v=torch.zeros(1, 2, 1, 6), beta=one, log_decay=one)


def test_attention_refuses_packed():
    p = dict(q=torch.zeros(10, 4, 8), k=torch.zeros(10, 2, 8), v=torch.zeros(10, 2, 6),
             beta=torch.zeros(10, 4), log_decay=torch.zeros(10, 4))
    cu = torch.tensor([0, 4, 10], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        _attn(**p, cu_seqlens=cu)
    for bad, error, match in ((cu.float(), TypeError, "cu_seqlens must be"),
                              (cu[None], ValueError, "one-dimensional"),
                              (cu[:0], ValueError, "one-dimensional"),
                              ([0, 4, 10], ValueError, "one-dimensional"),
                              (cu[::2].as_strided((2,), (2,)), ValueError, "contiguous")):
        with pytest.raises(error, match=match):
            _attn(**p, cu_seqlens=bad)
    with pytest.raises(ValueError, match="dimensions"):
        _attn(cu_seqlens=cu)
    many = torch.zeros(65537, dtype=torch.int32)
    with pytest.raises(ValueError, match="65536 sequences"):
        _attn(**p, cu_seqlens=many)


def _step(**change):
    a = dict(q=torch.zeros(3, 4, 8), k=torch.zeros(3, 2, 8), v=torch.zeros(3, 4, 6),
             beta=torch.zeros(3, 4), log_decay=torch.zeros(3, 4), state=torch.zeros(5, 4, 8, 6),
             slots=torch.zeros(3, dtype=torch.int32))
    a.update(change)
    return kernels.delta_attention_step(**a)


@pytest.mark.parametrize("error,match,change", [
    (RuntimeError, "GPU tensor", {}),
    (RuntimeError, "GPU tensor", dict(log_decay=None)),
    (ValueError, "dimensions", dict(q=torch.zeros(1, 3, 4, 8))),
    (ValueError, "has to divide", dict(k=torch.zeros(3, 3, 8))),
    (ValueError, "beta must be", dict(beta=torch.zeros(4, 4))),
    (TypeError, "state must be", dict(state=torch.zeros(5, 4, 8, 6, dtype=torch.bfloat16))),
    (ValueError, "state must be", dict(state=torch.zeros(5, 4, 6, 8))),
    (ValueError, "state must be", dict(state=torch.zeros(5, 4, 6, 8).transpose(2, 3))),
    (ValueError, "overlap each other", dict(state=torch.zeros(1, 4, 8, 6).expand(5, 4, 8, 6))),
    (ValueError, "slots are needed", dict(slots=None)),
    (ValueError, "slots must be", dict(slots=torch.zeros(4, dtype=torch.int32))),
    (TypeError, "slots must be", dict(slots=torch.zeros(3))),
    (ValueError, "out has shape", dict(out=torch.zeros(3, 4, 8))),
    (RuntimeError, "gradient", dict(state=torch.zeros(5, 4, 8, 6, requires_grad=True))),
])
def test_step_refuses(error, match, change):
    with pytest.raises(error, match=match):
        _step(**change)


def test_step_refuses_overlaps():
    state = torch.zeros(5, 4, 8, 6)
    with pytest.raises(ValueError, match="state overlaps"):
        _step(state=state, v=state.flatten()[:72].view(3, 4, 6))
    with pytest.raises(ValueError, match="out overlaps"):
        _step(state=state, out=state.flatten()[:72].view(3, 4, 6))
    assert math.prod(state.shape) == 960


def test_workspace_refuses():
    """The sizes that a call refuses, and none of its strides."""
    L, fine = _hip.lib(), dict(segment=0, workspace=256, workspace_bytes=1 << 40)
    assert L.cf_delta_workspace(None) == -1
    for bad in (dict(seqs=-1), dict(seqs=65536), dict(tokens=-1), dict(tokens=2 * 10 ** 9 + 1),
                dict(heads=0), dict(heads=-2), dict(heads=4097), dict(q_heads=2), dict(k_heads=0),
                dict(heads=3, v_heads=2), dict(dk=0), dict(dk=257), dict(dv=0), dict(dv=1025),
                dict(dv=2000), dict(dtype=3), dict(dtype=9), dict(dtype=-1), dict(segment=100),
                dict(segment=-64), dict(segment=64, tokens=64 * 65536),
                dict(segment=64, tokens=64 * 65536, cu_seqlens=0)):
        block = _attention(**dict(fine, **bad))
        assert L.cf_delta_workspace(block) == -1, bad
        assert L.cf_delta_attention(block) == INVALID, bad
    assert L.cf_delta_workspace(_attention(**dict(fine, q_token=-1, out_head=-5, scale=0.0))) > 0


@pytest.mark.parametrize("seqs", [16, 31, 63, 64, 1000])
def test_workspace_of_packed_rows(seqs):
    """The rows that packed sequences begin at and the segments before them, two
    64-bit numbers for each and one end."""
    f = dict(dtype=0, dk=32, dv=32, seqs=seqs, cu_seqlens=256, segment=0)
    begins = (16 * (seqs + 1) + 255) // 256 * 256
    assert _hip.lib().cf_delta_workspace(_attention(tokens=0, **f)) == begins
    chunks = (5000 // 32 + seqs) * (6144 + 12 * 32)
    assert _hip.lib().cf_delta_workspace(_attention(tokens=5000, **f)) == begins + chunks


@pytest.mark.parametrize("dtype,dk,a_token", [(2, 128, 300), (2, 64, 204), (0, 128, 204), (1, 256, 204)])
@pytest.mark.parametrize("heads", [1, 32, 4096])
def test_workspace_of_short_sequences(dtype, dk, a_token, heads):
    """At most three times what the tokens take and 1 GiB (or one sequence's), by
    however many sequences; what the tokens take and a chunk for each sequence
    where they have half a chunk on average."""
    C = 64 if a_token == 300 else 32
    def need(**f):
        return _hip.lib().cf_delta_workspace(_attention(dtype=dtype, dk=dk, dv=dk, heads=heads,
                                                        segment=0, **f))
    for seqs in (1, 100, 256, 4096, 65535):
        for mean in (0, 1, 3, C // 2 - 1, C // 2, C, 1000):
            for cu in (0, 256):
                tokens = mean * (seqs if cu else 1) + (5 if cu else 0)
                begins = (16 * (seqs + 1) + 255) // 256 * 256 if cu else 0
                total = tokens if cu else tokens * seqs
                got = need(seqs=seqs, tokens=tokens, cu_seqlens=cu) - begins
                one = a_token * C * heads
                assert 0 <= got <= 3 * a_token * heads * total + max(1 << 30, one) + one
                if mean >= C // 2:
                    assert got == (tokens // C + seqs if cu else seqs * -(-tokens // C)) * one
