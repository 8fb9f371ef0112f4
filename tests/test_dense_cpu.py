"""The dense products' argument block and refusals, without a GPU: what is wrong
with a call is said before the device is asked for."""
import itertools
import os
import re

import pytest
import torch

from catfuse_amd import _hip, dense, kernels

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = open(os.path.join(ROOT, "include", "catfuse_amd.h")).read()
BODY = re.search(r"typedef struct CfLinearArgs \{(.*?)\} CfLinearArgs;", HEADER, re.S).group(1)
INVALID = 1


def test_block_mirrors_the_header():
    kinds = ""
    for line in BODY.split(";"):
        if line.strip():
            kinds += ("Q" if "*" in line else "q") * (line.count(",") + 1)
    want = "".join(f"{n}{c}" for c, n in ((c, len(list(g))) for c, g in itertools.groupby(kinds)))
    assert _hip.LINEAR_ARGS[0].format + _hip.LINEAR_ARGS[1].format[1:] == "=" + want


def test_limits_mirror_the_header():
    def limit(name):
        return int(re.search(rf"#define {name} (\d+)", HEADER).group(1))
    assert dense.MAX_ROWS == limit("CF_LINEAR_MAX_ROWS")
    assert dense.MAX_WIDTH == limit("CF_LINEAR_MAX_WIDTH")
    for name, value in dense.ACTIVATIONS.items():
        assert value == limit(f"CF_ACT_{(name or 'none').upper()}")


def _block(**f):
    names = [re.findall(r"\w+", part)[-1] for line in BODY.split(";") if line.strip()
             for part in line.split(",")]
    assert set(f) <= set(names)
    values = [f.get(n, 0 if n in ("w2", "bias", "bias2", "residual") else 1) for n in names]
    return _hip.LINEAR_ARGS[0].pack(*values[:9]) + _hip.LINEAR_ARGS[1].pack(*values[9:])


def test_c_entries_refuse():
    L = _hip.lib()
    assert L.cf_linear(None) == INVALID and L.cf_linear_workspace(None) == -1
    for bad in (dict(dtype=3), dict(dtype=-1), dict(rows=-1), dict(rows=10 ** 9 + 1), dict(inner=-1),
                dict(inner=16 * 10 ** 6 + 1), dict(cols=0), dict(cols=16 * 10 ** 6 + 1)):
        assert L.cf_linear(_block(**bad)) == INVALID and L.cf_linear_workspace(_block(**bad)) == -1, bad
    for bad in (dict(activation=5), dict(activation=-1), dict(x_row=-1), dict(w_row=-1),
                dict(w2_row=-1), dict(residual_row=-1), dict(out_row=0), dict(cols=2),
                dict(workspace_bytes=-1), dict(x=0), dict(w=0), dict(out=0),
                dict(w2=256, residual=256)):
        assert L.cf_linear(_block(**bad)) == INVALID, bad
    big = dict(rows=64, inner=8192, cols=64, x_row=8192, w_row=8192, out_row=64, dtype=2)
    need = L.cf_linear_workspace(_block(**big))
    assert need > 0 and need % (64 * 64 * 4) == 0
    for bad in (dict(workspace=0, workspace_bytes=need), dict(workspace=256, workspace_bytes=need - 1),
                dict(workspace=8, workspace_bytes=need)):
        assert L.cf_linear(_block(**big, **bad)) == INVALID, bad
    assert L.cf_linear(_block(rows=0)) == 0           # nothing to do, nothing launched


def _linear(**change):
    a = dict(x=torch.zeros(3, 5, 8), w=torch.zeros(6, 8), bias=torch.zeros(6))
    a.update(change)
    return kernels.linear(**a)


@pytest.mark.parametrize("error,match,change", [
    (RuntimeError, "GPU tensor", {}),
    (RuntimeError, "GPU tensor", dict(activation="gelu", residual=torch.zeros(3, 5, 6))),
    (TypeError, "torch.Tensor", dict(x=None)),
    (TypeError, "torch.Tensor", dict(w=None)),
    (TypeError, "x must be", dict(x=torch.zeros(3, 8, dtype=torch.float64))),
    (TypeError, "w must be", dict(w=torch.zeros(6, 8, dtype=torch.float16))),
    (TypeError, "bias must be", dict(bias=torch.zeros(6, dtype=torch.float16))),
    (ValueError, "x must be", dict(x=torch.zeros(()))),
    (ValueError, "does not belong", dict(w=torch.zeros(6, 9))),
    (ValueError, "does not belong", dict(w=torch.zeros(8))),
    (ValueError, "widths", dict(w=torch.zeros(0, 8), bias=None)),
    (ValueError, "bias must be", dict(bias=torch.zeros(7))),
    (ValueError, "bias must be", dict(bias=torch.zeros(12)[::2])),
    (ValueError, "activation", dict(activation="tanh")),
    (ValueError, "activation", dict(activation=1)),
    (ValueError, "residual has shape", dict(residual=torch.zeros(5, 6))),
    (TypeError, "residual must be", dict(residual=torch.zeros(3, 5, 6, dtype=torch.bfloat16))),
    (ValueError, "last dimension of x", dict(x=torch.zeros(3, 8, 5).transpose(1, 2))),
    (ValueError, "last dimension of w", dict(w=torch.zeros(8, 6).t())),
    (ValueError, "evenly apart", dict(x=torch.zeros(5, 3, 8).transpose(0, 1))),
    (ValueError, "out has shape", dict(out=torch.zeros(3, 5, 8))),
    (TypeError, "out must be", dict(out=torch.zeros(3, 5, 6, dtype=torch.float16))),
    (ValueError, "evenly apart", dict(out=torch.zeros(3, 7, 6)[:, :5])),
    (ValueError, "overlap each other", dict(out=torch.zeros(1, 5, 6).expand(3, 5, 6))),
    (RuntimeError, "gradient", dict(x=torch.zeros(3, 5, 8, requires_grad=True))),
    (RuntimeError, "gradient", dict(w=torch.zeros(6, 8, requires_grad=True))),
])
def test_linear_refuses(error, match, change):
    with pytest.raises(error, match=match):
        _linear(**change)


def test_linear_refuses_overlaps():
    x = torch.zeros(5, 8)
    w = torch.zeros(8, 8)
    with pytest.raises(ValueError, match="overlaps"):
        kernels.linear(x, w, out=x)
    with pytest.raises(ValueError, match="overlaps"):
        kernels.linear(torch.zeros(8, 8), w, out=w)
    buf = torch.zeros(60)
    with pytest.raises(ValueError, match="overlaps"):      # not the residual's own rows
        kernels.linear(x, w, residual=buf[:40].view(5, 8), out=buf[4:44].view(5, 8))
    wide = torch.zeros(5, 16)
    with pytest.raises(RuntimeError, match="GPU tensor"):  # columns beside each other
        kernels.linear(wide[:, :8], w, out=wide[:, 8:])
    r = torch.zeros(5, 8)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        kernels.linear(x, w, residual=r, out=r)


@pytest.mark.parametrize("error,match,change", [
    (RuntimeError, "GPU tensor", {}),
    (ValueError, "w_up .* does not belong", dict(w_up=torch.zeros(7, 8))),
    (TypeError, "w_up must be", dict(w_up=torch.zeros(6, 8, dtype=torch.float16))),
    (TypeError, "of one type", dict(x=torch.zeros(3, 8).half(), w_gate=torch.zeros(6, 8).half(),
                                    w_up=torch.zeros(6, 8).half(), bias_gate=torch.zeros(6),
                                    bias_up=torch.zeros(6).half())),
    (ValueError, "bias_up must be", dict(bias_up=torch.zeros(5))),
    (ValueError, "activation", dict(activation="swish")),
    (RuntimeError, "gradient", dict(w_up=torch.zeros(6, 8, requires_grad=True))),
])
def test_gated_linear_refuses(error, match, change):
    a = dict(x=torch.zeros(3, 8), w_gate=torch.zeros(6, 8), w_up=torch.zeros(6, 8))
    a.update(change)
    with pytest.raises(error, match=match):
        kernels.gated_linear(**a)
