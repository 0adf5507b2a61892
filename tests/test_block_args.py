"""What the calls of norms between blocks and 8-bit products refuse, on the host:
arguments are checked before the context is looked at, so that no GPU and no
memory are needed."""
import ctypes

import pytest

from hachiue_amd import sampler as hs

INVALID, UNSUPPORTED = 1, 4
A = 1 << 20           # addresses far from each other
B, C, D, E, F = (A * i for i in (2, 3, 4, 5, 6))


def outcome(rc):
    return rc, hs.lib().hs_last_error().decode()


def norm_call(M=4, cols=64, **kw):
    kw = dict(dict(x=hs.rows(0, A, 64), residual=hs.rows(0, B, 64), sum=hs.rows(0, C, 64),
                   out=hs.rows(30, D, 64)), **kw)
    block = hs.block_norm(M, cols, kw.pop("x"), **kw)
    return outcome(hs.lib().hs_block_norm_device(None, block, None))


def accepted(result):
    """Checked, and stopped at the missing context."""
    assert result[0] == INVALID and "null context" in result[1], result


def refused(result, status, word):
    assert result[0] == status and word in result[1], result


def test_norms_that_are_accepted():
    accepted(norm_call())
    accepted(norm_call(gate=hs.rows(1, E, 0), gate_act=hs.ACT_TANH))
    accepted(norm_call(out=hs.rows(24, D, 64, E)))
    accepted(norm_call(sum=hs.rows(0, B, 64), out=hs.rows(0, A, 64)))        # in place
    accepted(norm_call(x=hs.rows(0, A, 128), out=hs.rows(0, A + 256, 128)))  # beside each other
    accepted(norm_call(M=0, x=hs.rows(0, 0, 0)))
    accepted(norm_call(cols=32768, x=hs.rows(0, A * 64, 32768), residual=None, sum=None, out=hs.rows(0, A * 128, 32768)))


@pytest.mark.parametrize("kw,status,word", [
    (dict(M=-1), INVALID, "-1 x 64"),
    (dict(cols=-2), INVALID, "4 x -2"),
    (dict(cols=32769), UNSUPPORTED, "32769"),
    (dict(M=(1 << 24) + 1), UNSUPPORTED, "2^24"),
    (dict(x=hs.rows(0, 0, 64)), INVALID, "x must not be null"),
    (dict(x=hs.rows(24, A, 64, B)), UNSUPPORTED, "x of type 24"),
    (dict(x=hs.rows(2, A, 64)), UNSUPPORTED, "type 2"),
    (dict(sum=hs.rows(24, C, 64, F)), UNSUPPORTED, "sum of type 24"),
    (dict(residual=hs.rows(24, B, 64, F)), UNSUPPORTED, "residual of type 24"),
    (dict(gate=hs.rows(24, E, 64, F)), UNSUPPORTED, "gate of type 24"),
    (dict(x=hs.rows(0, A, 63)), INVALID, "stride 63"),
    (dict(x=hs.rows(0, A, 0)), INVALID, "stride 0"),
    (dict(out=hs.rows(0, D, -64)), INVALID, "stride -64"),
    (dict(x=hs.rows(0, A, (1 << 36) + 1)), UNSUPPORTED, "2^36"),
    (dict(x=hs.rows(0, A + 2, 64)), INVALID, "aligned"),
    (dict(out=hs.rows(1, D + 1, 64)), INVALID, "aligned"),
    (dict(out=hs.rows(24, D, 64)), INVALID, "scales"),
    (dict(out=hs.rows(24, D, 64, E + 1)), INVALID, "aligned"),
    (dict(out=hs.rows(0, D, 64, E)), INVALID, "scales"),
    (dict(before=hs.norm(3)), UNSUPPORTED, "norm 3"),
    (dict(after=hs.norm(-1)), UNSUPPORTED, "norm -1"),
    (dict(before=hs.norm(1, -1.0)), INVALID, "eps"),
    (dict(before=hs.norm(1, float("nan"))), INVALID, "eps"),
    (dict(before=hs.norm(1, 0.0, E + 2)), INVALID, "aligned"),
    (dict(gate=hs.rows(0, E, 64), gate_act=7), UNSUPPORTED, "activation 7"),
    (dict(gate=hs.rows(0, E, 64), gate_act=-1), UNSUPPORTED, "activation -1"),
    # what overlaps: another row, another type, another stride, another output
    (dict(sum=hs.rows(0, B + 4, 64)), INVALID, "overlaps an input"),
    (dict(sum=hs.rows(30, B, 64)), INVALID, "overlaps an input"),
    (dict(out=hs.rows(0, A, 65)), INVALID, "overlaps an input"),
    (dict(x=hs.rows(0, A, 100), out=hs.rows(0, A + 256 - 4, 100)), INVALID, "overlaps an input"),
    (dict(gate=hs.rows(0, D, 0), out=hs.rows(0, D, 64)), INVALID, "overlaps an input"),
    (dict(sum=hs.rows(0, C, 64), out=hs.rows(0, C, 64)), INVALID, "sum overlaps out"),
    (dict(before=hs.norm(1, 0.0, C)), INVALID, "parameters"),
    (dict(after=hs.norm(2, 0.0, None, D + 8)), INVALID, "parameters"),
    (dict(out=hs.rows(24, D, 64, D + 64)), INVALID, "scales overlap"),
    (dict(out=hs.rows(24, D, 64, A)), INVALID, "scales overlap"),
    (dict(out=hs.rows(24, D, 64, E), before=hs.norm(1, 0.0, E + 8)), INVALID, "scales overlap"),
])
def test_norms_that_are_refused(kw, status, word):
    refused(norm_call(**kw), status, word)


def test_a_missing_norm():
    refused(outcome(hs.lib().hs_block_norm_device(None, None, None)), INVALID, "null norm")


W = hs.weights(24, 100, 64, A, B)


def product_call(M=4, x=hs.rows(24, C, 64, D), w=W, bias=None, y=hs.rows(0, E, 100)):
    return outcome(hs.lib().hs_matmul_int_device(None, M, x, w, bias, y, None))


def gated_call(M=4, x=hs.rows(24, C, 64, D), gate=W, up=hs.weights(24, 100, 64, F, F + 65536), act=1,
               y=hs.rows(0, E, 100)):
    return outcome(hs.lib().hs_gated_int_device(None, M, x, gate, up, act, y, None))


def test_products_that_are_accepted():
    accepted(product_call())
    accepted(product_call(x=hs.rows(1, C + 2, 65), bias=F, y=hs.rows(24, E, 100, D)))
    accepted(product_call(M=0, x=hs.rows(24, 0, 0), y=hs.rows(0, 0, 0)))
    accepted(product_call(w=hs.weights(24, 0, 64, 0), y=hs.rows(0, 0, 0)))
    accepted(product_call(w=hs.weights(24, 10, 65536, A * 16, A * 32), x=hs.rows(24, A * 64, 65536, D)))
    accepted(gated_call())
    accepted(gated_call(up=W))                                   # one weight for both


BAD_WEIGHTS = [
    (hs.weights(0, 100, 64, A), UNSUPPORTED, "type 0"),
    (hs.weights(14, 100, 256, A), UNSUPPORTED, "type 14"),
    (hs.weights(24, -1, 64, A, B), INVALID, "-1 x 64"),
    (hs.weights(24, 100, 0, A, B), INVALID, "100 x 0"),
    (hs.weights(24, 100, 72, A, B), INVALID, "multiple of 16"),
    (hs.weights(24, 100, 65552, A, B), UNSUPPORTED, "65536"),
    (hs.weights(24, (1 << 24) + 1, 64, A, B), UNSUPPORTED, "2^24"),
    (hs.weights(24, 100, 64, A, B, True), UNSUPPORTED, "Hadamard"),
    (hs.weights(24, 100, 64, 0, B), INVALID, "must not be null"),
    (hs.weights(24, 100, 64, A, None), INVALID, "must not be null"),
    (hs.weights(24, 100, 64, A + 8, B), INVALID, "16-byte"),
    (hs.weights(24, 100, 64, A, B + 2), INVALID, "4-byte"),
]


@pytest.mark.parametrize("w,status,word", BAD_WEIGHTS)
def test_weights_that_are_refused(w, status, word):
    refused(product_call(w=w), status, word)
    refused(gated_call(gate=w), status, word)
    refused(gated_call(up=w), status, word)
    if w.type == 24:
        L = hs.lib()
        one = hs.SampleConfigC()
        block = hs.block_norm(2, w.cols, hs.rows(0, C, max(w.cols, 1)), out=hs.rows(0, D * 16, max(w.cols, 1)))
        if 0 < w.cols <= 32768:
            refused(outcome(L.hs_lm_head_norm_sample_device(None, block, w, F, 1 << 25, None, None,
                                                            ctypes.pointer(one), A, B, None)), status, word)


@pytest.mark.parametrize("kw,status,word", [
    (dict(M=-1), INVALID, "M must be"),
    (dict(M=(1 << 20) + 1), UNSUPPORTED, "2^20"),
    (dict(M=1 << 20, w=hs.weights(24, 1 << 17, 64, A, B)), UNSUPPORTED, "2^36"),
    (dict(w=None), INVALID, "null w"),
    (dict(x=None), INVALID, "must not be null"),
    (dict(y=None), INVALID, "must not be null"),
    (dict(x=hs.rows(24, 0, 64, D)), INVALID, "x must not be null"),
    (dict(x=hs.rows(24, C, 64)), INVALID, "scales"),
    (dict(x=hs.rows(24, C, 48, D)), INVALID, "stride 48"),
    (dict(x=hs.rows(24, C, 72, D)), INVALID, "multiple of 16"),
    (dict(x=hs.rows(24, C + 8, 64, D)), INVALID, "16-byte"),
    (dict(x=hs.rows(24, C, (1 << 23) + 16, D)), UNSUPPORTED, "2^23"),
    (dict(x=hs.rows(3, C, 64)), UNSUPPORTED, "type 3"),
    (dict(w=hs.weights(24, 10, 40000, A * 16, A * 32), x=hs.rows(0, A * 64, 40000)), UNSUPPORTED, "32768"),
    (dict(w=hs.weights(24, 32769, 64, A * 16, A * 32), y=hs.rows(24, A * 64, 32769, F)), UNSUPPORTED, "32768"),
    (dict(y=hs.rows(0, E, 99)), INVALID, "stride 99"),
    (dict(y=hs.rows(24, E, 100)), INVALID, "scales"),
    (dict(y=hs.rows(2, E, 100)), UNSUPPORTED, "type 2"),
    (dict(bias=F + 2), INVALID, "bias"),
    (dict(y=hs.rows(0, C, 100)), INVALID, "overlaps"),
    (dict(y=hs.rows(0, A + 16, 100)), INVALID, "overlaps"),
    (dict(y=hs.rows(0, B, 100)), INVALID, "overlaps"),
    (dict(y=hs.rows(0, D, 100)), INVALID, "overlaps"),
    (dict(bias=E + 4), INVALID, "overlaps"),
    (dict(y=hs.rows(24, E, 100, E + 100)), INVALID, "overlaps its scales"),
    (dict(y=hs.rows(24, E, 100, A)), INVALID, "overlaps"),
])
def test_products_that_are_refused(kw, status, word):
    refused(product_call(**kw), status, word)


@pytest.mark.parametrize("kw,status,word", [
    (dict(up=None), INVALID, "null up"),
    (dict(gate=None), INVALID, "null gate"),
    (dict(up=hs.weights(24, 99, 64, F, F + 65536)), INVALID, "99 x 64"),
    (dict(up=hs.weights(24, 100, 80, F, F + 65536)), INVALID, "100 x 80"),
    (dict(act=7), UNSUPPORTED, "activation 7"),
    (dict(act=-1), UNSUPPORTED, "activation -1"),
    (dict(y=hs.rows(0, F + 16, 100)), INVALID, "overlaps"),
])
def test_pairs_that_are_refused(kw, status, word):
    refused(gated_call(**kw), status, word)


def lm_head_call(M=2, cols=64, w=W, out=hs.rows(0, D, 64), logits=F, ldl=100, cfgs=True, u=E, tokens=E + 4096,
                 ids=None, off=None):
    block = hs.block_norm(M, cols, hs.rows(0, C, max(cols, 1)), out=out)
    c = ctypes.pointer(hs.SampleConfigC()) if cfgs else None
    return outcome(hs.lib().hs_lm_head_norm_sample_device(None, block, w, logits, ldl, ids, off, c, u, tokens, None))


def test_lm_heads_behind_a_norm():
    accepted(lm_head_call())
    accepted(lm_head_call(out=hs.rows(24, D, 64, D + 4096)))
    accepted(lm_head_call(w=hs.weights(0, 100, 64, A)))
    accepted(lm_head_call(M=0))


@pytest.mark.parametrize("kw,status,word", [
    (dict(w=None), INVALID, "null weights"),
    (dict(cols=32), INVALID, "32 columns"),
    (dict(M=65536, out=hs.rows(0, A << 8, 64)), UNSUPPORTED, "65535"),
    (dict(out=None), INVALID, "F32 or I8"),
    (dict(out=hs.rows(30, D, 64)), INVALID, "F32 or I8"),
    (dict(out=hs.rows(24, D, 64, D + 4096), w=hs.weights(0, 100, 64, A)), INVALID, "type I8"),
    (dict(out=hs.rows(24, D, 65, D + 4096)), INVALID, "multiple of 16"),
    (dict(w=hs.weights(7, 100, 64, A)), UNSUPPORTED, "weight type 7"),
    (dict(w=hs.weights(0, 100, 64, A + 4)), INVALID, "16-byte"),
    (dict(ldl=99), INVALID, "99"),
    (dict(logits=0), INVALID, "null"),
    (dict(cfgs=False), INVALID, "configs"),
    (dict(u=None), INVALID, "configs"),
    (dict(tokens=None), INVALID, "configs"),
    (dict(ids=A), INVALID, "history"),
    (dict(off=A), INVALID, "history"),
])
def test_lm_heads_behind_a_norm_that_are_refused(kw, status, word):
    refused(lm_head_call(**kw), status, word)
