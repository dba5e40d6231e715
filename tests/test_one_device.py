"""Operands on two devices are refused before anything is launched.  The checks run on the host, so
tensors without memory (meta) beside CPU ones stand for a second GPU's."""
import pytest
import torch

from femtotron_b200.ops.ext import has_native, native

pytestmark = pytest.mark.skipif(not has_native(), reason="the native extension is not built")
BF16 = torch.bfloat16


def t(*shape, dtype=torch.float32, device="cpu"):
    return torch.empty(*shape, dtype=dtype, device=device)


CALLS = {
    "act8.dequantize": (lambda q, s: native().act8_dequantize(q, s, [2, 64], 64, BF16, 64),
                        [t(2, 64, dtype=torch.int8), t(2, 1)]),
    "act8.rms_norm": (lambda x, w: native().act8_rms_norm(x, w, 1e-5, 64), [t(2, 64, dtype=BF16), t(64, dtype=BF16)]),
    "act8.rms_norm_bwd": (lambda dy, q, s, w, r, err: native().act8_rms_norm_bwd(dy, q, s, w, r, 64, err),
                          [t(2, 64, dtype=BF16), t(2, 64, dtype=torch.int8), t(2, 1), t(64, dtype=BF16), t(2),
                           t(1, dtype=torch.int32)]),
    "act8.swiglu_bwd": (lambda dh, q, s: native().act8_swiglu_bwd(dh, q, s, 64),
                        [t(2, 64, dtype=BF16), t(4, 64, dtype=torch.int8), t(4, 1)]),
    "linear_xent": (lambda h, w, lab, err: native().linear_xent_fwd(h, w, lab, 0, -100, 0, True, err),
                    [t(2, 64, dtype=BF16), t(9, 64, dtype=BF16), t(2, dtype=torch.int64), t(1, dtype=torch.int32)]),
    "rotary_qk": (lambda q, k, c, s, pos, err: native().rotary_qk(q, k, c, s, pos, False, False, False, err),
                  [t(1, 2, 3, 8), t(1, 2, 1, 8), t(4, 4), t(4, 4), t(2, dtype=torch.int64), t(1, dtype=torch.int32)]),
}


@pytest.mark.parametrize("op,which", [(op, i) for op, (_, a) in CALLS.items() for i in range(1, len(a))])
def test_an_operand_elsewhere_is_named(op, which):
    call, args = CALLS[op]
    moved = [a.to("meta") if i == which else a for i, a in enumerate(args)]
    want = "one device, got cpu and meta"
    if op == "rotary_qk" and which == 1:
        want = "must agree in batch, tokens, d, dtype and device"
    with pytest.raises((RuntimeError, ValueError), match=want):
        call(*moved)


def test_operands_of_the_loss_backward():
    h, w, lab, err = CALLS["linear_xent"][1]
    vectors = [t(2), t(()), t(())]
    outs = [t(2, 64, dtype=BF16), t(9, 64, dtype=BF16)]
    for which in range(5):
        a = [v.to("meta") if i == which else v for i, v in enumerate(vectors + outs)]
        with pytest.raises(RuntimeError, match="one device, got cpu and meta"):
            native().linear_xent_bwd(h, w, lab, a[0], a[1], a[2], a[3], a[4], False, 0, -100, 1 << 20, err)
