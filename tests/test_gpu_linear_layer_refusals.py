"""moe_experts refuses a call as a whole: what one of its operators would refuse is refused before the first of them runs."""
import pytest
import torch

from unimonomoe_b200 import linear, moe_experts

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn
TOKENS, HIDDEN, INTER, EXPERTS, TOP = 3, 256, 128, 4, 2


def arguments():
    def zeros(*shape, dtype=torch.bfloat16):
        return torch.zeros(shape, dtype=dtype, device="cuda")
    return dict(x=zeros(TOKENS, HIDDEN), ids=zeros(TOKENS, TOP, dtype=torch.int32), weights=zeros(TOKENS, TOP, dtype=torch.float32),
                w13=zeros(EXPERTS, 2 * INTER, HIDDEN, dtype=E4M3), w13_scale=zeros(EXPERTS, 2, 2, dtype=torch.float32),
                w2=zeros(EXPERTS, HIDDEN, INTER, dtype=E4M3), w2_scale=zeros(EXPERTS, 2, 1, dtype=torch.float32), residual=zeros(TOKENS, HIDDEN))


WRONG = {
    "x: type": ("x", lambda t: t.float()),
    "x: 8 bits": ("x", lambda t: t.to(E4M3)),
    "x: dimensions": ("x", lambda t: t[None]),
    "x: columns": ("x", lambda t: t[:, :128]),
    "x: tokens": ("x", lambda t: t[:2]),
    "x: on the CPU": ("x", lambda t: t.cpu()),
    "ids: type": ("ids", lambda t: t.float()),
    "ids: dimensions": ("ids", lambda t: t[0]),
    "ids: on the CPU": ("ids", lambda t: t.cpu()),
    "ids: one column more": ("ids", lambda t: t[:, [0, 1, 1]]),
    "weights: type": ("weights", lambda t: t.to(torch.bfloat16)),
    "weights: columns": ("weights", lambda t: t[:, :1]),
    "weights: on the CPU": ("weights", lambda t: t.cpu()),
    "w13: type": ("w13", lambda t: t.to(torch.bfloat16)),
    "w13: dense": ("w13", lambda t: t[0]),
    "w13: halves": ("w13", lambda t: t[:, :128].contiguous()),
    "w13: half as wide": ("w13", lambda t: t[:, :, :128].contiguous()),
    "w13: strides": ("w13", lambda t: t[:, :, ::1].transpose(1, 2)),
    "w13: scales": ("w13_scale", lambda t: t[:, :1]),
    "w13: type of scales": ("w13_scale", lambda t: t.half()),
    "w2: experts": ("w2", lambda t: t[:3]),
    "w2: rows": ("w2", lambda t: t[:, :128].contiguous()),
    "w2: columns": ("w2", lambda t: torch.cat([t, t], 2)),
    "w2: type": ("w2", lambda t: t.view(torch.float8_e5m2)),
    "w2: scales": ("w2_scale", lambda t: t[:3]),
    "residual: type": ("residual", lambda t: t.float()),
    "residual: tokens": ("residual", lambda t: t[:2]),
    "residual: on the CPU": ("residual", lambda t: t.cpu()),
}


@pytest.mark.parametrize("wrong", WRONG)
def test_nothing_runs_of_a_layer_that_is_refused(linear_lib, monkeypatch, wrong):
    ran, module = [], linear._load()

    class Watched:
        def __getattr__(self, name):
            if name in ("plan", "quantize", "linear", "experts", "combine"):
                ran.append(name)
            return getattr(module, name)

    monkeypatch.setattr(linear, "_C", Watched())
    a = arguments()
    assert moe_experts(**a).shape == (TOKENS, HIDDEN) and ran == ["plan", "quantize", "experts", "experts", "combine"]
    ran.clear()
    name, change = WRONG[wrong]
    with pytest.raises(ValueError) as e:
        moe_experts(**{**a, name: change(a[name])})
    assert str(e.value) and not ran
    linear.check_status()


def test_what_is_no_tensor(linear_lib):
    a = arguments()
    for name in ("x", "ids", "weights", "w13", "w2_scale"):
        with pytest.raises(TypeError):
            moe_experts(**{**a, name: [1.0]})
