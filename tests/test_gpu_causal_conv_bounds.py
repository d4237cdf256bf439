"""The causal convolution and its gradients against float64, element by element.

u = 2^-24 is half a step of float32.  P = sum |w| |x| + |bias| is what a pre-activation p's terms add up to: W + 1 roundings, p is off by
(W + 2) u P.  y = p sigmoid(p), slope below 1.1: off by 1.1 (W + 2) u P and by its own exponential, sum, reciprocal and product: 8 u (|p| + 1)
|p| sigmoid at most 8 u (1 + P).  dp = dy s (1 + p (1 - s)): the factor's slope is below 1/2 and its own roundings are 14 u of 1.1 (|p| e^-|p| < 1), so dp is
off by E = |dy| u ((W + 2) P / 2 + 16).  Without the activation E = 0.  dx sums W products of w and dp, the state's gradient among them, so
it is off by what the same sums give for |w| and E + (W + 2) u |dp|; dweight sums |x| times that over all B T steps, in any order:
E + (B T + 2) u |dp|.  A result is rounded once to its type."""
import pytest
import torch

from oracle import sequence_ref as ref

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}

CASES = [  # B, T, D, W, silu, lengths, resets
    (1, 1, 1, 2, True, None, 0.0),
    (2, 5, 7, 8, True, [5, 0], 0.0),
    (3, 40, 33, 4, True, None, 0.1),
    (2, 129, 65, 4, True, [129, 70], 0.05),
    (2, 70, 130, 5, False, [70, 33], 0.1),
    (2, 40, 129, 3, True, None, 0.0),
    (1, 300, 24, 6, True, None, 0.02),
    # channels that 16, 8 and 4 bytes do not divide
    (2, 33, 132, 4, True, [33, 20], 0.1),
    (2, 35, 1039, 4, True, None, 0.1),
    (3, 34, 1040, 4, True, [34, 0, 17], 0.0),
    (1, 20, 2047, 8, True, None, 0.1),
    (40, 24, 260, 4, True, None, 0.05),
]


def inputs(case, dtype):
    B, T, D, W, silu, lengths, p = case
    g = torch.Generator().manual_seed(B * T + D)

    def r(*s):
        return torch.randn(*s, generator=g)

    x, dy = r(B, T, D).to(dtype), r(B, T, D).to(dtype)
    resets = torch.rand(B, T, generator=g) < p if p else None
    ln = None if lengths is None else torch.tensor(lengths, dtype=torch.int32)
    return x, r(D, W) / W ** 0.5, r(D) * 0.1, r(B, W - 1, D).to(dtype), ln, resets, dy, r(B, W - 1, D).to(dtype)


def reference(x, w, b, s, ln, resets, dy, dlast, silu):
    lv = [t.double().requires_grad_() for t in (x, w, b, s)]
    y, last = ref.causal_conv(*lv, silu, ln, resets)
    return y.detach(), torch.autograd.grad([y, last], lv, [dy.double(), dlast.double()])


def bounds(x, w, b, s, ln, resets, dy, dlast, silu):
    """What y, dx, dweight, dbias and dstate may be off by in float32."""
    B, T, D = x.shape
    W = w.shape[1]
    ax, aw, ab, as_, ady, adl = (t.double().abs() for t in (x, w, b, s, dy, dlast))
    P, _ = ref.causal_conv(ax, aw, ab, as_, False, ln, resets)            # zero behind a sequence's end
    on = torch.ones(B, T, 1, dtype=torch.float64)
    if ln is not None:
        on = (torch.arange(T) < ln[:, None])[..., None].double()
    ady = ady * on
    y = U * (1.1 * (W + 2) * P + 8 * (1 + P) * on) if silu else U * (W + 2) * P
    E = ady * U * ((W + 2) * P / 2 + 16) if silu else 0 * ady
    adp = (1.1 if silu else 1.0) * ady

    def sums(rounds):
        lv = [t.clone().requires_grad_() for t in (ax, aw, ab, as_)]
        out, last = ref.causal_conv(*lv, False, ln, resets)
        return torch.autograd.grad([out, last], lv, [E + rounds * U * adp, rounds * U * adl])

    dx, _, _, ds = sums(W + 3)
    _, dw, db, _ = sums(B * T + 2)
    return y, (dx, dw, db, ds)


def within(name, got, want, room):
    got64 = got.detach().double().cpu()
    half = 0.0 if got.dtype == torch.float32 else torch.finfo(got.dtype).eps / 2
    room = room * (1 + half) + half * want.abs() + torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps / 2 + U * want.abs()
    assert torch.isfinite(got64).all(), name
    off = (got64 - want).abs()
    bad = off > room
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} off, worst {float((off / room).max()):.3g} times the bound"
    return room


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c[:4])))
def test_causal_conv_and_gradients_element_by_element(case, dtype):
    from airgym_amd.lib.network.causal_conv import causal_conv
    data, silu = inputs(case, DTYPES[dtype]), case[4]
    x, w, b, s, ln, resets, dy, dlast = data
    y64, g64 = reference(*data, silu)
    ry, rg = bounds(*data, silu)
    dev = [t.cuda().requires_grad_() for t in (x, w, b, s)]
    y, last = causal_conv(*dev[:3], activation="silu" if silu else None, initial_state=dev[3], lengths=None if ln is None else ln.cuda(),
                          resets=None if resets is None else resets.cuda(), return_state=True)
    got = torch.autograd.grad([y, last], dev, [dy.cuda(), dlast.cuda()])
    within("y", y, y64, ry)
    rooms = [within(n, a, c, r) for n, a, c, r in zip(("dx", "dweight", "dbias", "dstate"), got, g64, rg)]
    # a tap dropped from the sums, a step's gradient lost: beyond the bound wherever there is something to lose
    if case[0] * case[1] > 8:
        fewer = [None if t is None else t.clone() for t in data]
        fewer[6][:, case[1] // 2] = 0
        _, other = reference(*fewer, silu)
        for k in (0, 1, 2):
            gone = (other[k] - g64[k]).abs()
            assert bool((gone > rooms[k]).any())
            if k:
                assert float((gone > rooms[k]).double()[gone > 0].mean()) > 0.8
