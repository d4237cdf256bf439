"""The selective scan and its gradients against float64, element by element, over sequences that are cut into chunks and such that are not.

u = 2^-24 is half a step of float32.  Every result is a sum of products of non-negative magnitudes times signs; its error is at most what the
sum of the magnitudes grows by when every factor grows by its own relative error (1 + k u).  `magnitudes` forms those sums, forward and
backward, in float64, plain and grown; the difference is the bound.  The k, with raw = delta + bias, 4 u |raw| + 14 u the time step's own error
(a rounded sum in its exponential: u |raw| at slope at most 1 relative to softplus, 2 u |raw| for the rounded log2(e), and the function's own
operations):
  decay exp(dt A)       its argument z = dt |A| is off by (time step) + 30: rounded A log2(e), the product, and where a chunk's decay is formed
                        from the sum of its time steps, up to 16 of them added in a row by each of 4 waves plus 4; 4 more for exponential and FMA
  input dt u B          (time step) + 4
  sums over N states    N + 4 (four or eight waves' parts joined)
  gate z sigmoid(z)     2 |z| + 10; its slope and softplus' slope 3 |.| + 12, of a magnitude below 1.1
  sums over channels    D + 6;  sums over all steps  B T + 6
A result is rounded once to its type."""
import pytest
import torch

from oracle import sequence_ref as ref

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
NAMES = ("u", "delta", "A", "B", "C", "D", "z", "bias", "state")

CASES = [  # B, T, D, N, G, lengths, resets, state, z, D, bias
    (1, 1, 3, 4, 1, None, 0.0, True, True, True, True),
    (2, 9, 65, 16, 1, [9, 0], 0.1, True, True, True, True),
    (3, 24, 40, 13, 2, None, 0.1, True, True, True, True),
    (5, 33, 130, 16, 1, [33, 0, 7, 32, 17], 0.0, True, False, True, False),
    (2, 40, 36, 32, 3, None, 0.05, False, True, False, True),
    # cut into chunks
    (1, 300, 20, 16, 1, None, 0.0, True, True, True, True),
    (3, 200, 12, 8, 2, [200, 64, 0], 0.0, True, True, True, True),
    (2, 260, 9, 3, 1, [129, 260], 0.01, True, True, True, True),
    (1, 257, 8, 32, 1, None, 0.02, True, True, True, True),
    (4, 700, 40, 16, 1, [700, 0, 5, 333], 0.0, True, True, True, True),
    (3, 515, 70, 13, 1, [16, 515, 257], 0.004, True, True, True, True),
    (1, 1100, 5, 16, 1, None, 0.0, False, False, False, True),
]


def inputs(case, dtype):
    B, T, D, N, G, lengths, p, with_state, with_z, with_d, with_bias = case
    g = torch.Generator().manual_seed(B * T + D)

    def r(*s):
        return torch.randn(*s, generator=g)

    # time steps of about 0.01 to 0.1 and decays that let a state live over a chunk's border
    t = dict(u=r(B, T, D).to(dtype), delta=(0.5 * r(B, T, D) - (0.0 if with_bias else 3.5)).to(dtype), A=-torch.rand(D, N, generator=g) * 2 - 0.05,
             B=r(B, T, G, N).to(dtype), C=r(B, T, G, N).to(dtype), D=r(D) if with_d else None, z=r(B, T, D).to(dtype) if with_z else None,
             bias=0.5 * r(D) - 3.5 if with_bias else None, state=r(B, D, N) if with_state else None)
    resets = torch.rand(B, T, generator=g) < p if p else None
    ln = None if lengths is None else torch.tensor(lengths, dtype=torch.int32)
    return t, ln, resets, r(B, T, D).to(dtype), r(B, D, N)


def reference(t, ln, resets, dy, dlast, cut=None):
    """cut: a step before which the state is lost (a mistake, to see that it is noticed)."""
    lv = [None if t[k] is None else t[k].double().requires_grad_() for k in NAMES]
    if cut is not None:
        resets = torch.zeros(dy.shape[:2], dtype=torch.bool) if resets is None else resets.clone()
        resets[:, cut] = True
    out, last = ref.selective_scan(*lv, lengths=ln, resets=resets)
    live = [v for v in lv if v is not None]
    g = iter(torch.autograd.grad([out, last], live, [dy.double(), dlast.double()], allow_unused=True))
    return {"out": out.detach(), "last": last.detach()} | {k: torch.zeros_like(v) if (w := next(g)) is None else w for k, v in zip(NAMES, lv) if v is not None}


def magnitudes(t, ln, resets, dy, dlast, grown):
    """The sums of the terms' magnitudes; grown: with every factor a little larger."""
    k = U if grown else 0.0
    B, T, D = dy.shape
    N, G = t["A"].shape[1], t["B"].shape[2]
    f = {n: None if v is None else v.double() for n, v in t.items()}
    raw = f["delta"] + (0.0 if f["bias"] is None else f["bias"])
    dt, slope = torch.nn.functional.softplus(raw, threshold=1e3), torch.sigmoid(raw) * (1 + k * (3 * raw.abs() + 12))
    step = 4 * raw.abs() + 14                                             # the time step's relative error, in u
    A = f["A"].abs()
    arg = dt[..., None] * A
    decay = torch.exp(-arg) * (1 + k * (arg * (step[..., None] + 30) + 4))
    dts = dt * (1 + k * (step + 4))
    u, dyv = f["u"].abs(), dy.double().abs()
    Bm, C = (f[n].abs().repeat_interleave(D // G, 2) for n in ("B", "C"))
    skip = torch.zeros(D, dtype=torch.float64) if f["D"] is None else f["D"].abs()
    on = torch.ones(B, T, dtype=torch.bool) if ln is None else torch.arange(T) < ln[:, None]
    cut = torch.zeros(B, T, dtype=torch.bool) if resets is None else resets
    z = None if f["z"] is None else f["z"]
    gate = torch.ones(()) if z is None else z.abs() * torch.sigmoid(z) * (1 + k * (2 * z.abs() + 10))
    h = torch.zeros(B, D, N, dtype=torch.float64) if f["state"] is None else f["state"].abs()
    hs, before, ys = [], [], []
    for s in range(T):
        live = on[:, s, None, None]
        prev = torch.where(cut[:, s, None, None], 0.0, h)
        new = decay[:, s] * prev + (dts[:, s] * u[:, s])[..., None] * Bm[:, s] * (1 + 2 * k)
        before.append(prev)
        h = torch.where(live, new, h)
        hs.append(h)
        ys.append((h * C[:, s]).sum(-1) * (1 + k * (N + 4)) + skip * u[:, s] * (1 + 3 * k))
    y = torch.stack(ys, 1)
    o = {"out": torch.where(on[..., None], y * gate * (1 + 2 * k), 0.0), "last": h}
    dyv = torch.where(on[..., None], dyv, 0.0)
    dp = dyv * gate
    du, ddt, dA = torch.zeros_like(u), torch.zeros_like(u), torch.zeros_like(A)
    dB, dC = torch.zeros(B, T, G, N, dtype=torch.float64), torch.zeros(B, T, G, N, dtype=torch.float64)
    carry = dlast.double().abs()
    for s in reversed(range(T)):
        live = on[:, s, None, None]
        g = (C[:, s] * dp[:, s, :, None] + carry) * (1 + 2 * k)
        g = torch.where(live, g, 0.0)
        q = g * decay[:, s] * before[s] * (1 + 2 * k)
        s1 = (g * Bm[:, s]).sum(-1) * (1 + k * (N + 4))
        du[:, s] = dts[:, s] * s1 * (1 + 2 * k) + skip * dp[:, s] * (1 + 2 * k)
        ddt[:, s] = u[:, s] * s1 * (1 + 2 * k) + (q * A).sum(-1) * (1 + k * (N + 10))
        dA += (q * dts[:, s, :, None]).sum(0)
        dB[:, s] = (g * (dts[:, s] * u[:, s])[..., None]).unflatten(1, (G, D // G)).sum(2) * (1 + k * (D + 6))
        dC[:, s] = (dp[:, s, :, None] * torch.where(live, hs[s], 0.0)).unflatten(1, (G, D // G)).sum(2) * (1 + k * (D + 6))
        carry = torch.where(live, torch.where(cut[:, s, None, None], 0.0, decay[:, s] * g), carry)
    every = 1 + k * (B * T + 6)
    draw = ddt * slope
    o |= {"u": du, "delta": draw, "A": dA * every, "B": dB, "C": dC, "D": (dp * u).sum((0, 1)) * every, "bias": draw.sum((0, 1)) * every, "state": carry}
    if z is not None:
        sz = torch.sigmoid(z)
        o["z"] = dyv * y * (sz * (1 + z * (1 - sz))).abs() * (1 + 2 * k) + dyv * y * k * (3 * z.abs() + 12) * 1.1
    return o


def bounds(*data):
    plain, grown = magnitudes(*data, False), magnitudes(*data, True)
    return {n: grown[n] - plain[n] for n in grown}


def room_of(room, want, dtype):
    half = U if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    return room * (1 + half) + half * want.abs() + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c[:5])))
def test_selective_scan_and_gradients_element_by_element(case, dtype):
    from airgym_amd.lib.network.selective_scan import selective_scan
    data = inputs(case, DTYPES[dtype])
    t, ln, resets, dy, dlast = data
    want, room = reference(*data), bounds(*data)
    dev = {k: None if v is None else v.cuda().requires_grad_() for k, v in t.items()}
    out, last = selective_scan(*(dev[k] for k in NAMES[:-1]), initial_state=dev["state"], lengths=None if ln is None else ln.cuda(),
                               resets=None if resets is None else resets.cuda(), return_state=True)
    live = [k for k in NAMES if dev[k] is not None]
    got = dict(zip(live, torch.autograd.grad([out, last], [dev[k] for k in live], [dy.cuda(), dlast.cuda()])))
    got |= {"out": out.detach(), "last": last.detach()}
    for k, v in got.items():
        assert torch.isfinite(v).all(), k
        r = room_of(room[k], want[k], v.dtype)
        off = (v.double().cpu() - want[k]).abs()
        bad = off > r
        assert not bad.any(), f"{k}: {int(bad.sum())} of {bad.numel()} off, worst {float((off / r).max()):.3g} times the bound"
        some = want[k] != 0
        if some.sum() > 50:             # zeros in its place would be noticed
            assert float((want[k].abs() > r)[some].double().mean()) > 0.95, k
    if case[1] > 128 and dtype == "f32":
        # ... and so would a state or a gradient that does not come over a chunk's border
        lost = reference(*data, cut=64)
        for k in ("out", "A", "delta", "u", "B", "C"):
            gone = (lost[k] - want[k]).abs()
            assert bool((gone > room_of(room[k], want[k], got[k].dtype)).any()), k
