"""The policy loss against its formula in float64, element by element.

u = 2^-24 is half a step of float32.  With Y the spread of a row's finite logits (natural units) and at most 130 additions in a row on the
way to a sum (per lane up to 128 elements, or 18 passes of 8 elements and a join of 5 roundings, then 6 + 4 joins):
  x - max, times log2(e) (a rounded constant): 3 roundings of a number up to Y; the exponential 2: a term of the sum is off by (3 Y + 2) u,
  the sum by 130 u more, log2 of it (up to 17 + Y) by 2 ulp and its rest: lse by (3 Y + 2 + 130 + 40) u at most; a log-probability lp, a
  difference of such, by Y u + that; p by its argument's error and the exponential's: 2 (3 Y + 2) + 174 u of itself.
All are below n u, n = 8 Y + 350.  The factors f = -A r + kl (1 - e^d) take lp through an exponential: off by n u of |A| r and kl (e^d + 1) (and
a few u, which n has room for).  A gradient f (delta - p) + ent p (log p + H) is then off by n u of
  mag = (|A| r + kl (e^d + 1)) (p + delta) + ent p (|log p| + H + 1 + Y)        (H: n u of 1 + Y)
times its factor, one rounding to its type (half a step of its value), and half of the type's smallest number."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
E_CLIP, KL, ENT = 0.2, 0.1, 0.01


def formula(logits, actions, old, adv, refl, mask, kl=KL, ent=ENT):
    """-> loss, the six statistics, dloss / dlogits, and what their errors are counted in, all float64."""
    x = logits.double()
    on = torch.ones(x.shape[0], dtype=torch.bool, device=x.device) if mask is None else mask.bool()
    x = torch.where(on[:, None], x, 0.0)
    act, old, adv, refl = (torch.where(on, t, torch.zeros_like(t)) for t in (actions, old, adv, refl))
    logp = torch.log_softmax(x, 1)
    p = logp.exp()
    plogp = torch.where(p > 0, p * logp, 0.0)
    H = -plogp.sum(1)
    lp = logp.gather(1, act[:, None])[:, 0]
    r, d = (lp - old.double()).exp(), refl.double() - lp
    A = adv.double()
    plain, held = -A * r, -A * r.clamp(1 - E_CLIP, 1 + E_CLIP)
    n = max(int(on.sum()), 1)
    f = torch.where(plain >= held, plain, 0.0) - kl * torch.expm1(d)
    delta = torch.zeros_like(x).scatter_(1, act[:, None], 1.0)
    grad = f[:, None] * (delta - p) + ent * (plogp + p * H[:, None])
    finite = torch.where(torch.isfinite(x), x, x.amax(1, keepdim=True))
    Y = float((finite.amax(1) - finite.amin(1)).max())
    fm = torch.where(plain >= held, plain.abs(), 0.0) + kl * (d.exp() + 1)
    mag = fm[:, None] * (p + delta) + ent * (plogp.abs() + p * (H[:, None] + 1 + Y))
    terms = torch.stack((torch.maximum(plain, held), torch.expm1(d) - d, H, r - 1 - (lp - old.double()), ((r - 1).abs() > E_CLIP).double()))
    sizes = torch.stack(((A * r).abs(), d.exp() + 1, 1 + Y + 0 * H, r + 1, 0 * H))
    w = on.double() / n
    stats, size = (terms * w).sum(1), (sizes * w).sum(1)
    loss = stats[0] + kl * stats[1] - ent * stats[2]
    return dict(loss=loss, stats=torch.cat((stats, torch.tensor([float(int(on.sum()))], dtype=torch.float64, device=x.device))), grad=grad * w[:, None],
                mag=mag * w[:, None], size=size, lp=lp, H=H, Y=Y, n=8 * Y + 350, on=on)


def room_of(want, mag, n, dtype, factor=1.0):
    half = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    smallest = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    return n * U * mag * abs(factor) * (1 + half) + half * (want * factor).abs() + smallest


def within(name, got, want, room):
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all(), f"{name}: not finite"
    bad = off > room
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} off, worst {float((off / room).max()):.3g} times the bound"


def rows(R, V, dtype, masked=False, minus_inf=None, seed=0):
    """minus_inf: None, "some", or (first, last): all choices between are unavailable, in every second row."""
    g = torch.Generator("cuda").manual_seed(seed + 7 * R + V)
    logits = (2 * torch.randn(R, V, generator=g, device="cuda")).to(dtype)
    actions = torch.randint(0, V, (R,), generator=g, device="cuda")
    off = torch.zeros(R, V, dtype=torch.bool, device="cuda")
    if minus_inf == "some":
        off = torch.rand(R, V, generator=g, device="cuda") < 0.3
    elif minus_inf is not None:
        off[::2, minus_inf[0]:minus_inf[1]] = True
    off[torch.arange(R), actions] = False
    logits = logits.masked_fill(off, -float("inf"))
    lp = torch.log_softmax(logits.double(), 1).gather(1, actions[:, None])[:, 0]
    moved = 0.2 * torch.randn(R, generator=g, device="cuda").double()
    for border in (1.2, 0.8):           # on the border itself there are two right gradients
        b = torch.tensor(border).double().log().item()
        moved = torch.where((moved - b).abs() < 1e-3, moved + 3e-3, moved)
    old, refl = (lp - moved).float(), (lp + 0.2 * torch.randn(R, generator=g, device="cuda")).float()
    adv = torch.randn(R, generator=g, device="cuda")
    mask = None
    if masked:
        mask = torch.rand(R, generator=g, device="cuda") < 0.6
        mask[0] = True
        mask[1] = False
        logits[~mask], old[~mask], adv[~mask], refl[~mask], actions[~mask] = float("nan"), float("inf"), float("nan"), float("nan"), -100
    return logits, actions, old, adv, refl, mask


def call(logits, actions, old, adv, refl, mask, kl=KL, ent=ENT, factor=None):
    from airgym_amd.lib.core.policy_loss import policy_loss
    leaf = logits.clone().requires_grad_()
    loss, stats = policy_loss(leaf, actions, old, adv, ref_logp=refl, mask=mask, e_clip=E_CLIP, kl_coef=kl, entropy_coef=ent)
    (grad,) = torch.autograd.grad(loss if factor is None else factor * loss, leaf)
    return loss.detach(), stats, grad


# ------------------------------------------------------------------------------------------------ float16
@pytest.mark.parametrize("V", [7, 200, 900, 9001])
@pytest.mark.parametrize("R,f", [(512, 8e4), (4096, 1.2e5)])
@pytest.mark.parametrize("term", ["ratio", "kl"])
@pytest.mark.parametrize("masked", [False, True])
def test_half_precision_rows_whose_factor_is_beyond_the_type(R, f, V, term, masked):
    """A row's factor above 65504 divided by the rows is well inside float16's range."""
    logits, actions, old, adv, refl, mask = rows(R, V, torch.float16, masked)
    lp = torch.log_softmax(logits.double(), 1).nan_to_num().gather(1, actions.clamp(min=0)[:, None])[:, 0]
    big = torch.zeros(R, dtype=torch.bool, device="cuda")
    big[::97] = True
    big &= torch.ones_like(big) if mask is None else mask
    if term == "ratio":
        old = torch.where(big, lp - torch.tensor(f).log().double().item(), old.double()).float()
        adv = torch.where(big, -1.0, adv)
    else:
        refl = torch.where(big, lp + torch.tensor(f / KL).log().double().item(), refl.double()).float()
    for factor in (1.0, 0.3, 2.0 ** -6):
        want = formula(logits, actions, old, adv, refl, mask)
        _, _, grad = call(logits, actions, old, adv, refl, mask, factor=factor)
        within("dlogits", grad, want["grad"] * factor, room_of(want["grad"], want["mag"], want["n"], grad.dtype, factor))
    assert float(want["grad"].abs().max()) > 10.0


@pytest.mark.parametrize("V", [2, 21, 129, 1000])
def test_half_precision_from_the_smallest_to_the_largest_factor(V):
    """Small rows under a loss scale beside large ones: nothing is lost at either end before the factor is known."""
    R = 30000
    logits, actions, old, adv, refl, mask = rows(R, V, torch.float16)
    adv = adv * torch.logspace(-4, 4, R, device="cuda")
    for factor in (1.0, 2.0 ** 12, 1.0 / 3.0):
        want = formula(logits, actions, old, adv, refl, mask, kl=0.0)
        top = float(want["grad"].abs().max()) * factor
        assert top < 60000
        _, _, grad = call(logits, actions, old, adv, refl, mask, kl=0.0, factor=factor)
        within("dlogits", grad, want["grad"] * factor, room_of(want["grad"], want["mag"], want["n"], grad.dtype, factor))


@pytest.mark.parametrize("V", [1, 3, 8, 13, 300, 4100])
@pytest.mark.parametrize("R", [1, 2, 9])
def test_half_precision_of_few_rows(R, V):
    """Fewer elements than one access, rows that end inside one, accesses over several rows; the inputs move on before the backward."""
    logits, actions, old, adv, refl, mask = rows(R, V, torch.float16, masked=R > 2)
    from airgym_amd.lib.core.policy_loss import policy_loss
    want = formula(logits, actions, old, adv, refl, mask)
    rest = [t.clone() for t in (actions, old, adv, refl)]
    leaf = logits.clone().requires_grad_()
    gone = leaf * 1.0
    loss, _ = policy_loss(gone, rest[0], rest[1], rest[2], ref_logp=rest[3], mask=mask, e_clip=E_CLIP, kl_coef=KL, entropy_coef=ENT)
    with torch.no_grad():
        gone.zero_()
        for t in rest:
            t.zero_()
    (grad,) = torch.autograd.grad(loss, leaf)
    within("dlogits", grad, want["grad"], room_of(want["grad"], want["mag"], want["n"], grad.dtype))
    assert not grad[~want["on"]].any()


# ------------------------------------------------------------------------------------------------ every form, element by element
# rows of 1 to 32 lanes, of one wave, 256 and 1024 threads, and (from 256 KB on) longer than registers hold; a wave's and a pass's elements there
FORMS = {"f32": [1, 2, 5, 21, 64, 129, 200, 256, 257, 300, 1000, 1500, 2049, 4099, 8193, 9001, 16385, 33001, 65536, 65537, 66001, 70001],
         "bf16": [3, 129, 257, 1000, 2500, 4099, 16385, 33001, 65537, 131072, 131080, 140003],
         "f16": [3, 129, 257, 1000, 2500, 4099, 16385, 33001, 65537, 131072, 131080, 140003]}
HOLES = {"f32": (256, 4096), "bf16": (512, 8192), "f16": (512, 8192)}


def check_all(logits, actions, old, adv, refl, mask, factor=None):
    from airgym_amd.lib.core.policy_loss import action_logp
    want = formula(logits, actions, old, adv, refl, mask)
    n, size = want["n"], want["size"]
    loss, stats, grad = call(logits, actions, old, adv, refl, mask, factor=factor)
    within("loss", loss, want["loss"], n * U * (size[0] + KL * size[1] + ENT * size[2]) + U * want["loss"].abs())
    for k in range(5):
        within(f"statistic {k}", stats[k], want["stats"][k], n * U * size[k] + U * want["stats"][k].abs())
    assert float(stats[5]) == float(want["stats"][5])
    f = 1.0 if factor is None else factor
    room = room_of(want["grad"], want["mag"], n, grad.dtype, f)
    if factor is not None and grad.dtype != torch.float16:              # rounded before the factor is known, and after
        room = room + (U if grad.dtype == torch.float32 else torch.finfo(grad.dtype).eps / 2) * (want["grad"] * f).abs()
    within("dlogits", grad, want["grad"] * f, room)
    assert not grad[~want["on"]].any()
    on = want["on"]
    lp, H = action_logp(logits[on], actions[on])
    within("logp", lp, want["lp"][on], n * U * torch.ones_like(want["lp"][on]))
    within("entropy", H, want["H"][on], n * U * (1 + want["Y"] + want["H"][on]))
    return want, room, f


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("dtype,V", [(d, v) for d, vs in FORMS.items() for v in vs])
def test_loss_statistics_and_gradient(dtype, V, masked):
    args = rows(7, V, DTYPES[dtype], masked)
    want, room, f = check_all(*args)
    if dtype == "f16":
        # Without a loss scale the type itself cannot tell: an entropy term ent p (|log p| + H) / rows of the longest rows is about
        # 0.01 x 20 / (140003 x 7) = 2e-7, and the numbers there are 6e-8 apart.
        want, room, f = check_all(*args, factor=2.0 ** 15)
    if V > 2:                           # the bound is narrow enough to miss neither small term
        for gone in (dict(ent=0.0), dict(kl=0.0)):
            other = formula(*args, **gone)["grad"]
            outside = ((other - want["grad"]).abs() * f > room)[want["on"]]
            few = dtype != "f32" and "kl" in gone
            assert float(outside.float().mean()) > (0.0 if few else 0.3), (gone, float(outside.float().mean()))


@pytest.mark.parametrize("where", ["some", "first wave", "first pass", "last pass", "all but one end"])
@pytest.mark.parametrize("dtype,V", [(d, v) for d, vs in FORMS.items() for v in vs if v > 8000])
def test_long_rows_with_choices_that_are_not_available(dtype, V, where):
    wave, one = HOLES[dtype]
    last = V // one * one
    hole = {"some": "some", "first wave": (0, wave), "first pass": (0, one), "last pass": (last - one, V), "all but one end": (0, V - 1)}[where]
    check_all(*rows(6, V, DTYPES[dtype], masked=where == "first pass", minus_inf=hole))


@pytest.mark.parametrize("V", [2, 21, 256, 300, 9001])
@pytest.mark.parametrize("dtype", DTYPES)
def test_short_rows_with_choices_that_are_not_available_and_a_factor(dtype, V):
    for masked in (False, True):
        check_all(*rows(40, V, DTYPES[dtype], masked, minus_inf="some"), factor=0.3)
