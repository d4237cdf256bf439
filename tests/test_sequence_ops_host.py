"""The sequence operators' C entries refuse bad arguments on the host, before anything is launched; layouts of their argument blocks;
the float64 restatement they are tested against, checked by differences.  No GPU needed."""
import ctypes
import os
import shutil
import subprocess

import pytest
import torch

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(REPO, "include", "airgym_hip.h")


@pytest.fixture(scope="module")
def lib():
    from airgym_amd import _native
    return _native.load()


def _blocks():
    from airgym_amd import _native as N
    p = ctypes.cast((ctypes.c_float * 64)(), ctypes.c_void_p).value
    conv = N.AgConvArgs(ctypes.sizeof(N.AgConvArgs), 0, 2, 5, 8, 4, 1, p, p, None, None, None, None, 40, 8, 0, 0, p, None)
    scan = N.AgScanArgs(ctypes.sizeof(N.AgScanArgs), 0, 2, 5, 8, 16, 1, 1, p, p, None, p, p, p)
    scan.out_dev = scan.state_out_dev = scan.ckpt_dev = p
    loss = N.AgTokenLossArgs(ctypes.sizeof(N.AgTokenLossArgs), 0, 9, 1, 3, 27, 9, p, p, p, p, None, None, 0.2, 0.0, 0.0, p, p, p, p, 1 << 20)
    return N, p, conv, scan, loss


def test_conv_entries_refuse(lib):
    N, p, a, _, _ = _blocks()
    fwd = lambda: lib.ag_causal_conv_fwd(ctypes.byref(a), None)      # noqa: E731
    for field, value, rc in [("struct_size", 4, -1), ("x_dev", None, -1), ("weight_dev", None, -1), ("y_dev", None, -1), ("B", 0, -1), ("T", 0, -1),
                             ("D", -1, -1), ("T", (1 << 30) + 1, -6), ("W", 1, -6), ("W", 9, -6), ("dtype", 3, -6), ("dtype", -1, -6)]:
        old = getattr(a, field)
        setattr(a, field, value)
        assert fwd() == rc, field
        setattr(a, field, old)
    g = N.AgConvGrads(ctypes.sizeof(N.AgConvGrads), p, None, 40, 8, p, p, None, None, p, 0)
    assert lib.ag_causal_conv_bwd(ctypes.byref(a), ctypes.byref(g), None) == -1          # workspace too small
    assert lib.ag_causal_conv_bwd(ctypes.byref(a), None, None) == -1 and lib.ag_causal_conv_fwd(None, None) == -1
    assert lib.ag_causal_conv_workspace_bytes(2, 5, 8, 4, 0) > 0 and lib.ag_causal_conv_workspace_bytes(2, 5, 8, 9, 0) == 0
    assert lib.ag_causal_conv_step(p, 8, None, p, None, None, p, 0, 2, 8, 4, 1, None) == -1
    assert lib.ag_causal_conv_step(p, 8, p, p, None, None, p, 0, 2, 8, 9, 1, None) == -6


def test_scan_entries_refuse(lib):
    N, p, _, a, _ = _blocks()
    for field, value, rc in [("struct_size", 4, -1), ("u_dev", None, -1), ("delta_dev", None, -1), ("Bm_dev", None, -1), ("A_dev", None, -1),
                             ("out_dev", None, -1), ("B", 0, -1), ("T", 0, -1), ("T", (1 << 30) + 1, -6), ("u_st", -1, -1), ("b_st", 1 << 26, -6), ("D", 1 << 28, -6), ("G", 3, -1), ("G", 0, -1), ("N", 33, -6), ("N", 0, -1), ("dtype", 7, -6)]:
        old = getattr(a, field)
        setattr(a, field, value)
        assert lib.ag_selective_scan_fwd(ctypes.byref(a), None) == rc, field
        setattr(a, field, old)
    assert lib.ag_selective_scan_step(ctypes.byref(a), None) == -1                       # T = 5
    g = N.AgScanGrads(ctypes.sizeof(N.AgScanGrads), p, 40, 8, None, p, p, None, p, p, p, None, None, None, p, 0)
    assert lib.ag_selective_scan_bwd(ctypes.byref(a), ctypes.byref(g), None) == -1       # workspace too small
    g.workspace_bytes, g.dz_dev = 1 << 30, p
    assert lib.ag_selective_scan_bwd(ctypes.byref(a), ctypes.byref(g), None) == -1       # dz without z
    g.dz_dev, a.T, a.ckpt_dev = None, 1000, None
    assert lib.ag_selective_scan_bwd(ctypes.byref(a), ctypes.byref(g), None) == -1       # long sequences need the forward's states
    assert lib.ag_selective_scan_ckpt_floats(2, 1, 8, 16) == 0 and lib.ag_selective_scan_workspace_bytes(2, 5, 8, 16, 3, 1) == 0


def test_loss_entries_refuse(lib):
    N, p, _, _, a = _blocks()
    for field, value, rc in [("struct_size", 4, -1), ("logits_dev", None, -1), ("actions_dev", None, -1), ("old_logp_dev", None, -1),
                             ("stats_dev", None, -1), ("loss_dev", None, -1), ("workspace_dev", None, -1), ("workspace_bytes", 4, -1), ("V", 0, -1), ("V", 2147483647, -6), ("R0", 0, -1),
                             ("dtype", 5, -6), ("R0", 1 << 31, -6)]:
        old = getattr(a, field)
        setattr(a, field, value)
        assert lib.ag_token_policy_loss(ctypes.byref(a), None) == rc, field
        setattr(a, field, old)
    assert lib.ag_token_logp(p, 1, 3, 27, 9, 9, 0, None, p, p, None) == -1 and lib.ag_token_logp(p, 1, 3, 27, 9, 9, 4, p, p, p, None) == -6
    # 64 threads per row of 257 to 2048 float32 logits, 1024 beyond 8192: more than one launch holds
    assert lib.ag_token_logp(p, 1 << 26, 1, 300, 300, 300, 0, p, p, p, None) == -6
    assert lib.ag_token_logp(p, 1 << 22, 1, 9000, 9000, 9000, 0, p, p, p, None) == -6
    assert lib.ag_token_policy_loss_workspace_bytes(3, 2147483647) > 0
    assert lib.ag_scale_by(p, 0, 0, p, None, None) == -1 and lib.ag_scale_by(p, 4, 9, p, None, None) == -6


def test_argument_blocks_match_the_header(tmp_path):
    N = _blocks()[0]
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    mirrors = {"ag_conv_args": N.AgConvArgs, "ag_conv_grads": N.AgConvGrads, "ag_scan_args": N.AgScanArgs, "ag_scan_grads": N.AgScanGrads,
               "ag_token_loss_args": N.AgTokenLossArgs}
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void) {"]
    for c, m in mirrors.items():
        lines.append(f'  printf("{c} size %zu\\n", sizeof({c}));')
        lines += [f'  printf("{c} {f} %zu\\n", offsetof({c}, {f}));' for f, _ in m._fields_]
    (tmp_path / "l.c").write_text("\n".join(lines + ["  return 0;", "}"]))
    subprocess.run([cc, "-std=c99", "-o", str(tmp_path / "l"), str(tmp_path / "l.c")], check=True, capture_output=True)
    for line in subprocess.run([str(tmp_path / "l")], check=True, capture_output=True, text=True).stdout.splitlines():
        c, what, val = line.split()
        assert (ctypes.sizeof(mirrors[c]) if what == "size" else getattr(mirrors[c], what).offset) == int(val), line


def test_calls_on_the_cpu_are_refused():
    from airgym_amd.lib.core.policy_loss import policy_loss
    from airgym_amd.lib.network.causal_conv import causal_conv
    from airgym_amd.lib.network.selective_scan import selective_scan
    x = torch.zeros(2, 5, 8)
    for call in (lambda: causal_conv(x, torch.zeros(8, 4)), lambda: selective_scan(x, x, torch.zeros(8, 16), torch.zeros(2, 5, 16), torch.zeros(2, 5, 16)),
                 lambda: policy_loss(x[0], torch.zeros(5, dtype=torch.int64), torch.zeros(5), torch.zeros(5))):
        with pytest.raises(ValueError, match="GPU"):
            call()


def test_the_restatement_against_differences():
    from oracle import sequence_ref as ref
    g = torch.Generator().manual_seed(0)

    def r(*s):
        return torch.randn(*s, generator=g, dtype=torch.float64).requires_grad_()

    ln, resets = torch.tensor([4, 6]), torch.rand(2, 6, generator=g) < 0.3
    A = (-torch.rand(4, 3, generator=g, dtype=torch.float64)).requires_grad_()
    assert torch.autograd.gradcheck(lambda *a: ref.selective_scan(*a, lengths=ln, resets=resets),
                                    (r(2, 6, 4), r(2, 6, 4), A, r(2, 6, 2, 3), r(2, 6, 2, 3), r(4), r(2, 6, 4), r(4), r(2, 4, 3)))
    assert torch.autograd.gradcheck(lambda x, w, b, s: ref.causal_conv(x, w, b, s, True, ln, resets), (r(2, 6, 4), r(4, 3), r(4), r(2, 2, 4)))
    actions, mask = torch.tensor([0, 2, 1]), torch.tensor([True, False, True])
    old, adv, refl = (torch.randn(3, generator=g, dtype=torch.float64) * 0.1 - 1.0 for _ in range(3))
    assert torch.autograd.gradcheck(lambda x: ref.policy_loss(x, actions, old, adv, refl, mask, 0.2, 0.1, 0.01)[0], (r(3, 4),))
