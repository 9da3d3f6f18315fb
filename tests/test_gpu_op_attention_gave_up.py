"""Attention's bounded waits giving up: with a limit of no polls (or very few) every wait (or some) ends at once, without what it
waited for.  Nothing hangs, the rows whose results did not come are NaN, whatever the buffers held, the rest are right, the
CTAs count themselves, and calls after that with the ordinary limit give the bits they gave before.  In a process of its own,
since the counter is the process's."""
import os
import subprocess
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CASES = [
    # B, Lq, Lk, H, Hkv, D, causal, buckets
    (64, 512, 512, 8, 8, 64, False, 16),     # several items a CTA
    (48, 512, 512, 16, 4, 128, True, 16),
    (64, 512, 512, 8, 2, 64, False, 0),
    (2, 300, 300, 4, 2, 128, True, 0),       # an item a CTA
    (1, 40, 3000, 2, 2, 64, False, 16),      # split keys
]


def child():
    import ctypes

    import d2p_b200  # noqa: F401
    from tests.test_encoder_host import AttentionArgs
    from tests.test_gpu_encoder import inputs

    lib = ctypes.CDLL(os.path.join(ROOT, "d2p_b200", "libd2p_b200.so"))
    P = ctypes.c_void_p
    lib.d2p_attention_forward.argtypes = [ctypes.POINTER(AttentionArgs), P, P, P, P, ctypes.c_size_t, P]
    lib.d2p_attention_backward.argtypes = [ctypes.POINTER(AttentionArgs)] + [P] * 9 + [ctypes.c_size_t, P]
    for f in (lib.d2p_attention_forward_workspace_bytes, lib.d2p_attention_backward_workspace_bytes):
        f.restype = ctypes.c_size_t
    dev = torch.device("cuda")

    def gave_up():
        n = ctypes.c_ulonglong()
        assert lib.d2p_attention_gave_up(ctypes.byref(n)) == 0
        return n.value

    for B, Lq, Lk, H, Hkv, D, causal, nb in CASES:
        q, k, v, do, bias = inputs(B, Lq, Lk, H, Hkv, D, torch.bfloat16, dev, nb)
        lengths = torch.tensor([[Lq, Lk]] * (B - 1) + [[Lq, 0] if B > 2 else [Lq, Lk]], dtype=torch.int32, device=dev)
        edges = d2p_b200.relative_bucket_edges(nb, 64, not causal) if nb else ()
        a = AttentionArgs(q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), bias=bias.data_ptr() if nb else None, lengths=lengths.data_ptr(),
                          bucket_edges=(ctypes.c_int * max(1, len(edges)))(*edges), n_edges=len(edges), bias_dtype=1, B=B, Lq=Lq, Lk=Lk, H=H,
                          Hkv=Hkv, D=D, dtype=1, causal=causal, scale=D ** -0.5)
        a.q_stride = (ctypes.c_longlong * 3)(Lq * H * D, H * D, D)
        a.k_stride = a.v_stride = (ctypes.c_longlong * 3)(Lk * Hkv * D, Hkv * D, D)
        fw, bw = lib.d2p_attention_forward_workspace_bytes(ctypes.byref(a)), lib.d2p_attention_backward_workspace_bytes(ctypes.byref(a), int(nb > 0))
        ws = torch.empty(max(fw, bw, 16), dtype=torch.uint8, device=dev)

        def fresh():
            sevens = {n: torch.full_like(t, 7.0) for n, t in (("out", q), ("rest", q), ("dq", q), ("dk", k), ("dv", v))}
            sevens["lse"] = torch.full((B, H, Lq), 7.0, device=dev)
            sevens["dbias"] = torch.full_like(bias, 7.0) if nb else None
            return sevens

        def forward(t):
            assert lib.d2p_attention_forward(ctypes.byref(a), t["out"].data_ptr(), t["lse"].data_ptr(), t["rest"].data_ptr(), ws.data_ptr(), fw, None) == 0
            torch.cuda.synchronize()

        def backward(t, saved):
            assert lib.d2p_attention_backward(ctypes.byref(a), saved["out"].data_ptr(), saved["rest"].data_ptr(), saved["lse"].data_ptr(), do.data_ptr(),
                                              t["dq"].data_ptr(), t["dk"].data_ptr(), t["dv"].data_ptr(),
                                              t["dbias"].data_ptr() if nb else None, ws.data_ptr(), bw, None) == 0
            torch.cuda.synchronize()

        want = fresh()
        forward(want)
        backward(want, want)
        for polls in (0,) + (1, 2, 4) * 20:   # (how far a CTA gets with a few goes by chance)
            before = gave_up()
            got = fresh()
            default = lib.d2p_attention_wait_limit(polls)
            forward(got)
            assert gave_up() > before or polls
            middle = gave_up()
            backward(got, want)
            assert gave_up() > middle or polls
            assert lib.d2p_attention_wait_limit(-1) == polls
            for n in ("out", "lse", "rest", "dq", "dk", "dv", "dbias"):
                if got[n] is None:
                    continue
                same, lost = got[n] == want[n], torch.isnan(got[n])
                assert (same | lost).all(), (n, polls, int((~(same | lost)).sum()))
                # what no wait stands before (rows and problems without keys): not lost
                if polls == 0 and n in ("out", "dq"):
                    live = lengths[:, 1] > 0
                    assert lost[live].all() and same[~live].all(), n
                if polls == 0 and n == "dbias":
                    assert lost.all()
        again = fresh()
        forward(again)
        backward(again, again)
        assert all(want[n] is None or torch.equal(want[n], again[n]) for n in want)
        assert default == 1 << 21
    print("gave up", gave_up())


def test_waits_that_give_up(cuda_device):
    r = subprocess.run([sys.executable, "-c", "import sys; sys.path.insert(0, sys.argv[1]); from tests.test_gpu_op_attention_gave_up import child; child()", ROOT],
                       capture_output=True, text=True, timeout=300, cwd=ROOT)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-4000:]
    assert "gave up" in r.stdout
