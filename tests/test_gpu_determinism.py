"""Race smoke test: kernels whose result does not depend on scheduling must return the same bits on every run.

There is no memory checker or race detector to run these kernels under, so a data race (a tile read before its copy
landed, an epilogue buffer reused too early, an accumulator shared by two CTAs) is looked for by its symptom: run the
same launch several times on the same inputs, interleaved with other work that perturbs the timing, and compare the
outputs bit for bit.  Kernels that combine partial results with floating-point atomics or TMA reductions in an order
that depends on scheduling (split / stream-K GEMM tails, norm weight gradients) are excluded by construction.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _perturb():
    a = torch.randn(1024, 1024, device="cuda")
    (a @ a).sum().item()


def _same_bits(fn, runs=4):
    first = None
    for i in range(runs):
        out = fn()
        torch.cuda.synchronize()
        out = [o.clone() for o in (out if isinstance(out, (tuple, list)) else [out])]
        if first is None:
            first = out
        else:
            for a, b in zip(first, out):
                assert torch.equal(a, b), f"run {i} differs from run 0 in {(a != b).sum().item()} elements"
        _perturb()


def test_gemm_batched_and_symmetric_are_bitwise_reproducible():
    from himuon_b200 import ops

    torch.manual_seed(0)
    x = torch.randn(24, 512, 384, device="cuda", dtype=torch.bfloat16)
    a = torch.randn(3, 640, 640, device="cuda", dtype=torch.bfloat16) / 25
    _same_bits(lambda: ops.gemm(x, x, trans_b=True))
    _same_bits(lambda: ops.gemm(x, x, trans_b=True, symmetric=True))
    _same_bits(lambda: ops.gemm(a, a, trans_b=True, alpha=2.0, beta=-4.7, aux=a, symmetric=True))
    _same_bits(lambda: ops.gemm(a, a, alpha=1.0, beta=3.4, aux=a, round_acc=True))
    ops.check_status()


def test_newton_schulz_paths_are_bitwise_reproducible():
    from himuon_b200 import ops
    from himuon_b200.ops import ns as ns_ops

    torch.manual_seed(1)
    for shape in [(64, 128, 128), (16, 512, 512), (9, 64, 256), (4, 768, 520)]:
        x = torch.randn(*shape, device="cuda", dtype=torch.bfloat16)
        _same_bits(lambda: ns_ops.newton_schulz(x, 5))
    ops.check_status()


def test_attention_forward_and_backward_are_bitwise_reproducible():
    from himuon_b200 import ops

    torch.manual_seed(2)
    B, S, Hq, Hkv = 2, 512, 8, 2
    q = torch.randn(B * S, Hq * 128, device="cuda", dtype=torch.bfloat16)
    k = torch.randn(B * S, Hkv * 128, device="cuda", dtype=torch.bfloat16)
    v = torch.randn(B * S, Hkv * 128, device="cuda", dtype=torch.bfloat16)
    do = torch.randn(B * S, Hq * 128, device="cuda", dtype=torch.bfloat16)

    def run():
        qq, kk, vv = (t.clone().requires_grad_(True) for t in (q, k, v))
        o = ops.attention(qq, kk, vv, B, S, Hq, Hkv, 128)
        o.backward(do)
        return o.detach(), qq.grad, kk.grad, vv.grad

    _same_bits(run)
    ops.check_status()


def test_optimizer_step_is_bitwise_reproducible():
    from helpers import make_linear_model, seed_grads
    from himuon_b200.optimizers import HiMuon

    def run():
        torch.manual_seed(3)
        model = make_linear_model([(512, 768), (256, 256), (300, 520)], dtype=torch.bfloat16, device="cuda")
        opt = HiMuon([{"params": list(model.parameters())}], tile_size=128, cuda_graph=False, lr=0.02)
        for s in range(3):
            seed_grads(model, s)
            opt.step()
        return [p.detach() for p in model.parameters()]

    _same_bits(run, runs=3)


@pytest.mark.parametrize("M,N,K", [(2048, 2560, 9728), (2560, 2048, 6144), (11520, 2560, 4096)])
def test_gemm_split_tail_is_bitwise_reproducible(M, N, K):
    """A last wave of tiles cut into three or more K-slices: they are added in their order, not in that of their arrival."""
    from himuon_b200 import ops

    torch.manual_seed(4)
    a = torch.randn(M, K, device="cuda", dtype=torch.bfloat16)
    b = torch.randn(N, K, device="cuda", dtype=torch.bfloat16)
    _same_bits(lambda: ops.gemm(a, b, trans_b=True), runs=6)
    ops.check_status()


def test_split_gemms_on_two_streams_do_not_meet():
    """Two products whose last waves are cut run at the same time; neither finds the other's partial sums."""
    from himuon_b200 import ops

    torch.manual_seed(5)
    operands = [(torch.randn(2048, 9728, device="cuda", dtype=torch.bfloat16), torch.randn(2560, 9728, device="cuda", dtype=torch.bfloat16)) for _ in range(2)]
    want = [ops.gemm(a, b, trans_b=True) for a, b in operands]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in operands]
    got = [[], []]
    for _ in range(10):
        for i, (a, b) in enumerate(operands):
            with torch.cuda.stream(streams[i]):
                got[i].append(ops.gemm(a, b, trans_b=True))
    torch.cuda.synchronize()
    for outs, w in zip(got, want):
        assert all(torch.equal(o, w) for o in outs)
    ops.check_status()
