"""The operators from a router to a loss together, as a program calls them, on the GPU."""
import os
import subprocess
import sys

import pytest
import torch

import rocm_wmma_gemm_amd as R

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("sizes", [(), ("--tokens", "33", "--experts", "9", "--choices", "9", "--hidden", "72", "--inner", "40",
                                        "--vocabulary", "301"),
                                   ("--tokens", "2500", "--experts", "40", "--choices", "2", "--hidden", "136", "--inner", "264",
                                    "--vocabulary", "4099")], ids=["default", "few", "many"])
def test_a_training_step_from_router_to_loss(sizes):
    """Loss and every gradient of the example's step against fp64; it ends with an error where one is off."""
    done = subprocess.run([sys.executable, os.path.join(ROOT, "examples", "expert_model.py"), *sizes], capture_output=True, text=True,
                          timeout=110)
    assert done.returncode == 0 and "decode" in done.stdout, done.stdout + done.stderr


def test_a_student_and_its_teacher():
    """The teacher's best logits by the same projection: a student with the teacher's states is at distance 0 from them where the list
    is the whole vocabulary, and its gradient is nothing but roundings."""
    L, M, N, K = R.Loader(), 40, 200, 64
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    a = torch.randn((M, K), device="cuda", generator=g).to(torch.bfloat16)
    w = (torch.randn((N, K), device="cuda", generator=g) / 8).to(torch.bfloat16)
    logits = torch.empty((M, N), device="cuda")
    L.linear(logits, a, w, M, N, K)
    teacher, entries = logits.sort(1, descending=True)
    entries, teacher = entries.to(torch.int32).contiguous(), teacher.contiguous()
    loss, lse, picked = torch.empty(M, device="cuda"), torch.empty(M, device="cuda"), torch.empty((M, N), device="cuda")
    L.linear_distillation(loss, lse, picked, a, w, entries, teacher, M, N, K, temperature=2.0)
    # every term is a difference of numbers up to about 12 that fp32 holds to 2^-24 of themselves, through some 40 roundings
    assert loss.abs().max() < 4 * 40 * 12 * 2.0 ** -24
    dA, dB = torch.empty_like(a), torch.empty_like(w)
    L.linear_distillation_backward(dA, dB, torch.ones(M, device="cuda"), lse, picked, a, w, entries, teacher, M, N, K, temperature=2.0)
    assert dA.float().abs().max() < 1e-4 and dB.float().abs().max() < 1e-3


def test_two_streams_and_two_graphs_share_the_scratch_buffer():
    """Losses and dispatches on two streams at a time, and two captured graphs replayed one after the other, leave what they leave alone."""
    L, M, N, K, k, E = R.Loader(), 700, 3001, 96, 8, 32
    g = torch.Generator(device="cuda")
    g.manual_seed(2)

    class Job:
        def __init__(self):
            self.a = torch.randn((M, K), device="cuda", generator=g).to(torch.bfloat16)
            self.w = (torch.randn((N, K), device="cuda", generator=g) / 8).to(torch.bfloat16)
            self.t = torch.randint(N, (M,), device="cuda", generator=g)
            self.chosen = torch.randint(E, (M, k), device="cuda", generator=g).to(torch.int32)
            new = lambda *s, d=torch.float32: torch.zeros(s, device="cuda", dtype=d)  # noqa: E731
            self.loss, self.lse, self.g = new(M), new(M), torch.ones(M, device="cuda")
            self.da, self.dw = torch.zeros_like(self.a), torch.zeros_like(self.w)
            self.rows, self.offsets, self.places = new(M * k, K, d=torch.bfloat16), new(E + 1, d=torch.int32), new(M, k, d=torch.int32)

        def run(self, stream=None):
            L.linear_cross_entropy(self.loss, self.lse, self.a, self.w, self.t, M, N, K, stream=stream)
            L.dispatch(self.rows, self.offsets, self.places, self.a, self.chosen, M, K, k, stream=stream)
            L.linear_cross_entropy_backward(self.da, self.dw, self.g, self.lse, self.a, self.w, self.t, M, N, K, stream=stream)

        def results(self):
            return [t.clone() for t in (self.loss, self.lse, self.da, self.dw, self.rows, self.offsets, self.places)]

        def clear(self):
            for t in (self.loss, self.lse, self.da, self.dw, self.rows, self.offsets, self.places):
                t.zero_()

    jobs, streams = [Job(), Job()], [torch.cuda.Stream(), torch.cuda.Stream()]
    want = []
    for j in jobs:
        j.run()
        torch.cuda.synchronize()
        want.append(j.results())
    for _ in range(3):
        for j in jobs:
            j.clear()
        torch.cuda.synchronize()
        for _ in range(2):
            for j, s in zip(jobs, streams):
                j.run(s)
        torch.cuda.synchronize()
        for j, w in zip(jobs, want):
            assert all(torch.equal(x, y) for x, y in zip(j.results(), w))
    graphs = []
    for j in jobs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            j.run()
    for _ in range(3):
        for j in jobs:
            j.clear()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for j, w in zip(jobs, want):
            assert all(torch.equal(x, y) for x, y in zip(j.results(), w))
