"""Child process of tests/test_attention.py (captured graphs; a process of its own because graph replay needs its environment
before the first HIP call).  ``layer``: layers.CrossAttention captured forward and backward, replayed between eager work, every
replay against the eager result.  ``step``: tests/hip_graph_worker.py with --fusion_attention 2."""
import functools
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path[:0] = [ROOT, os.path.join(ROOT, "tests")]

import torch  # noqa: E402


def layer():
    import mono_vifi_amd
    mono_vifi_amd.ensure_graph_replay_env()
    from mono_vifi_amd import layers
    worst = 0.0
    for seed, (B, H, W, C) in enumerate(((2, 6, 20, 512), (12, 12, 40, 256))):
        torch.manual_seed(seed)
        m = layers.CrossAttention(C, 8).cuda()
        pos, spos = layers.token_positions(H, W, (0,), "cuda"), layers.token_positions(H, W, (-1, 1), "cuda")
        x, states, go = (torch.randn(B, n, C, device="cuda") for n in (H * W, 2 * H * W, H * W))
        leaves = [x.requires_grad_(True), states.requires_grad_(True)] + list(m.parameters())

        def step():
            y = m(x, states, pos, spos)
            return [y.detach()] + list(torch.autograd.grad(y, leaves, go))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(3):
                step()
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = step()
        for turn in range(5):
            with torch.no_grad():
                x.mul_(0.9)
                states.add_(0.1)
            g.replay()
            torch.cuda.synchronize()
            for a, b in zip(got, step()):
                worst = max(worst, float((a.double() - b.double()).norm() / b.double().norm()))
            torch.cuda.synchronize()
    print("RESULT", worst, flush=True)


def step():
    from mono_vifi_amd import options
    options.default_options = functools.partial(options.default_options, fusion_attention=2)
    import hip_graph_worker
    hip_graph_worker.main()


if __name__ == "__main__":
    {"layer": layer, "step": step}[sys.argv.pop(1)]()
