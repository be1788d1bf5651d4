"""Times of the sequence operators (pnp_amd.seqops) beyond the cases of perf/operators.py: odd sizes beside aligned ones,
short and narrow ones, products of every depth, and the history encoder and learner over them.  Everything is captured into
a graph of several passes, so that the kernels are timed and not torch's engine; a gradient's time is that of the forward
with its gradient less that of the forward in training.  usage: python tools/seqops_sizes.py [norm conv scan i8 step history]"""
import os
import sys
import time

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path[:0] = [ROOT, os.path.join(ROOT, "mujoco-panda-pnp_amd")]
from pnp_amd import seqops as S  # noqa: E402

F32, BF16 = torch.float32, torch.bfloat16
NAME = {F32: "f32", BF16: "bf16"}


def rnd(*shape, dtype=BF16):
    return torch.randn(*shape, device="cuda", dtype=dtype)


def timed(f, passes=5, least_ms=150.0):
    """us a pass, the median of replays after 150 ms of them (a warm chip's clock)."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            f()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for _ in range(passes):
            f()
    begin, times = time.perf_counter(), []
    while (time.perf_counter() - begin) * 1e3 < least_ms or len(times) < 15:
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        g.replay()
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b) * 1e3 / passes)
    times = sorted(times[len(times) // 2:])
    del g
    return times[len(times) // 2]


def line(name, us, more=""):
    print(f"{name:44s} {us:9.2f}{more}", flush=True)


def gradient(name, leaves, forward, dy):
    """forward(*leaves) -> outputs; their gradients by dy."""
    def new():
        return [t.detach().requires_grad_() for t in leaves]

    def both():
        v = new()
        return torch.autograd.grad(forward(*v), v, dy)
    with torch.no_grad():
        serve = timed(lambda: forward(*leaves))
    train = timed(lambda: forward(*new()))
    whole = timed(both)
    line(name, serve, f"   training {train:9.2f}   gradient {whole - train:9.2f}")


def norm():
    for rows, dim, t in [(8192, d, BF16) for d in (4096, 4095, 4100)] + [(32768, d, F32) for d in (1024, 1023)] + \
            [(200000, d, BF16) for d in (64, 63, 77)] + [(16896, 256, F32)]:
        x, r, dy, w = rnd(rows, dim, dtype=t), rnd(rows, dim, dtype=t), rnd(rows, dim, dtype=t), rnd(dim, dtype=F32)
        gradient(f"norm {rows}x{dim} {NAME[t]}", [x, r, w], lambda x, r, w: S.add_rms_norm(x, w, r), [dy, dy])
    for dim in (1024, 1023):
        x = rnd(8192, dim)
        line(f"rows in 8 bits 8192x{dim} bf16", timed(lambda: S.quantize_rows(x)))


def conv():
    for B, L, D, t in [(2, 4096, d, BF16) for d in (2048, 2047, 2046, 2044)] + [(512, 33, d, F32) for d in (512, 511)]:
        x, dy, w = rnd(B, L, D, dtype=t), rnd(B, L, D, dtype=t), rnd(D, 4, dtype=F32)
        gradient(f"conv {B}x{L}x{D} {NAME[t]}", [x, w], lambda x, w: S.causal_conv(x, w, activation="silu")[0], dy)


def scan():
    sizes = [(2, 2048, d, 16, BF16) for d in (2048, 2047, 2044)] + [(64, 512, d, 16, F32) for d in (256, 255)]
    sizes += [(64, 512, 256, n, F32) for n in (12, 8, 4)]
    sizes += [(4, 32, 128, 16, F32), (4, 192, 128, 16, F32), (4, 192, 128, 4, F32), (1, 1000, 64, 16, F32), (1, 4000, 64, 16, F32),
              (1, 100000, 64, 16, F32), (16, 512, 100, 4, F32), (60, 200, 256, 16, F32), (32, 100, 256, 16, F32), (100, 128, 256, 16, F32),
              (64, 128, 256, 64, F32), (512, 33, 512, 16, F32), (1, 8192, 2048, 16, BF16), (4, 2048, 2048, 16, BF16)]
    # narrow: fewer channels than a workgroup has lanes for; short: fewer tokens than a tile holds
    sizes += [(256, 1024, 8, 4, F32), (256, 1024, 16, 4, F32), (256, 1024, 64, 4, F32), (256, 1024, 256, 4, F32), (256, 1024, 8, 16, F32),
              (256, 1024, 64, 16, F32), (40944, 3, 55, 8, BF16), (5000, 8, 200, 16, F32), (20000, 1, 256, 16, F32), (20000, 5, 64, 16, F32)]
    for B, L, D, N, t in sizes:
        u, d, z, dy = (rnd(B, L, D, dtype=t) for _ in range(4))
        Bm, Cm, A, skip = rnd(B, L, N, dtype=t), rnd(B, L, N, dtype=t), -torch.rand(D, N, device="cuda") - 0.1, rnd(D, dtype=F32)
        gradient(f"scan {B}x{L}x{D}x{N} {NAME[t]}", [u, d, A, Bm, Cm, skip, z],
                 lambda u, d, A, Bm, Cm, D, z: S.selective_scan(u, d, A, Bm, Cm, D=D, z=z)[0], dy)


def i8():
    square = [(8192, 8192, 8192), (8192, 8192, 1024), (8192, 8192, 8184), (8191, 8191, 8191), (4096, 4096, 4096), (2048, 2048, 8192),
              (1000, 1000, 1000), (1000, 1000, 1008), (999, 1001, 997), (8192, 1000, 257), (8192, 1000, 256)]
    few = [(1, 1000, 512), (1, 4096, 4096), (1, 8000, 8000), (1, 8000, 8001), (1, 16384, 8192)] + \
          [(m, 4096, 4096) for m in (16, 17, 33, 64, 65, 128, 256, 512, 1000)]
    deep = [(64, 16, 8192), (65, 64, 8192), (100, 100, 8192), (300, 300, 8192), (64, 1000, 1001), (64, 1000, 1008)]
    for M, N, K in square + few + deep:
        q, w = (torch.randint(-127, 128, (n, K), dtype=torch.int8, device="cuda") for n in (M, N))
        s, ws = torch.rand(M, device="cuda"), torch.rand(N, device="cuda")
        us = timed(lambda: S.matmul_i8(q, s, w, ws, out_dtype=BF16))
        line(f"i8 {M}x{N}x{K}", us, f"   {2e-6 * M * N * K / us:8.1f} TOP/s {(M * K + N * K + 2 * M * N) / us * 1e-6:6.2f} TB/s")


def step():
    for B, D, N in [(8192, 512, 16), (8192, 511, 16), (8192, 8, 4), (8192, 64, 4), (8192, 8, 16), (8192, 64, 16), (8192, 256, 4)]:
        for t in (F32, BF16):
            u, Bm, A, h = rnd(B, D, dtype=t), rnd(B, N, dtype=t), -torch.rand(D, N, device="cuda"), torch.zeros(B, D, N, device="cuda")
            line(f"scan step {B}x{D}x{N} {NAME[t]}", timed(lambda: S.selective_scan_step(u, h, u, A, Bm, Bm, z=u)))
    for D in (512, 511):
        for t in (F32, BF16):
            u, c, w = rnd(8192, D, dtype=t), rnd(8192, 3, D, dtype=t), rnd(D, 4, dtype=F32)
            line(f"conv step 8192x{D} {NAME[t]}", timed(lambda: S.causal_conv_step(u, c, w, activation="silu")))


def history():
    from pnp_amd.envs import BatchedFrankaShelfPNPEnv, EnvConfig
    from pnp_amd.history import HistoryEncoder
    from pnp_amd.tqc import TQC, TQCConfig
    torch.manual_seed(0)
    enc = HistoryEncoder(32).cuda()
    for n in (8192, 64, 1):
        x, state, reset = rnd(n, 32, dtype=F32), enc.new_state(n), torch.zeros(n, dtype=torch.bool, device="cuda")
        for name, q in (("fp32", None), ("8 bits", enc.int8_weights())):
            line(f"encoder step, {n} envs, {name}", timed(lambda: enc.step(x, state, reset=reset, int8=q)))
    env = BatchedFrankaShelfPNPEnv(64, config=EnvConfig(n_substeps=2, n_calls=2))
    for h in (0, 32):     # the PyTorch step either way, captured
        a = TQC(env, TQCConfig(fused=False, history=h))
        a.total_timesteps = 10 ** 6
        a.reset()
        for _ in range(40):
            a.collect_step()
        a.train(10)
        torch.cuda.synchronize()
        begin = time.perf_counter()
        a.train(200)
        torch.cuda.synchronize()
        line(f"learner's captured step, batch 512, history {h}", (time.perf_counter() - begin) / 200 * 1e6)


if __name__ == "__main__":
    print("us a pass; gradient: forward with gradient less the forward in training; all captured")
    for name in sys.argv[1:] or ("norm", "conv", "scan", "i8", "step", "history"):
        {"norm": norm, "conv": conv, "scan": scan, "i8": i8, "step": step, "history": history}[name]()
