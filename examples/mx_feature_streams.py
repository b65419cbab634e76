"""Recurrent feature planes of several streams, held and updated in microscaled formats.

Every frame, each stream's plane of features (pixels x channels, as the decoder
keeps it between frames) is read back from a paged cache, goes through a
feed-forward block of two 1x1 convolutions (products over the pixels) with a
residual, and is quantised into the cache again.  The planes of all streams go
through each call together, packed; each stream's pages lie where its table
says.

    python examples/mx_feature_streams.py [--format mxfp8] [--streams 3] [--height 34] [--width 60] [--frames 4]

Prints how far the planes are from the same frames computed in 32 bits
throughout, and the time of a frame.
"""

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "mlvc.cpp_b200"))

from mlvc_b200 import Backend  # noqa: E402
from mlvc_b200.mx import MxCache, MxLinear, MxMatrix  # noqa: E402


def alloc(nbytes):
    return torch.empty(nbytes, dtype=torch.uint8, device="cuda")


def tensor_scale(fmt, t, room=1.0):
    """nvfp4: brings `room` times the largest value to the largest code and scale."""
    return room * float(t.abs().max().float() / (6 * 448)) if fmt == "nvfp4" else 1.0


def run(fmt="mxfp8", streams=3, height=34, width=60, channels=256, hidden=512, frames=4, page_rows=64, seed=0):
    """(relative error of the planes against 32 bits, of the weights alone, ms a frame)."""
    backend = Backend(0)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    pixels = height * width
    plane = normal(streams * pixels, channels)
    w1, w2 = normal(hidden, channels) / channels**0.5, 0.25 * normal(channels, hidden) / hidden**0.5
    b1, b2 = 0.1 * normal(hidden), 0.1 * normal(channels)
    stream = torch.cuda.current_stream().cuda_stream

    # the weights, quantised once, and how far they are from what they were
    layers, off = [], 0.0
    for w, b, slope, x in ((w1, b1, 0.01, plane), (w2, b2, 1.0, plane)):
        held = MxMatrix.allocate(fmt, *w.shape, alloc, tensor_scale(fmt, w))
        backend.mx_quantise(w, held, stream=stream)
        back = torch.empty_like(w)
        backend.mx_dequantise(held, back, stream=stream)
        off = max(off, float((back - w).norm() / w.norm()))
        # calibrated on the first frame, with room for what follows
        layers.append(MxLinear(backend, held, bias=b, slope=slope, tensor_scale=tensor_scale(fmt, x, 2.0)))
    workspace = alloc(max(layer.workspace_bytes(streams * pixels) for layer in layers))

    # the cache: every stream's pages anywhere in it
    pages_each = -(-pixels // page_rows)
    cache = MxCache.allocate(fmt, streams * pages_each, page_rows, channels, alloc, tensor_scale(fmt, plane, 2.0))
    pages = torch.randperm(streams * pages_each, device="cuda", generator=gen).to(torch.int32).view(streams, pages_each)
    offsets = torch.arange(streams + 1, device="cuda", dtype=torch.int32) * pixels

    prior = torch.empty(streams * pixels, channels, dtype=torch.float16, device="cuda")
    inner = torch.empty(streams * pixels, hidden, dtype=torch.float16, device="cuda")
    feature = plane.half()
    backend.mx_cache_write(cache, feature, pages, offsets, stream=stream)

    def frame():
        backend.mx_cache_read(cache, prior, pages, offsets, stream=stream)
        layers[0](prior, inner, workspace=workspace, stream=stream)
        layers[1](inner, feature, residual=prior, workspace=workspace, stream=stream)
        backend.mx_cache_write(cache, feature, pages, offsets, stream=stream)

    want = plane
    for _ in range(frames):
        frame()
        want = want + torch.nn.functional.leaky_relu(want @ w1.t() + b1, 0.01) @ w2.t() + b2
    error = float((feature.float() - want).norm() / want.norm())
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    begin.record()
    for _ in range(20):
        frame()
    end.record()
    torch.cuda.synchronize()
    backend.synchronize()  # reports rows without a place and waits that ran out
    ms = begin.elapsed_time(end) / 20
    backend.close()
    return error, off, ms


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--format", choices=("mxfp4", "nvfp4", "mxfp8"), default="mxfp8")
    for name, default in (("streams", 3), ("height", 34), ("width", 60), ("channels", 256), ("hidden", 512), ("frames", 4)):
        ap.add_argument(f"--{name}", type=int, default=default)
    a = ap.parse_args()
    error, weights, ms = run(a.format, a.streams, a.height, a.width, a.channels, a.hidden, a.frames)
    print(f"{a.format}: weights {weights:.3f} off, planes {error:.3f} off after {a.frames} frames, {ms * 1e3:.1f} us a frame "
          f"of {a.streams} streams of {a.width} x {a.height} x {a.channels}")


if __name__ == "__main__":
    main()
