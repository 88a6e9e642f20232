"""An INT8 cross-attention layer over an image encoder's features, from the operators of
spinnv2_b200.transformer: what a decoder that reads images (captions, questions, object queries) runs next to
the graph runtime.

  encoder      a ResNet package of this runtime whose features (the last convolution's output) are an output
  keys/values  one int8 product per image, kept for all of the decoder's steps
  a step       residual + norm -> codes -> queries -> cross attention -> codes -> output product

`python -m spinnv2_b200.decoder` runs ResNet-50 on a batch of synthetic images, a prompt and a few
single-token steps of two layers with random weights, and prints the time of a step.
"""

from __future__ import annotations

import argparse

import numpy as np
import torch

from . import transformer as T


class CrossAttentionLayer:
    """norm -> queries -> attention over an encoder's states -> output product, weights in int8.

    width: of the decoder's stream; encoder_width: channels of the features; kv_heads: key heads, each
    shared by heads / kv_heads query heads.  weights: float tensors norm [width], q [heads * head_width,
    width], kv [2 * kv_heads * head_width, encoder_width], out [width, heads * head_width]; their codes
    are laid out once, here.
    """

    def __init__(self, weights: dict, heads: int, kv_heads: int, *, eps: float = 1e-6) -> None:
        self.heads, self.kv_heads, self.eps = heads, kv_heads, eps
        self.norm = weights["norm"]
        self.head_width = weights["q"].shape[0] // heads
        self.q, self.kv, self.out = (T.quantize_rows_i8(weights[n]) for n in ("q", "kv", "out"))

    @classmethod
    def random(cls, width: int, encoder_width: int, heads: int, kv_heads: int, head_width: int, *,
               dtype=torch.bfloat16, seed: int = 0, device="cuda") -> "CrossAttentionLayer":
        g = torch.Generator(device=device)
        g.manual_seed(seed)

        def matrix(n: int, k: int) -> torch.Tensor:
            return (torch.randn(n, k, generator=g, device=device) * k**-0.5).to(dtype)

        norm = (1.0 + 0.1 * torch.randn(width, generator=g, device=device)).to(dtype)
        return cls({"norm": norm, "q": matrix(heads * head_width, width),
                    "kv": matrix(2 * kv_heads * head_width, encoder_width),
                    "out": matrix(width, heads * head_width)}, heads, kv_heads)

    def states(self, features: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """Keys and values [batch, positions, kv_heads, head_width] of features [batch, positions,
        encoder_width] (any of the operators' types): once per image."""
        kv = T.linear_i8(*T.quantize_rows_i8(features), *self.kv, dtype=self.norm.dtype)
        kv = kv.view(*features.shape[:2], 2, self.kv_heads, self.head_width)
        return kv[:, :, 0], kv[:, :, 1]

    def step(self, x: torch.Tensor, residual: torch.Tensor | None, states, *, lengths=None,
             key_mask=None) -> tuple[torch.Tensor, torch.Tensor]:
        """(y, stream) for tokens x [batch, tokens, width] and the residual stream so far: stream = x +
        residual, y = what this layer adds to it.  The next layer's step takes (y, stream)."""
        codes, scale, stream = T.rms_norm_i8(x, self.norm, residual, eps=self.eps)
        q = T.linear_i8(codes, scale, *self.q, dtype=x.dtype)
        attended = T.cross_attention(q.view(*x.shape[:2], self.heads, self.head_width), *states, lengths=lengths,
                                     key_mask=key_mask)
        y = T.linear_i8(*T.quantize_rows_i8(attended.flatten(2)), *self.out, dtype=x.dtype)
        return y, stream


def encoder_package(config: str = "resnet50", batch: int = 1) -> bytes:
    """The config's `cuda_b200` package with its features as a second output."""
    from .compiler import builders, pipeline
    from .compiler.ir import ROLE_OUTPUT

    graph = pipeline.fuse(builders.build_config(config, batch))
    pool = next(n for n in graph.nodes if n.op_type == "ReduceMean")
    graph.tensors[pool.inputs[0]].role = ROLE_OUTPUT
    graph.outputs = [*graph.outputs, pool.inputs[0]]
    return pipeline.package(graph, "cuda_b200")


class ImageEncoder:
    """Features of images on the device, by the graph runtime.

    The runtime writes one buffer on a stream of its own; `free` marks where torch's work on that buffer ends,
    and each run waits for it.
    """

    def __init__(self, config: str = "resnet50", batch: int = 1, *, device: int = 0) -> None:
        from .runtime import Runtime

        self.rt = Runtime(encoder_package(config, batch), device=device)
        shape = self.rt.package.outputs[1].shape  # [batch, channels, height, width]
        self.features = torch.empty(tuple(shape), device=f"cuda:{device}")
        self.rt.bind_output(1, self.features.data_ptr())  # written in place, no copy
        self.stream = torch.cuda.ExternalStream(self.rt.stream(), device=self.features.device)
        self.free = torch.cuda.Event()
        # Work that is queued may still use the block that the buffer lies in.
        self.free.record(torch.cuda.current_stream(self.features.device))

    def __call__(self, images: np.ndarray) -> torch.Tensor:
        """[batch, positions, channels] float32 of images [batch, 3, 224, 224], a tensor of its own, on
        torch's current stream."""
        self.rt.set_input(0, images)
        self.stream.wait_event(self.free)
        self.rt.run()  # returns when the features are written
        answer = self.features.flatten(2).transpose(1, 2).clone(memory_format=torch.contiguous_format)
        self.free.record(torch.cuda.current_stream(self.features.device))
        return answer

    def close(self) -> None:
        self.rt.close()


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--batch", type=int, default=4)
    ap.add_argument("--prompt", type=int, default=12)
    ap.add_argument("--steps", type=int, default=8)
    a = ap.parse_args()
    encoder = ImageEncoder("resnet50", a.batch)
    images = np.random.default_rng(0).standard_normal((a.batch, 3, 224, 224), dtype=np.float32)
    features = encoder(images)
    layers = [CrossAttentionLayer.random(1024, features.shape[2], 16, 4, 64, seed=i) for i in range(2)]
    states = [layer.states(features) for layer in layers]
    g = torch.Generator(device="cuda")
    g.manual_seed(1)

    def run(tokens: int) -> torch.Tensor:
        y = torch.randn(a.batch, tokens, 1024, generator=g, device="cuda").bfloat16()
        stream = None
        for layer, kv in zip(layers, states):
            y, stream = layer.step(y, stream, kv)
        return stream + y

    out = run(a.prompt)
    print(f"features {tuple(features.shape)}, prompt {tuple(out.shape)}, |out| {out.float().abs().mean():.3f}")
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    run(1)
    start.record()
    for _ in range(a.steps):
        out = run(1)
    end.record()
    end.synchronize()
    T.check()
    print(f"{a.steps} steps of {len(layers)} layers: {start.elapsed_time(end) / a.steps * 1e3:.1f} us a step, "
          f"out {tuple(out.shape)}, |out| {out.float().abs().mean():.3f}")
    encoder.close()


if __name__ == "__main__":
    main()
