"""A layer that mixes a sequence, trained and then served with the library's plans.

The layer is x + W_o attention(W_q n, W_k n, W_v n) with n = norm(x): layer norm
and linear attention with a decay for each head, forward and backward. What it
learns is a fixed causal filter of the sequence, decay^t, that a zero-padded
convolution plan applies to its inputs: the same mixing by a filter given
beforehand, where the layer finds it. Served, the trained layer takes a prompt
in one call and then token by token, from the state the prompt left.

  python3 examples/sequence_mixer.py [steps]
"""
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vkfft-rs_amd"))
import vkfft_amd as vk  # noqa: E402

BATCH, TOKENS, WIDTH, HEADS, DIM = 4, 300, 64, 4, 32
DECAYS = [0.5, 0.875, 0.96875, 0.9921875]
FILTER = 0.95


class Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, plan, x, weight, bias):
        y, stats = torch.empty_like(x), x.new_empty(x.shape[0], 2)
        plan.forward_tensors(x, weight, bias, y, stats)
        ctx.plan = plan
        ctx.save_for_backward(x, weight, stats)
        return y

    @staticmethod
    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        dx, dweight, dbias = torch.empty_like(x), torch.empty_like(weight), torch.empty_like(weight)
        ctx.plan.backward_tensors(x, weight, stats, dy.contiguous(), dx, dweight, dbias)
        return None, dx, dweight, dbias


class Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, plan, q, k, v):
        out = torch.empty_like(v)
        plan.forward_tensors(q, k, v, out)
        ctx.plan = plan
        ctx.save_for_backward(q, k, v)
        return out

    @staticmethod
    def backward(ctx, dout):
        q, k, v = ctx.saved_tensors
        dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
        ctx.plan.backward_tensors(q, k, v, dout.contiguous(), dq, dk, dv)
        return None, dq, dk, dv


class Mixer(torch.nn.Module):
    def __init__(self, ctx):
        super().__init__()
        self.weight = torch.nn.Parameter(torch.ones(WIDTH))
        self.bias = torch.nn.Parameter(torch.zeros(WIDTH))
        self.qkv = torch.nn.Linear(WIDTH, 3 * HEADS * DIM)
        self.out = torch.nn.Linear(HEADS * DIM, WIDTH)
        self.norm = vk.LayerNormPlan(ctx, vk.LayerNormConfig.new(WIDTH))
        config = vk.LinearAttentionConfig.new(HEADS, DIM, DIM).with_decay(DECAYS).with_capacity(BATCH, TOKENS).with_gradient()
        self.attention = vk.LinearAttentionPlan(ctx, config)

    def _heads(self, x, norm):
        b, t = x.shape[:2]
        n = norm(x.reshape(b * t, WIDTH))
        return self.qkv(n).view(b, t, 3, HEADS, DIM).unbind(2)  # strided views: the plan takes them as they are

    def forward(self, x):
        q, k, v = self._heads(x, lambda r: Norm.apply(self.norm, r, self.weight, self.bias))
        return x + self.out(Attention.apply(self.attention, q, k, v).flatten(2))

    @torch.no_grad()
    def serve(self, x, state):
        """Any number of new tokens of each sequence; the state is updated in place."""
        def norm(rows):
            y = torch.empty_like(rows)
            self.norm.forward_tensors(rows, self.weight, self.bias, y)
            return y

        q, k, v = self._heads(x, norm)
        out = torch.empty(v.shape, device=v.device)
        self.attention.forward_tensors(q, k, v, out, state_in=state, state_out=state)
        return x + self.out(out.flatten(2))


def filtered(ctx, x):
    """Every channel of [batch][token][channel] through the causal filter FILTER^t: one convolution plan over rows of
    twice the length, the second half zeros."""
    b, t, c = x.shape
    n = 1024
    h = np.zeros(n)
    h[:t] = FILTER ** np.arange(t)
    config = vk.FftConfig.new([n]).with_batch_count(b * c).with_convolution(True)
    rows = np.zeros((b * c, n), np.complex64)
    rows[:, :t] = x.transpose(1, 2).reshape(b * c, t).cpu().numpy()
    y = ctx.execute_convolution(vk.ConvolutionIr.build(config, np.fft.fft(h).astype(np.complex64)), rows)
    y = y.reshape(b, c, n)[:, :, :t].real
    return torch.from_numpy(np.ascontiguousarray(y.transpose(0, 2, 1))).to(x.device)


def main(steps=200):
    torch.manual_seed(1)
    torch.cuda.init()  # torch's HIP runtime is the one the library binds to
    ctx = vk.HipExecutionContext(0)
    layer = Mixer(ctx).cuda()
    optimizer = torch.optim.Adam(layer.parameters(), 1e-2)
    losses = []
    for step in range(steps):
        x = torch.randn(BATCH, TOKENS, WIDTH, device="cuda")
        want = x + 0.3 * filtered(ctx, x)
        loss = (layer(x) - want).square().mean()
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.item())
        if step % 20 == 0 or step == steps - 1:
            print(f"step {step}: loss {losses[-1]:.4f}", flush=True)

    x = torch.randn(BATCH, TOKENS, WIDTH, device="cuda")
    with torch.no_grad():
        whole = layer(x)
    state = torch.zeros(BATCH, HEADS, DIM, DIM, device="cuda")
    served = [layer.serve(x[:, :200], state)] + [layer.serve(x[:, t:t + 1], state) for t in range(200, TOKENS)]
    apart = ((torch.cat(served, 1) - whole).norm() / whole.norm()).item()
    print(f"prompt of 200 tokens, then {TOKENS - 200} one by one: {apart:.1e} from the whole sequence at once", flush=True)
    ctx.close()
    return losses, apart


if __name__ == "__main__":
    main(int(sys.argv[1]) if len(sys.argv) > 1 else 200)
