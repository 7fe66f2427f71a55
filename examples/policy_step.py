"""Policy-gradient steps of a small model built of mHC layers, on one GPU.

Each block is MHCRewire around a feed-forward pair of FusedLinear layers; the loss is the clipped policy loss with a KL
term on the head's logits; AdamW updates the mHC parameters (float32) and the weights (bfloat16 with float32 masters,
states in 8 bits where they are large).  The task is synthetic: an action is rewarded if it is the token's successor.

    python examples/policy_step.py --steps 20
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch
import torch.nn as nn

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "mhc-mlx_amd"))

from mhc_mlx_amd import AdamW, FusedLinear, MHCRewire, policy_loss  # noqa: E402


class Policy(nn.Module):
    def __init__(self, vocab: int, width: int, blocks: int, streams: int, dtype=torch.bfloat16, device="cuda"):
        super().__init__()
        kw = dict(device=device, dtype=dtype)
        self.embed = nn.Embedding(vocab, width, **kw)
        self.blocks = nn.ModuleList(
            MHCRewire(nn.Sequential(FusedLinear(width, 2 * width, activation="gelu", **kw), FusedLinear(2 * width, width, **kw)),
                      dims=width, n=streams, return_dtype=dtype, identity_init=False, device=device)
            for _ in range(blocks))
        self.head = FusedLinear(width, vocab, bias=False, **kw)

    def forward(self, tokens: torch.Tensor) -> torch.Tensor:
        x = self.embed(tokens)
        for block in self.blocks:
            x = block(x)
        return self.head(x)


def logp_of(logits: torch.Tensor, actions: torch.Tensor) -> torch.Tensor:
    return torch.log_softmax(logits.float(), -1).gather(-1, actions[..., None])[..., 0]


def train(steps: int = 20, tokens: int = 2048, vocab: int = 512, width: int = 256, blocks: int = 2, streams: int = 4, lr: float = 3e-3,
          seed: int = 0, say=print) -> list[float]:
    """Mean reward of the actions sampled at each step."""
    torch.manual_seed(seed)
    model = Policy(vocab, width, blocks, streams)
    opt = AdamW(model.parameters(), lr=lr, betas=(0.9, 0.95), weight_decay=0.0, state_bits=8)
    first = Policy(vocab, width, blocks, streams)
    first.load_state_dict(model.state_dict())  # the reference policy of the KL term
    rewards = []
    for step in range(steps):
        state = torch.randint(0, vocab, (tokens,), device="cuda")
        with torch.no_grad():  # act, half of the tokens on the rewarded action, so that there is something to learn from
            logits = model(state)
            actions = torch.multinomial(torch.softmax(logits.float(), -1), 1)[:, 0]
            target = (state + 1) % vocab
            actions = torch.where(torch.rand(tokens, device="cuda") < 0.5, target, actions)
            old, ref = logp_of(logits, actions), logp_of(first(state), actions)
            reward = (actions == target).float()
            sampled = (torch.softmax(logits.float(), -1).gather(1, target[:, None])).mean()  # chance of the rewarded action
            # some stand for padding; an imposed action that the policy all but excludes would be nearly all of the KL
            # term, whose estimate exp(ref - lp) takes actions to be the policy's own
            mask = (torch.rand(tokens, device="cuda") < 0.9) & (old > -10.0)
        for _ in range(2):  # two passes over the same actions: the second is off the acting policy, and clipped
            opt.zero_grad(set_to_none=True)
            loss, _ = policy_loss(model(state), actions, old, reward - reward.mean(), ref_logp=ref, mask=mask, kl_coef=0.001)
            loss.backward()
            opt.step()
        rewards.append(float(sampled))
        say(f"step {step:3d}  loss {float(loss.detach()):8.4f}  chance of the rewarded action {rewards[-1]:.4f}")
    return rewards


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--tokens", type=int, default=2048)
    ap.add_argument("--vocab", type=int, default=512)
    ap.add_argument("--width", type=int, default=256)
    ap.add_argument("--blocks", type=int, default=2)
    ap.add_argument("--streams", type=int, default=4)
    ap.add_argument("--lr", type=float, default=3e-3)
    args = ap.parse_args()
    if not torch.cuda.is_available():
        raise SystemExit("policy_step needs a GPU")
    train(**vars(args))


if __name__ == "__main__":
    main()
