"""Oracle of the linear cross entropy (test infrastructure only; see ``oracle/__init__.py``), in 64 bits."""
import torch


def forward(x, w, target, ignore_index=-100):
    """(loss, lse, logits) in fp64; targets outside the vocabulary count as ignored."""
    z = x.double() @ w.double().t()
    lse = torch.logsumexp(z, dim=1)
    live = (target != ignore_index) & (target >= 0) & (target < w.shape[0])
    at = torch.where(live, target, 0).long()
    return torch.where(live, lse - z[torch.arange(len(z)), at], 0.0), lse, z


def d_logits(x, w, target, d_loss, ignore_index=-100):
    """Gradient of sum(d_loss * loss) with respect to the logits, in fp64."""
    _, lse, z = forward(x, w, target, ignore_index)
    live = (target != ignore_index) & (target >= 0) & (target < w.shape[0])
    p = torch.exp(z - lse.unsqueeze(1))
    p[torch.arange(len(z)), torch.where(live, target, 0).long()] -= 1
    return p * torch.where(live, d_loss.double(), 0.0).unsqueeze(1)
