"""The training loop's autograd path with a foreign model, on the CPU."""
import torch


class _Seen(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, seen):
        ctx.seen = seen
        return x.clone()

    @staticmethod
    def backward(ctx, g):
        ctx.seen.append(torch._C._is_multithreading_enabled())
        return g, None


def test_the_loop_leaves_the_autograd_engines_setting_to_its_caller():
    import vae_amd
    seen, fc = [], torch.nn.Linear(4, 4)

    class Model(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.fc = fc

        def forward(self, x):
            y = _Seen.apply(self.fc(x), seen)
            return y, y, y

    loader = torch.utils.data.DataLoader(torch.randn(6, 4), batch_size=3)
    opt = torch.optim.SGD(fc.parameters(), lr=0.1)

    def epoch():
        seen.clear()
        vae_amd.train.train(Model(), loader, lambda y, t, mu, lv: ((y - t) ** 2).sum(), opt, "cpu", 1)
        return list(seen)

    assert epoch() == [True, True]
    with torch.autograd.set_multithreading_enabled(False):
        assert epoch() == [False, False]
