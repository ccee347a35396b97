"""Drawn tokens on fp32 weights: how often they decide otherwise than doubles do, and how many rows a bound of their error
leaves open (csrc/rules.hip sums doubles).  Plain torch on the GPU; python tools/lab/draw_in_fp32.py"""
import torch, math
dev = "cuda"; U = 2.0 ** -24
print("512 x 131072 logits a batch (bf16, N(0, 2.5)) + an fp32 bias (N(0, 1)), 12 batches, sums in double")
for T0, T1 in ((0.75, 0.75), (1.0, 1.0), (1.5, 1.5), (0.5, 1.5)):
    diff = [0, 0, 0]; flag = [0, 0]; rows = 0
    for seed in range(12):
        g = torch.Generator(device=dev); g.manual_seed(seed)
        x64 = (torch.randn(512, 131072, generator=g, device=dev) * 2.5).bfloat16().double() + torch.randn(131072, generator=g, device=dev).double()
        u = torch.rand(512, 1, generator=g, device=dev).double()
        t = T0 + (T1 - T0) * torch.rand(512, 1, generator=g, device=dev)
        w64 = ((x64 - x64.amax(1, keepdim=True)) / t.double()).exp()
        r64 = w64.cumsum(1); d64 = (r64 > u * r64[:, -1:]).to(torch.uint8).argmax(1)
        del w64, r64
        x = x64.float(); del x64
        m = x.amax(1, keepdim=True)
        a32 = (x - m) * (1.4426950408889634 / t)
        w32 = torch.exp2(a32)
        top = x.abs() * (1.0 / t)
        r32 = w32.double().cumsum(1); e32 = u * r32[:, -1:]
        d32 = (r32 > e32).to(torch.uint8).argmax(1)
        diff[0] += int((d32 != d64).sum())
        f = w32.cumsum(1); diff[1] += int(((f > u.float() * f[:, -1:]).to(torch.uint8).argmax(1) != d64).sum()); del f
        at = d32[:, None]
        for k, rel in enumerate((U * (math.log(2) * 3 * a32.abs() + 2), U * (math.log(2) * 3 * a32.abs() + 2 + top))):
            err = (w32 * rel).double().cumsum(1)
            lim = err + u * err[:, -1:]
            low = torch.where(at > 0, r32.gather(1, (at - 1).clamp(min=0)), torch.zeros_like(e32))
            o = (r32.gather(1, at) - e32 <= lim.gather(1, at)) | ((at > 0) & (e32 - low <= lim.gather(1, (at - 1).clamp(min=0))))
            flag[k] += int(o.sum()); del err, lim
        rows += 512
        del x, a32, w32, r32, top
    print("T %.2f .. %.2f, %d rows: decided otherwise by fp32 weights of values rounded to fp32 %.2f in a thousand, with fp32 sums as well %.2f; "
          "left open by a bound of the weights' error %.1f %%, with the values' rounding %.1f %%" % (T0, T1, rows, 1e3 * diff[0] / rows, 1e3 * diff[1] / rows, 100.0 * flag[0] / rows, 100.0 * flag[1] / rows), flush=True)
