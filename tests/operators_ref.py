"""
The operators of simurlacra_amd.operators written out in float64, row by row, with their gradients by the chain rule.

With `mag=True` every term is taken by its magnitude, which gives for each result the sum of the magnitudes of everything that is
added up in it: M.  A computation in a type of unit roundoff u whose longest chain to a result has n roundings is off by
at most about n u M.
"""
import torch


def _f(t):
    return None if t is None else t.detach().cpu().double()


def _id(mag):
    return torch.abs if mag else (lambda v: v)


def linear(x, w, b, off, nonlin=None, dy=None, mag=False):
    x, w, b, dy = _f(x), _f(w), _f(b), _f(dy)
    off = [0] + [int(o) for o in off[1:]]
    m = _id(mag)
    G, N, K = w.shape
    pre = torch.zeros(x.shape[0], N, dtype=torch.float64)
    absolute = torch.zeros_like(pre)
    for g in range(G):
        r = slice(off[g], off[g + 1])
        pre[r] = x[r] @ w[g].t() + (0 if b is None else b[g])
        absolute[r] = x[r].abs() @ w[g].abs().t() + (0 if b is None else b[g].abs())
    f = {None: lambda v: v, 'tanh': torch.tanh, 'relu': torch.relu, 'sigmoid': torch.sigmoid}[nonlin]
    y = f(pre)
    y[off[G]:] = 0
    out = dict(y=absolute if mag else y)
    if dy is None:
        return out
    slope = {None: torch.ones_like(y), 'tanh': 1 - y*y, 'relu': (y > 0).double(), 'sigmoid': y*(1 - y)}[nonlin]
    dp = m(dy*slope)
    dx, dw, db = torch.zeros_like(x), torch.zeros_like(w), torch.zeros(G, N, dtype=torch.float64)
    for g in range(G):
        r = slice(off[g], off[g + 1])
        dx[r], dw[g], db[g] = dp[r] @ m(w[g]), dp[r].t() @ m(x[r]), dp[r].sum(0)
    out.update(dx=dx, dw=dw, db=db)
    return out


def policy_of(groups, S, P):
    pol = [0]*S
    if groups is not None:
        for p in range(P):
            for s in range(int(groups[p]) if p else 0, int(groups[p + 1]) if p + 1 < P else S):
                pol[s] = p
    return pol


def conv(x, w, b, off, groups=None, state=None, silu=True, dy=None, dlast=None, mag=False):
    x, w, b, state, dy, dlast = (_f(t) for t in (x, w, b, state, dy, dlast))
    off = [0] + [int(o) for o in off[1:]]
    m = _id(mag)
    (R, D), (P, _, K), S = x.shape, w.shape, len(off) - 1
    pol = policy_of(groups, S, P)
    y, last = torch.zeros(R, D, dtype=torch.float64), torch.zeros(S, D, K - 1, dtype=torch.float64)
    dx, dw, db = torch.zeros_like(x), torch.zeros_like(w), torch.zeros(P, D, dtype=torch.float64)
    ds = torch.zeros(S, D, K - 1, dtype=torch.float64)
    for s in range(S):
        p, a, e = pol[s], off[s], off[s + 1]
        st = torch.zeros(D, K - 1, dtype=torch.float64) if state is None else state[s]
        line = torch.cat([st.t(), x[a:e]])                    # [K - 1 + L, D]
        dline = torch.zeros_like(line)
        for t in range(e - a):
            win = line[t:t + K]                               # [K, D]
            pre = (w[p].t()*win).sum(0) + (0 if b is None else b[p])
            sig = torch.sigmoid(pre)
            y[a + t] = (w[p].t()*win).abs().sum(0) + (0 if b is None else b[p].abs()) if mag else (pre*sig if silu else pre)
            if dy is not None:
                slope = sig*(1 + pre*(1 - sig)) if silu else torch.ones_like(pre)
                if mag and silu:                              # the error of pre moves the slope by at most half of it
                    slope = slope.abs() + (w[p].t()*win).abs().sum(0) + (0 if b is None else b[p].abs())
                dp = m(dy[a + t]*slope)
                dline[t:t + K] += dp*m(w[p].t())
                dw[p] += (dp*m(win)).t()
                db[p] += dp
        last[s] = line[e - a:].t()
        if dlast is not None:
            dline[e - a:] += m(dlast[s].t())
        ds[s], dx[a:e] = dline[:K - 1].t(), dline[K - 1:]
    out = dict(y=y, last=last)
    if dy is not None:
        out.update(dx=dx, dw=dw, db=db, dstate=ds)
    return out


def scan(u, delta, A, B, C, D, z, bias, off, groups=None, state=None, dy=None, dlast=None, mag=False):
    u, delta, A, B, C, D, z, bias, state, dy, dlast = (_f(t) for t in (u, delta, A, B, C, D, z, bias, state, dy, dlast))
    off = [0] + [int(o) for o in off[1:]]
    m = _id(mag)
    (R, ch), (P, _, N), S = u.shape, A.shape, len(off) - 1
    pol = policy_of(groups, S, P)
    y, last = torch.zeros(R, ch, dtype=torch.float64), torch.zeros(S, ch, N, dtype=torch.float64)
    g = {k: torch.zeros_like(v) for k, v in dict(du=u, ddelta=u, dz=u, dB=B, dC=C, dA=A, dstate=last).items()}
    g.update(dD=torch.zeros(P, ch, dtype=torch.float64), dbias=torch.zeros(P, ch, dtype=torch.float64))
    for s in range(S):
        p, a, e = pol[s], off[s], off[s + 1]
        h = torch.zeros(ch, N, dtype=torch.float64) if state is None else m(state[s])
        skip = torch.zeros(ch, dtype=torch.float64) if D is None else m(D[p])
        raw = delta[a:e] + (0 if bias is None else bias[p])
        dt = torch.logaddexp(raw, torch.zeros_like(raw))
        gate = torch.ones_like(raw) if z is None else m(z[a:e]*torch.sigmoid(z[a:e]))
        hs, y0 = [h], []
        for t in range(e - a):
            h = torch.exp(dt[t][:, None]*A[p])*h + (dt[t]*m(u[a + t]))[:, None]*m(B[a + t])
            hs.append(h)
            y0.append((h*m(C[a + t])).sum(1) + skip*m(u[a + t]))
            y[a + t] = y0[t]*gate[t]
        last[s] = h
        if dy is None:
            continue
        G = torch.zeros(ch, N, dtype=torch.float64) if dlast is None else m(dlast[s])
        for t in reversed(range(e - a)):
            r, d = a + t, m(dy[a + t])*gate[t]
            av = torch.exp(dt[t][:, None]*A[p])
            gt = d[:, None]*m(C[r]) + G
            G = av*gt
            gah = G*hs[t]
            g['dC'][r] = (d[:, None]*hs[t + 1]).sum(0)
            g['dB'][r] = (gt*(dt[t]*m(u[r]))[:, None]).sum(0)
            gb = (gt*m(B[r])).sum(1)
            ddt = (gah*m(A[p])).sum(1) + gb*m(u[r])
            g['ddelta'][r] = ddt*torch.sigmoid(raw[t])
            g['du'][r] = dt[t]*gb + skip*d
            g['dA'][p] += gah*dt[t][:, None]
            g['dD'][p] += d*m(u[r])
            g['dbias'][p] += g['ddelta'][r]
            if z is not None:
                sg = torch.sigmoid(z[r])
                g['dz'][r] = m(dy[r])*y0[t]*m(sg*(1 + z[r]*(1 - sg))) if not mag else m(dy[r])*y0[t]*(sg*(1 + z[r].abs()))
        g['dstate'][s] = G
    out = dict(y=y, last=last)
    if dy is not None:
        out.update(g)
    return out
