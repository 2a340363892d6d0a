"""Rotary frequencies from their formulas in 70 decimal digits (nothing of the library is used)."""

import math
from decimal import Decimal, localcontext

PI = Decimal("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899")


def turns_per_position(rotary_dim, theta, scaling=None):
    """Each pair's turns per position, as Decimals."""
    s = scaling or {"type": "none"}
    kind, one = s["type"], Decimal(1)
    with localcontext() as ctx:
        ctx.prec = 70
        base = Decimal(theta)
        f = Decimal(s.get("factor", 1.0))
        if kind == "ntk":
            base *= (Decimal(rotary_dim) / Decimal(rotary_dim - 2) * f.ln()).exp()
        if kind == "yarn":
            def dim(turns):
                return rotary_dim * math.log(s["original_max_position"] / (turns * 2 * math.pi)) / (2 * math.log(theta))
            lo = max(math.floor(dim(s.get("beta_fast", 32.0))), 0)
            hi = min(math.ceil(dim(s.get("beta_slow", 1.0))), rotary_dim - 1)
        out = []
        for i in range(rotary_dim // 2):
            r = (-Decimal(2 * i) / rotary_dim * base.ln()).exp()
            if kind == "linear":
                r /= f
            elif kind == "yarn":
                ramp = min(max((i - Decimal(lo)) / max(Decimal(hi - lo), Decimal(0.001)), Decimal(0)), one)
                r = r / f * ramp + r * (one - ramp)
            elif kind == "llama3":
                low, high = Decimal(s["low_freq_factor"]), Decimal(s["high_freq_factor"])
                t = min(max((s["original_max_position"] * r / (2 * PI) - low) / (high - low), Decimal(0)), one)
                r = (one - t) * r / f + t * r
            elif kind == "divisors":
                r /= Decimal(s["divisors"][i])
            out.append(r / (2 * PI))
        return out


def fraction_of_a_turn(position, turns):
    """position * turns without its whole turns, nearest to zero, as a float."""
    with localcontext() as ctx:
        ctx.prec = 70
        x = position * turns
        return float(x - x.to_integral_value())
