"""How far products of fp32 vectors with 4-bit weights may be off, on the average over their results."""
import math

U = 2.0 ** -24


def fp32_rms_bound(group, n_groups, zeros):
  """Bound of rms(error) / rms(result) for vectors of independent elements of mean 0 and uniform codes (and zero points).

  A group's result is s (sum c x - z sum x).  With elements of rms a and codes of rms 8.8 (0 .. 15) a partial sum of j terms c x has
  rms 8.8 a sqrt(j).  A group has 3 g terms (x is three exact parts); were every one rounded by itself, each rounding had rms U / sqrt(3) of
  the partial sum, and independent ones add up to sqrt(3 sum_j (U^2 / 3) 77.5 a^2 j) = 8.8 a U g / sqrt(2).  The sums z x (8 x without
  zero points) are the same with z's rms.  The result has rms d a sqrt(g), d^2 the mean of (c - z)^2: 42.5 for two uniform numbers 0 .. 15, 21.5
  for z = 8.  So the error of a group is sqrt(77.5 + z^2) / d U sqrt(g / 2) of it, and errors and results of groups add up alike.  Taking
  the offset off, scaling and rounding once are three roundings, a sum of n groups at most U sqrt(n / 6) more."""
  z2, d2 = (77.5, 42.5) if zeros else (64.0, 21.5)
  return U * (math.sqrt((77.5 + z2) / d2 * group / 2) + 3 + math.sqrt(n_groups / 6))


def rms_error(got, want):
  """rms(got - want) / rms(want) in 64 bits."""
  return ((got.double() - want).square().mean().sqrt() / want.square().mean().sqrt()).item()
