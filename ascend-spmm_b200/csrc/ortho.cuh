// Shared by the two forms of the orthogonalised update (ortho.cu, ortho_small.cu).
#pragma once

#include <algorithm>
#include <cmath>

namespace spmmb {

// Stored fp16 operand = value * scale.  With the usual coefficients singular
// values are of order one, so a matrix's elements are of order 1 / sqrt(size):
// the scales keep them out of fp16's subnormals and leave a factor of 100
// below its maximum.
constexpr float kScaleX = 512.f, kScaleG = 256.f, kScaleP = 256.f;
// What a stored operand may reach: half of fp16's maximum.
constexpr double kMostStored = 32768.0;

// `scale`, or the power of two below it that keeps values up to `most` in
// fp16's range.  No element of a matrix is larger than its largest singular value.
inline double scale_for(double scale, double most)
{
    if (!(most * scale > kMostStored)) return scale;
    return std::exp2(std::floor(std::log2(kMostStored / std::min(most, 0x1p100))));
}

// Bounds over the singular values s in [0, reach] that a step can meet, with
// u = s^2 an eigenvalue of G (host, 64 bits).  They start in [0, 1]; with the
// default coefficients they stay below 1.2024.
struct OrthoReach {
    double reach = 1.0;
    double a, b, c;
    OrthoReach(double a, double b, double c) : a(a), b(b), c(c) {}
    // The largest |b u + c u^2| and |a + b u + c u^2|, at an end or where b + 2 c u is zero.
    double poly() const { return extreme(0.0); }
    double factor() const { return extreme(a); }
    // The largest factor of an error of G's eigenvalues in a step G <- T G T,
    // T = a + b u + c u^2: |d (u T^2) / du| = |T (a + 3 b u + 5 c u^2)|, sampled.
    double growth() const
    {
        double most = 0.0;
        const double step = reach * reach / 32;
        for (int i = 0; i <= 32; ++i) {
            const double u = step * i;
            most = std::max(most, std::fabs((a + u * (b + u * c)) * (a + u * (3 * b + 5 * u * c))));
        }
        return most;
    }
    // To the next step: the largest |s T(s^2)|, at an end or where its derivative a + 3 b u + 5 c u^2 is zero.
    void step()
    {
        double most = value(reach * reach);
        const double disc = 9 * b * b - 20 * a * c;
        if (c != 0.0 && disc >= 0.0)
            for (const double sign : {-1.0, 1.0}) most = std::max(most, value((-3 * b + sign * std::sqrt(disc)) / (10 * c)));
        else if (c == 0.0 && b != 0.0)
            most = std::max(most, value(-a / (3 * b)));
        reach = most;
    }

private:
    double extreme(double t) const
    {
        const double end = reach * reach, middle = c != 0.0 ? -b / (2 * c) : 0.0;
        double most = std::max(std::fabs(t), std::fabs(t + end * (b + end * c)));
        if (middle > 0.0 && middle < end) most = std::max(most, std::fabs(t + middle * (b + middle * c)));
        return most;
    }
    double value(double u) const
    {
        return u >= 0.0 && u <= reach * reach ? std::sqrt(u) * std::fabs(a + u * (b + u * c)) : 0.0;
    }
};

}  // namespace spmmb
