// sas_exp.h - the exponential of sums of many masses, table-driven in double
// precision, shared by the verify and the filtered sampling kernels (gfx950).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "sas_device.h"

namespace sas {
namespace {

typedef double f64x2 __attribute__((ext_vector_type(2)));

// 2^(j / 64), j = 0 .. 63: the nearest double and the nearest double to what
// it leaves (computed with 80 decimal digits).
constexpr int kExpTab = 64;
__device__ const f64x2 kExp2Tab[kExpTab] = {
    {0x1.p+0, 0.0}, {0x1.02c9a3e778061p+0, -0x1.19083535b085dp-56},
    {0x1.059b0d3158574p+0, 0x1.d73e2a475b465p-55}, {0x1.0874518759bc8p+0, 0x1.186be4bb284ffp-57},
    {0x1.0b5586cf9890fp+0, 0x1.8a62e4adc610bp-54}, {0x1.0e3ec32d3d1a2p+0, 0x1.03a1727c57b53p-59},
    {0x1.11301d0125b51p+0, -0x1.6c51039449b3ap-54}, {0x1.1429aaea92de0p+0, -0x1.32fbf9af1369ep-54},
    {0x1.172b83c7d517bp+0, -0x1.19041b9d78a76p-55}, {0x1.1a35beb6fcb75p+0, 0x1.e5b4c7b4968e4p-55},
    {0x1.1d4873168b9aap+0, 0x1.e016e00a2643cp-54}, {0x1.2063b88628cd6p+0, 0x1.dc775814a8495p-55},
    {0x1.2387a6e756238p+0, 0x1.9b07eb6c70573p-54}, {0x1.26b4565e27cddp+0, 0x1.2bd339940e9d9p-55},
    {0x1.29e9df51fdee1p+0, 0x1.612e8afad1255p-55}, {0x1.2d285a6e4030bp+0, 0x1.0024754db41d5p-54},
    {0x1.306fe0a31b715p+0, 0x1.6f46ad23182e4p-55}, {0x1.33c08b26416ffp+0, 0x1.32721843659a6p-54},
    {0x1.371a7373aa9cbp+0, -0x1.63aeabf42eae2p-54}, {0x1.3a7db34e59ff7p+0, -0x1.5e436d661f5e3p-56},
    {0x1.3dea64c123422p+0, 0x1.ada0911f09ebcp-55}, {0x1.4160a21f72e2ap+0, -0x1.ef3691c309278p-58},
    {0x1.44e086061892dp+0, 0x1.89b7a04ef80d0p-59}, {0x1.486a2b5c13cd0p+0, 0x1.3c1a3b69062f0p-56},
    {0x1.4bfdad5362a27p+0, 0x1.d4397afec42e2p-56}, {0x1.4f9b2769d2ca7p+0, -0x1.4b309d25957e3p-54},
    {0x1.5342b569d4f82p+0, -0x1.07abe1db13cadp-55}, {0x1.56f4736b527dap+0, 0x1.9bb2c011d93adp-54},
    {0x1.5ab07dd485429p+0, 0x1.6324c054647adp-54}, {0x1.5e76f15ad2148p+0, 0x1.ba6f93080e65ep-54},
    {0x1.6247eb03a5585p+0, -0x1.383c17e40b497p-54}, {0x1.6623882552225p+0, -0x1.bb60987591c34p-54},
    {0x1.6a09e667f3bcdp+0, -0x1.bdd3413b26456p-54}, {0x1.6dfb23c651a2fp+0, -0x1.bbe3a683c88abp-57},
    {0x1.71f75e8ec5f74p+0, -0x1.16e4786887a99p-55}, {0x1.75feb564267c9p+0, -0x1.0245957316dd3p-54},
    {0x1.7a11473eb0187p+0, -0x1.41577ee04992fp-55}, {0x1.7e2f336cf4e62p+0, 0x1.05d02ba15797ep-56},
    {0x1.82589994cce13p+0, -0x1.d4c1dd41532d8p-54}, {0x1.868d99b4492edp+0, -0x1.fc6f89bd4f6bap-54},
    {0x1.8ace5422aa0dbp+0, 0x1.6e9f156864b27p-54}, {0x1.8f1ae99157736p+0, 0x1.5cc13a2e3976cp-55},
    {0x1.93737b0cdc5e5p+0, -0x1.75fc781b57ebcp-57}, {0x1.97d829fde4e50p+0, -0x1.d185b7c1b85d1p-54},
    {0x1.9c49182a3f090p+0, 0x1.c7c46b071f2bep-56}, {0x1.a0c667b5de565p+0, -0x1.359495d1cd533p-54},
    {0x1.a5503b23e255dp+0, -0x1.d2f6edb8d41e1p-54}, {0x1.a9e6b5579fdbfp+0, 0x1.0fac90ef7fd31p-54},
    {0x1.ae89f995ad3adp+0, 0x1.7a1cd345dcc81p-54}, {0x1.b33a2b84f15fbp+0, -0x1.2805e3084d708p-57},
    {0x1.b7f76f2fb5e47p+0, -0x1.5584f7e54ac3bp-56}, {0x1.bcc1e904bc1d2p+0, 0x1.23dd07a2d9e84p-55},
    {0x1.c199bdd85529cp+0, 0x1.11065895048ddp-55}, {0x1.c67f12e57d14bp+0, 0x1.2884dff483cadp-54},
    {0x1.cb720dcef9069p+0, 0x1.503cbd1e949dbp-56}, {0x1.d072d4a07897cp+0, -0x1.cbc3743797a9cp-54},
    {0x1.d5818dcfba487p+0, 0x1.2ed02d75b3707p-55}, {0x1.da9e603db3285p+0, 0x1.c2300696db532p-54},
    {0x1.dfc97337b9b5fp+0, -0x1.1a5cd4f184b5cp-54}, {0x1.e502ee78b3ff6p+0, 0x1.39e8980a9cc8fp-55},
    {0x1.ea4afa2a490dap+0, -0x1.e9c23179c2893p-54}, {0x1.efa1bee615a27p+0, 0x1.dc7f486a4b6b0p-54},
    {0x1.f50765b6e4540p+0, 0x1.9d3e12dd8a18bp-54}, {0x1.fa7c1819e90d8p+0, 0x1.74853f3a5931ep-55},
};

// The table in LDS.  Every wave writes all of it (its lanes one entry each,
// the same values), so no barrier is needed before a wave reads it.
struct ExpTab {
  f64x2 e[kExpTab];
  __device__ __forceinline__ void fill(const f64x2 &mine) {
    e[threadIdx.x & (kExpTab - 1)] = mine;
    wave_lds_sync();
  }
};
__device__ __forceinline__ f64x2 exp_tab_entry() { return kExp2Tab[threadIdx.x & (kExpTab - 1)]; }

// e^x for sums of many weights, x <= 0, where the order of the additions
// already differs from a sequential loop (the table-driven method of P. T. P.
// Tang, ACM TOMS 15, 1989): within 0.82 ulp of the exact value (rms 0.296
// ulp, over 8 million x in [-700, 0] against 113-bit arithmetic;
// a degree-13 series without a table: 0.86 and 0.302), with no division.
// x = k ln2 / 64 + r, |r| <= ln2 / 128 (k by adding 1.5 * 2^52, ln2 / 64
// split in two parts, the high one with 21 zero bits), e^r - 1 by its Taylor
// series to degree 5 (truncation below 3.5e-17), times 2^((k mod 64) / 64)
// from the table, scaled by ldexp (subnormal results included).  x = -inf
// and NaN give 0; x > 0 is not used (but harmless).  The statistics pass
// without a mask is bound by these double operations: 15 here, 22 in the
// degree-13 series (32 x 5 positions of 151,936 ids: 106 -> 80 us a call), 17
// with 16 entries, whose reads never conflict (83 us).
__device__ __forceinline__ double exp_sum(double x, const ExpTab &tab) {
  const double magic = 6755399441055744.0;
  const double xc = fmax(x, -1100.0);
  const double kf = fma(xc, 0x1.71547652b82fep+6, magic);
  const int k = (int)(uint32_t)(uint64_t)__double_as_longlong(kf);
  const f64x2 T = tab.e[k & (kExpTab - 1)];
  const double kd = kf - magic;
  const double r = fma(-kd, 0x1.a39ef35793c76p-39, fma(-kd, 0x1.62e42fee00000p-7, xc));
  const double q = fma(fma(fma(r, 1.0 / 120.0, 1.0 / 24.0), r, 1.0 / 6.0), r, 0.5);
  const double p = fma(r * r, q, r);
  return __builtin_amdgcn_ldexp(T.x + fma(T.x, p, T.y), k >> 6);
}

}  // namespace
}  // namespace sas
