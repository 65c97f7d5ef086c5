// GENERATED by flashns_b200/codegen.py -- do not edit.

#pragma once

namespace flashns_b200 {

// v = d * d, dim 2
__device__ __forceinline__ void jet_square_2d3(const double* d, double* v) {
  v[0] = d[0] * d[0];
  v[1] = 2.0 * (d[0] * d[1]);
  v[2] = 2.0 * (d[0] * d[2]);
  v[3] = 2.0 * (d[0] * d[3]) + d[1] * d[1];
  v[4] = 2.0 * (d[0] * d[4]) + 2.0 * (d[1] * d[2]);
  v[5] = 2.0 * (d[0] * d[5]) + d[2] * d[2];
  v[6] = 2.0 * (d[0] * d[6]) + 2.0 * (d[1] * d[3]);
  v[7] = 2.0 * (d[0] * d[7]) + 2.0 * (d[1] * d[4]) + 2.0 * (d[2] * d[3]);
  v[8] = 2.0 * (d[0] * d[8]) + 2.0 * (d[1] * d[5]) + 2.0 * (d[2] * d[4]);
  v[9] = 2.0 * (d[0] * d[9]) + 2.0 * (d[2] * d[5]);
}

// out = a * b, dim 2
__device__ __forceinline__ void jet_mul_2d3(const double* a, const double* b, double* out) {
  out[0] = a[0] * b[0];
  out[1] = a[0] * b[1] + a[1] * b[0];
  out[2] = a[0] * b[2] + a[2] * b[0];
  out[3] = a[0] * b[3] + a[1] * b[1] + a[3] * b[0];
  out[4] = a[0] * b[4] + a[1] * b[2] + a[2] * b[1] + a[4] * b[0];
  out[5] = a[0] * b[5] + a[2] * b[2] + a[5] * b[0];
  out[6] = a[0] * b[6] + a[1] * b[3] + a[3] * b[1] + a[6] * b[0];
  out[7] = a[0] * b[7] + a[1] * b[4] + a[2] * b[3] + a[3] * b[2] + a[4] * b[1] + a[7] * b[0];
  out[8] = a[0] * b[8] + a[1] * b[5] + a[2] * b[4] + a[4] * b[2] + a[5] * b[1] + a[8] * b[0];
  out[9] = a[0] * b[9] + a[2] * b[5] + a[5] * b[2] + a[9] * b[0];
}

// adjoint of b -> a * b at s: out_k = sum_j a_j s_(j+k), dim 2
__device__ __forceinline__ void jet_corr_2d3(const double* a, const double* s, double* out) {
  out[0] = a[0] * s[0] + a[1] * s[1] + a[2] * s[2] + a[3] * s[3] + a[4] * s[4] + a[5] * s[5] + a[6] * s[6] + a[7] * s[7] + a[8] * s[8] + a[9] * s[9];
  out[1] = a[0] * s[1] + a[1] * s[3] + a[2] * s[4] + a[3] * s[6] + a[4] * s[7] + a[5] * s[8];
  out[2] = a[0] * s[2] + a[1] * s[4] + a[2] * s[5] + a[3] * s[7] + a[4] * s[8] + a[5] * s[9];
  out[3] = a[0] * s[3] + a[1] * s[6] + a[2] * s[7];
  out[4] = a[0] * s[4] + a[1] * s[7] + a[2] * s[8];
  out[5] = a[0] * s[5] + a[1] * s[8] + a[2] * s[9];
  out[6] = a[0] * s[6];
  out[7] = a[0] * s[7];
  out[8] = a[0] * s[8];
  out[9] = a[0] * s[9];
}

// out_k += sum_j a_j s_(j+k), dim 2
__device__ __forceinline__ void jet_corr_add_2d3(const double* a, const double* s, double* out) {
  out[0] += a[0] * s[0] + a[1] * s[1] + a[2] * s[2] + a[3] * s[3] + a[4] * s[4] + a[5] * s[5] + a[6] * s[6] + a[7] * s[7] + a[8] * s[8] + a[9] * s[9];
  out[1] += a[0] * s[1] + a[1] * s[3] + a[2] * s[4] + a[3] * s[6] + a[4] * s[7] + a[5] * s[8];
  out[2] += a[0] * s[2] + a[1] * s[4] + a[2] * s[5] + a[3] * s[7] + a[4] * s[8] + a[5] * s[9];
  out[3] += a[0] * s[3] + a[1] * s[6] + a[2] * s[7];
  out[4] += a[0] * s[4] + a[1] * s[7] + a[2] * s[8];
  out[5] += a[0] * s[5] + a[1] * s[8] + a[2] * s[9];
  out[6] += a[0] * s[6];
  out[7] += a[0] * s[7];
  out[8] += a[0] * s[8];
  out[9] += a[0] * s[9];
}

// r = v^(-1/2), v_0 > 0, dim 2
__device__ __forceinline__ void jet_rsqrt_2d3(const double* v, double* r) {
  const double r0 = 1.0 / sqrt(v[0]);
  const double w = r0 * r0;
  const double n1 = v[1] * w;
  const double n2 = v[2] * w;
  const double n3 = v[3] * w;
  const double n4 = v[4] * w;
  const double n5 = v[5] * w;
  const double n6 = v[6] * w;
  const double n7 = v[7] * w;
  const double n8 = v[8] * w;
  const double n9 = v[9] * w;
  const double s3 = n1 * n1;
  const double s4 = 2.0 * (n1 * n2);
  const double s5 = n2 * n2;
  const double s6 = 2.0 * (n1 * n3);
  const double s7 = 2.0 * (n1 * n4) + 2.0 * (n2 * n3);
  const double s8 = 2.0 * (n1 * n5) + 2.0 * (n2 * n4);
  const double s9 = 2.0 * (n2 * n5);
  r[0] = r0;
  r[1] = r0 * (-0.5 * n1);
  r[2] = r0 * (-0.5 * n2);
  r[3] = r0 * (-0.5 * n3 + 0.375 * s3);
  r[4] = r0 * (-0.5 * n4 + 0.375 * s4);
  r[5] = r0 * (-0.5 * n5 + 0.375 * s5);
  r[6] = r0 * (-0.5 * n6 + 0.375 * s6 - 0.3125 * (s3 * n1));
  r[7] = r0 * (-0.5 * n7 + 0.375 * s7 - 0.3125 * (s3 * n2 + s4 * n1));
  r[8] = r0 * (-0.5 * n8 + 0.375 * s8 - 0.3125 * (s4 * n2 + s5 * n1));
  r[9] = r0 * (-0.5 * n9 + 0.375 * s9 - 0.3125 * (s5 * n2));
}

// v = d * d, dim 3
__device__ __forceinline__ void jet_square_3d3(const double* d, double* v) {
  v[0] = d[0] * d[0];
  v[1] = 2.0 * (d[0] * d[1]);
  v[2] = 2.0 * (d[0] * d[2]);
  v[3] = 2.0 * (d[0] * d[3]);
  v[4] = 2.0 * (d[0] * d[4]) + d[1] * d[1];
  v[5] = 2.0 * (d[0] * d[5]) + 2.0 * (d[1] * d[2]);
  v[6] = 2.0 * (d[0] * d[6]) + d[2] * d[2];
  v[7] = 2.0 * (d[0] * d[7]) + 2.0 * (d[1] * d[3]);
  v[8] = 2.0 * (d[0] * d[8]) + 2.0 * (d[2] * d[3]);
  v[9] = 2.0 * (d[0] * d[9]) + d[3] * d[3];
  v[10] = 2.0 * (d[0] * d[10]) + 2.0 * (d[1] * d[4]);
  v[11] = 2.0 * (d[0] * d[11]) + 2.0 * (d[1] * d[5]) + 2.0 * (d[2] * d[4]);
  v[12] = 2.0 * (d[0] * d[12]) + 2.0 * (d[1] * d[6]) + 2.0 * (d[2] * d[5]);
  v[13] = 2.0 * (d[0] * d[13]) + 2.0 * (d[2] * d[6]);
  v[14] = 2.0 * (d[0] * d[14]) + 2.0 * (d[1] * d[7]) + 2.0 * (d[3] * d[4]);
  v[15] = 2.0 * (d[0] * d[15]) + 2.0 * (d[1] * d[8]) + 2.0 * (d[2] * d[7]) + 2.0 * (d[3] * d[5]);
  v[16] = 2.0 * (d[0] * d[16]) + 2.0 * (d[2] * d[8]) + 2.0 * (d[3] * d[6]);
  v[17] = 2.0 * (d[0] * d[17]) + 2.0 * (d[1] * d[9]) + 2.0 * (d[3] * d[7]);
  v[18] = 2.0 * (d[0] * d[18]) + 2.0 * (d[2] * d[9]) + 2.0 * (d[3] * d[8]);
  v[19] = 2.0 * (d[0] * d[19]) + 2.0 * (d[3] * d[9]);
}

// out = a * b, dim 3
__device__ __forceinline__ void jet_mul_3d3(const double* a, const double* b, double* out) {
  out[0] = a[0] * b[0];
  out[1] = a[0] * b[1] + a[1] * b[0];
  out[2] = a[0] * b[2] + a[2] * b[0];
  out[3] = a[0] * b[3] + a[3] * b[0];
  out[4] = a[0] * b[4] + a[1] * b[1] + a[4] * b[0];
  out[5] = a[0] * b[5] + a[1] * b[2] + a[2] * b[1] + a[5] * b[0];
  out[6] = a[0] * b[6] + a[2] * b[2] + a[6] * b[0];
  out[7] = a[0] * b[7] + a[1] * b[3] + a[3] * b[1] + a[7] * b[0];
  out[8] = a[0] * b[8] + a[2] * b[3] + a[3] * b[2] + a[8] * b[0];
  out[9] = a[0] * b[9] + a[3] * b[3] + a[9] * b[0];
  out[10] = a[0] * b[10] + a[1] * b[4] + a[4] * b[1] + a[10] * b[0];
  out[11] = a[0] * b[11] + a[1] * b[5] + a[2] * b[4] + a[4] * b[2] + a[5] * b[1] + a[11] * b[0];
  out[12] = a[0] * b[12] + a[1] * b[6] + a[2] * b[5] + a[5] * b[2] + a[6] * b[1] + a[12] * b[0];
  out[13] = a[0] * b[13] + a[2] * b[6] + a[6] * b[2] + a[13] * b[0];
  out[14] = a[0] * b[14] + a[1] * b[7] + a[3] * b[4] + a[4] * b[3] + a[7] * b[1] + a[14] * b[0];
  out[15] = a[0] * b[15] + a[1] * b[8] + a[2] * b[7] + a[3] * b[5] + a[5] * b[3] + a[7] * b[2] + a[8] * b[1] + a[15] * b[0];
  out[16] = a[0] * b[16] + a[2] * b[8] + a[3] * b[6] + a[6] * b[3] + a[8] * b[2] + a[16] * b[0];
  out[17] = a[0] * b[17] + a[1] * b[9] + a[3] * b[7] + a[7] * b[3] + a[9] * b[1] + a[17] * b[0];
  out[18] = a[0] * b[18] + a[2] * b[9] + a[3] * b[8] + a[8] * b[3] + a[9] * b[2] + a[18] * b[0];
  out[19] = a[0] * b[19] + a[3] * b[9] + a[9] * b[3] + a[19] * b[0];
}

// adjoint of b -> a * b at s: out_k = sum_j a_j s_(j+k), dim 3
__device__ __forceinline__ void jet_corr_3d3(const double* a, const double* s, double* out) {
  out[0] = a[0] * s[0] + a[1] * s[1] + a[2] * s[2] + a[3] * s[3] + a[4] * s[4] + a[5] * s[5] + a[6] * s[6] + a[7] * s[7] + a[8] * s[8] + a[9] * s[9] + a[10] * s[10] + a[11] * s[11] + a[12] * s[12] + a[13] * s[13] + a[14] * s[14] + a[15] * s[15] + a[16] * s[16] + a[17] * s[17] + a[18] * s[18] + a[19] * s[19];
  out[1] = a[0] * s[1] + a[1] * s[4] + a[2] * s[5] + a[3] * s[7] + a[4] * s[10] + a[5] * s[11] + a[6] * s[12] + a[7] * s[14] + a[8] * s[15] + a[9] * s[17];
  out[2] = a[0] * s[2] + a[1] * s[5] + a[2] * s[6] + a[3] * s[8] + a[4] * s[11] + a[5] * s[12] + a[6] * s[13] + a[7] * s[15] + a[8] * s[16] + a[9] * s[18];
  out[3] = a[0] * s[3] + a[1] * s[7] + a[2] * s[8] + a[3] * s[9] + a[4] * s[14] + a[5] * s[15] + a[6] * s[16] + a[7] * s[17] + a[8] * s[18] + a[9] * s[19];
  out[4] = a[0] * s[4] + a[1] * s[10] + a[2] * s[11] + a[3] * s[14];
  out[5] = a[0] * s[5] + a[1] * s[11] + a[2] * s[12] + a[3] * s[15];
  out[6] = a[0] * s[6] + a[1] * s[12] + a[2] * s[13] + a[3] * s[16];
  out[7] = a[0] * s[7] + a[1] * s[14] + a[2] * s[15] + a[3] * s[17];
  out[8] = a[0] * s[8] + a[1] * s[15] + a[2] * s[16] + a[3] * s[18];
  out[9] = a[0] * s[9] + a[1] * s[17] + a[2] * s[18] + a[3] * s[19];
  out[10] = a[0] * s[10];
  out[11] = a[0] * s[11];
  out[12] = a[0] * s[12];
  out[13] = a[0] * s[13];
  out[14] = a[0] * s[14];
  out[15] = a[0] * s[15];
  out[16] = a[0] * s[16];
  out[17] = a[0] * s[17];
  out[18] = a[0] * s[18];
  out[19] = a[0] * s[19];
}

// out_k += sum_j a_j s_(j+k), dim 3
__device__ __forceinline__ void jet_corr_add_3d3(const double* a, const double* s, double* out) {
  out[0] += a[0] * s[0] + a[1] * s[1] + a[2] * s[2] + a[3] * s[3] + a[4] * s[4] + a[5] * s[5] + a[6] * s[6] + a[7] * s[7] + a[8] * s[8] + a[9] * s[9] + a[10] * s[10] + a[11] * s[11] + a[12] * s[12] + a[13] * s[13] + a[14] * s[14] + a[15] * s[15] + a[16] * s[16] + a[17] * s[17] + a[18] * s[18] + a[19] * s[19];
  out[1] += a[0] * s[1] + a[1] * s[4] + a[2] * s[5] + a[3] * s[7] + a[4] * s[10] + a[5] * s[11] + a[6] * s[12] + a[7] * s[14] + a[8] * s[15] + a[9] * s[17];
  out[2] += a[0] * s[2] + a[1] * s[5] + a[2] * s[6] + a[3] * s[8] + a[4] * s[11] + a[5] * s[12] + a[6] * s[13] + a[7] * s[15] + a[8] * s[16] + a[9] * s[18];
  out[3] += a[0] * s[3] + a[1] * s[7] + a[2] * s[8] + a[3] * s[9] + a[4] * s[14] + a[5] * s[15] + a[6] * s[16] + a[7] * s[17] + a[8] * s[18] + a[9] * s[19];
  out[4] += a[0] * s[4] + a[1] * s[10] + a[2] * s[11] + a[3] * s[14];
  out[5] += a[0] * s[5] + a[1] * s[11] + a[2] * s[12] + a[3] * s[15];
  out[6] += a[0] * s[6] + a[1] * s[12] + a[2] * s[13] + a[3] * s[16];
  out[7] += a[0] * s[7] + a[1] * s[14] + a[2] * s[15] + a[3] * s[17];
  out[8] += a[0] * s[8] + a[1] * s[15] + a[2] * s[16] + a[3] * s[18];
  out[9] += a[0] * s[9] + a[1] * s[17] + a[2] * s[18] + a[3] * s[19];
  out[10] += a[0] * s[10];
  out[11] += a[0] * s[11];
  out[12] += a[0] * s[12];
  out[13] += a[0] * s[13];
  out[14] += a[0] * s[14];
  out[15] += a[0] * s[15];
  out[16] += a[0] * s[16];
  out[17] += a[0] * s[17];
  out[18] += a[0] * s[18];
  out[19] += a[0] * s[19];
}

// r = v^(-1/2), v_0 > 0, dim 3
__device__ __forceinline__ void jet_rsqrt_3d3(const double* v, double* r) {
  const double r0 = 1.0 / sqrt(v[0]);
  const double w = r0 * r0;
  const double n1 = v[1] * w;
  const double n2 = v[2] * w;
  const double n3 = v[3] * w;
  const double n4 = v[4] * w;
  const double n5 = v[5] * w;
  const double n6 = v[6] * w;
  const double n7 = v[7] * w;
  const double n8 = v[8] * w;
  const double n9 = v[9] * w;
  const double n10 = v[10] * w;
  const double n11 = v[11] * w;
  const double n12 = v[12] * w;
  const double n13 = v[13] * w;
  const double n14 = v[14] * w;
  const double n15 = v[15] * w;
  const double n16 = v[16] * w;
  const double n17 = v[17] * w;
  const double n18 = v[18] * w;
  const double n19 = v[19] * w;
  const double s4 = n1 * n1;
  const double s5 = 2.0 * (n1 * n2);
  const double s6 = n2 * n2;
  const double s7 = 2.0 * (n1 * n3);
  const double s8 = 2.0 * (n2 * n3);
  const double s9 = n3 * n3;
  const double s10 = 2.0 * (n1 * n4);
  const double s11 = 2.0 * (n1 * n5) + 2.0 * (n2 * n4);
  const double s12 = 2.0 * (n1 * n6) + 2.0 * (n2 * n5);
  const double s13 = 2.0 * (n2 * n6);
  const double s14 = 2.0 * (n1 * n7) + 2.0 * (n3 * n4);
  const double s15 = 2.0 * (n1 * n8) + 2.0 * (n2 * n7) + 2.0 * (n3 * n5);
  const double s16 = 2.0 * (n2 * n8) + 2.0 * (n3 * n6);
  const double s17 = 2.0 * (n1 * n9) + 2.0 * (n3 * n7);
  const double s18 = 2.0 * (n2 * n9) + 2.0 * (n3 * n8);
  const double s19 = 2.0 * (n3 * n9);
  r[0] = r0;
  r[1] = r0 * (-0.5 * n1);
  r[2] = r0 * (-0.5 * n2);
  r[3] = r0 * (-0.5 * n3);
  r[4] = r0 * (-0.5 * n4 + 0.375 * s4);
  r[5] = r0 * (-0.5 * n5 + 0.375 * s5);
  r[6] = r0 * (-0.5 * n6 + 0.375 * s6);
  r[7] = r0 * (-0.5 * n7 + 0.375 * s7);
  r[8] = r0 * (-0.5 * n8 + 0.375 * s8);
  r[9] = r0 * (-0.5 * n9 + 0.375 * s9);
  r[10] = r0 * (-0.5 * n10 + 0.375 * s10 - 0.3125 * (s4 * n1));
  r[11] = r0 * (-0.5 * n11 + 0.375 * s11 - 0.3125 * (s4 * n2 + s5 * n1));
  r[12] = r0 * (-0.5 * n12 + 0.375 * s12 - 0.3125 * (s5 * n2 + s6 * n1));
  r[13] = r0 * (-0.5 * n13 + 0.375 * s13 - 0.3125 * (s6 * n2));
  r[14] = r0 * (-0.5 * n14 + 0.375 * s14 - 0.3125 * (s4 * n3 + s7 * n1));
  r[15] = r0 * (-0.5 * n15 + 0.375 * s15 - 0.3125 * (s5 * n3 + s7 * n2 + s8 * n1));
  r[16] = r0 * (-0.5 * n16 + 0.375 * s16 - 0.3125 * (s6 * n3 + s8 * n2));
  r[17] = r0 * (-0.5 * n17 + 0.375 * s17 - 0.3125 * (s7 * n3 + s9 * n1));
  r[18] = r0 * (-0.5 * n18 + 0.375 * s18 - 0.3125 * (s8 * n3 + s9 * n2));
  r[19] = r0 * (-0.5 * n19 + 0.375 * s19 - 0.3125 * (s9 * n3));
}

}  // namespace flashns_b200
